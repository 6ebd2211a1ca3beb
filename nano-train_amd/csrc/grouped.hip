// bf16 products grouped by expert: the rows of x [R, K] are sorted by expert, expert e
// owns rows offsets[e] .. offsets[e + 1] - 1 and the weight W_e [N, K]:
//   y = x W_e^T,  dx = dy W_e (by the row's expert),  dW_e = dy^T x over e's rows
// Products of bf16 values are exact in fp32 and summed in fp32 on the matrix cores;
// results are rounded once.  Rows behind the last expert's are zero in y and dx, and
// so is dW_e of an expert without rows.  How the rows divide is known to the device
// only: each workgroup reads the offsets (clamped to R and to what came before, so that no table
// leads out of a buffer or leaves a row out) and finds its tile.
//
// Matrix-core bound where experts have a few hundred rows and more, on the tiles of
// ntlb_bf16_tile.h (32768 rows of 32 experts, 4096 x 7168: y 1.66 ms, 1.16 PFLOP/s; dx 1.75;
// dW 1.89); bound by the weights' way from HBM below (256 rows of them: y 307 to 316 us, 6 TB/s).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "ntlb_bf16_tile.h"
#include "ntlb_device.h"
#include "ntlb_host.h"
#include "ntlb_kept.h"
#include "ntlb_splitk.h"

namespace ntlb {
namespace grouped {

using namespace tile;

struct Args {
  const uint8_t* a;  // x or dy
  int64_t lda;       // bytes, as the others
  const uint8_t* b;  // W, or x (dW)
  int64_t ldb, b_expert;
  const int32_t* offsets;
  int64_t R;
  int E;
  int64_t k;  // contraction (y: K, dx: N)
  int64_t M;  // rows of the result (dW: N)
  int64_t N;  // columns of the result
  uint16_t* out;
  int64_t ldo;  // elements
  int parts;    // y, dx by tiles of 128: ranges of the contraction, each to a matrix of its own in `sums`
  float* sums;  // [parts][R][lds]
  int64_t lds;
};

// over the lanes up to each, of values that are not negative
__device__ __forceinline__ int wave_scan_max(int v) {
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false));  // from 1, 2, 4 and 8 lanes before, of 16
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false));
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false));
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false));
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false));  // lane 15 to 16 .. 31, 47 to 48 .. 63
  return max(v, __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false));  // lane 31 to 32 .. 63
}

// The rows of experts c .. c + 63, a lane each (E: those behind the last expert's; past it: none).
// An offset below one before it counts as that one: whatever the table holds, experts' rows
// follow one another and cover all R, so their tiles are never more than the grid has
// and no row is left out.  reached: where the experts before c end; then where these do.
struct Rows {
  int lo, n;
  __device__ __forceinline__ Rows(const Args& g, int c, int lane, int& reached) {
    const int R = (int)g.R, e = c + lane;
    const int to = wave_scan_max(max(e < g.E ? min(g.offsets[e + 1], R) : R, reached)), before = __shfl_up(to, 1);
    lo = lane ? before : reached;
    n = to - lo;
    reached = __builtin_amdgcn_readlane(to, 63);
  }
};

__device__ __forceinline__ int wave_scan(int v, int lane) {  // inclusive
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int o = __shfl_up(v, d);
    v += lane >= d ? o : 0;
  }
  return v;
}

// The order of a grid's tiles.  Workgroup pid runs on XCD pid % 8, 32 of one XCD at a
// time (its compute units): those take 32 tiles next to each other, which share
// their operands in the XCD's L2.
__device__ __forceinline__ int order(int pid) {
  const int at = pid >> 3;
  return (((pid & 7) + 8 * (at >> 5)) << 5) + (at & 31);
}
static int64_t ordered_grid(int64_t tiles) { return cdiv(tiles, 256) * 256; }

// how many of the wave's values come before this lane's, highest first
__device__ __forceinline__ int wave_place(int v, int lane, int lanes) {
  int place = 0;
  for (int j = 0; j < lanes; ++j) {
    const int o = __builtin_amdgcn_readlane(v, j);
    place += o > v || (o == v && j < lane);
  }
  return lane < lanes ? place : -1;
}

// Tile pid of all experts' rows (D each) by num_n column tiles, expert after expert,
// then the rows behind the last expert's (e == E), each as often as the contraction
// has ranges.  Each XCD walks a contiguous range, so that few of them read one
// expert's weights.  m0: first row, of the expert's n; tn:
// column tile.
struct Found {
  int e, lo, n, m0, tn, part;
};
// row tiles walked side by side: of an expert for y and dx, of dW (32768 rows, 32 experts,
// 4096 x 7168: y 1716 us with four, 1698 with eight; dx 1810, 1798; dW 1903, 1947)
constexpr int GROUP_M = 8, GROUP_W = 4;
template <int D>
__device__ __forceinline__ bool find(const Args& g, int num_n, int pid, Found& f) {
  const int lane = threadIdx.x & 63;
  int total = 0, reached = 0;
  for (int c = 0; c <= g.E; c += 64) total += __builtin_amdgcn_readlane(wave_scan((Rows(g, c, lane, reached).n + D - 1) / D, lane), 63);
  total *= num_n * g.parts;
  if (pid >= total) return false;
  const int xcd = pid & 7, per = total >> 3, extra = total & 7;
  int q = xcd * per + min(xcd, extra) + (pid >> 3);
  f.part = D == 128 ? q % g.parts : 0;  // a tile's ranges on one XCD
  if (D == 128) q /= g.parts;
  reached = 0;
  for (int c = 0; c <= g.E; c += 64) {
    const Rows r(g, c, lane, reached);
    const int m = (r.n + D - 1) / D * num_n, upto = wave_scan(m, lane);
    const uint64_t b = __ballot(upto > q);
    if (b) {
      const int at = __builtin_ctzll(b);
      f.e = c + at;
      f.lo = __builtin_amdgcn_readlane(r.lo, at);
      f.n = __builtin_amdgcn_readlane(r.n, at);
      const int t = q - (__builtin_amdgcn_readlane(upto, at) - __builtin_amdgcn_readlane(m, at));
      const int first = t / (GROUP_M * num_n) * GROUP_M, side = min((f.n + D - 1) / D - first, GROUP_M), in = t - first * num_n;
      f.m0 = (first + in % side) * D;
      f.tn = in / side;
      return true;
    }
    q -= __builtin_amdgcn_readlane(upto, 63);
  }
  return false;
}

// the steps of a tile's range
template <int D>
__device__ __forceinline__ void steps_of(const Args& g, const Found& f, int& k0, int& k1) {
  const int nk = (int)((g.k + KSTEP - 1) / KSTEP);
  k0 = D == 128 ? f.part * nk / g.parts : 0;
  k1 = D == 128 ? (f.part + 1) * nk / g.parts : nk;
}

// A wave's result rows through its part of a stage
template <int D>
__device__ __forceinline__ void store_tile(const v4f (&acc)[D / 32][4], int wave, int wm, int wn, int lane, int64_t m0,
                                           int64_t n0, int64_t M, int64_t N, uint16_t* out, int64_t ldo, uint8_t* stage) {
  constexpr int MT = D / 32;
  store_bf16<MT, true>(stage + wave * 4096, lane, m0 + wm * 16 * MT, n0 + wn * 64, M, N, out, ldo, [&](int tm, int tn, float (&v)[4]) {
#pragma unroll
    for (int r = 0; r < 4; ++r) v[r] = acc[tm][tn][r];
  });
}

// the same of one range's sums, fp32
template <int D>
__device__ __forceinline__ void store_sums(const v4f (&acc)[D / 32][4], int wm, int wn, int lane, int64_t m0, int64_t n0,
                                           int64_t M, float* out, int64_t ldo) {
  constexpr int MT = D / 32;
#pragma unroll
  for (int tm = 0; tm < MT; ++tm) {
    const int64_t m = m0 + wm * 16 * MT + tm * 16 + (lane & 15);
    if (m >= M) continue;
#pragma unroll
    for (int tn = 0; tn < 4; ++tn) {
      const int64_t n = n0 + wn * 64 + tn * 16 + (lane >> 4) * 4;
      if (n < ldo) *reinterpret_cast<v4f*>(out + m * ldo + n) = acc[tm][tn];  // the pitch is a multiple of four
    }
  }
}

// the ranges' sums added in their order
__global__ void __launch_bounds__(256) join_kernel(Args g) {
  const int64_t quads = g.lds / 4, i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= g.R * quads) return;
  const int64_t m = i / quads, n = (i - m * quads) * 4;
  const float* p = g.sums + m * g.lds + n;
  v4f v = *reinterpret_cast<const v4f*>(p);
#pragma unroll 4
  for (int k = 1; k < g.parts; ++k) v += *reinterpret_cast<const v4f*>(p + k * (g.R * g.lds));
  uint16_t* o = g.out + m * g.ldo + n;
  const uint32_t a = pack_bf16(v[0], v[1]), b = pack_bf16(v[2], v[3]);
  if (n + 4 <= g.N) {
    *reinterpret_cast<u32x2_2*>(o) = (u32x2_2){a, b};
  } else {
    o[0] = (uint16_t)a;
    if (n + 1 < g.N) o[1] = (uint16_t)(a >> 16);
    if (n + 2 < g.N) o[2] = (uint16_t)b;
  }
}

#define NTLB_ZERO_ACC(D)                   \
  v4f acc[D / 32][4];                      \
  _Pragma("unroll") for (int i = 0; i < D / 32; ++i) _Pragma("unroll") for (int j = 0; j < 4; ++j) acc[i][j] = (v4f){0.f, 0.f, 0.f, 0.f}

// y: W by rows.  Both operands come in the same way.  By 256 tiles x's copies run two
// steps ahead (32768 rows of 32 experts, 4096 x 7168: 1640 us, W's instead 1733), by 128
// those of W, which then is the larger and read once (64 experts of 16 rows, 2048 x
// 4096: x's 243 us, W's 233; 32 of 40, 4096 x 7168: 430, 418).
template <int D>
__global__ void __launch_bounds__(2 * D, D == 256 ? 1 : 2) rows_kernel(Args g) {
  NTLB_TILE_STAGES_AHEAD(D);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  constexpr int WAVES_N = D / 64;
  const int wm = wave / WAVES_N, wn = wave % WAVES_N;
  Found f;
  if (!find<D>(g, (int)((g.N + D - 1) / D), (int)blockIdx.x, f)) return;
  const int64_t m0 = f.m0, n0 = (int64_t)f.tn * D;
  const bool idle = __builtin_amdgcn_readfirstlane(f.m0 + wm * (D / 2) >= f.n);
  NTLB_ZERO_ACC(D);
  if (f.e < g.E) {
    RowWalk<D> ca, cb;
    ca.init(Mat{g.a + (int64_t)f.lo * g.lda, g.lda, f.n, g.k}, m0, wave, lane);
    cb.init(Mat{g.b + (int64_t)f.e * g.b_expert, g.ldb, g.N, g.k}, n0, wave, lane);
    int k0, k1;
    steps_of<D>(g, f, k0, k1);
    prime_ahead<D == 128>(ca, cb, k0, wave, stages);
    multiply_ahead<D, D == 128>(ca, cb, k0, k1, acc, wm, wn, wave, lane, stages, idle);
  }
  if (D == 128 && g.parts > 1)
    store_sums<D>(acc, wm, wn, own_lane(), m0, n0, f.n, g.sums + (f.part * g.R + f.lo) * g.lds, g.lds);
  else
    store_tile<D>(acc, wave, wm, wn, own_lane(), m0, n0, f.n, g.N, g.out + (int64_t)f.lo * g.ldo, g.ldo, stage_4);
}

// dx: W transposed
template <int D>
__global__ void __launch_bounds__(2 * D, D == 256 ? 1 : 2) inputs_kernel(Args g) {
  NTLB_TILE_STAGES(D);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  constexpr int WAVES_N = D / 64;
  const int wm = wave / WAVES_N, wn = wave % WAVES_N;
  Found f;
  if (!find<D>(g, (int)((g.N + D - 1) / D), (int)blockIdx.x, f)) return;
  const int64_t m0 = f.m0, n0 = (int64_t)f.tn * D;
  const bool idle = __builtin_amdgcn_readfirstlane(f.m0 + wm * (D / 2) >= f.n);
  NTLB_ZERO_ACC(D);
  if (f.e < g.E) {
    RowCopy<D> ca;
    TrCopy<D> cb;
    ca.init(Mat{g.a + (int64_t)f.lo * g.lda, g.lda, f.n, g.k}, m0, wave, lane);
    cb.init(Mat{g.b + (int64_t)f.e * g.b_expert, g.ldb, g.N, g.k}, n0, wave, lane);
    int k0, k1;
    steps_of<D>(g, f, k0, k1);
    multiply<D, false, true>(ca, cb, k0, k1, acc, wm, wn, wave, lane, la0, lb0, la1, lb1, idle);
  }
  if (D == 128 && g.parts > 1)
    store_sums<D>(acc, wm, wn, lane, m0, n0, f.n, g.sums + (f.part * g.R + f.lo) * g.lds, g.lds);
  else
    store_tile<D>(acc, wave, wm, wn, lane, m0, n0, f.n, g.N, g.out + (int64_t)f.lo * g.ldo, g.ldo, la1);
}

// dW: every expert's tiles, each with the expert's rows as its contraction.  Experts
// with many rows come first (among 64 neighbours).  A contraction of a few hundred
// rows is 10 to 20 steps, so what stands around it counts: a workgroup stays for
// tile after tile, and the next one's first copies are under way while this one is
// stored.  Measured at 32 experts of 1024 rows on average, 4096 x 7168: 2.01 ms with an
// eighth of each expert's tiles to each XCD, whose compute units then work on
// different ones and read twice as much into L2 (3.2 GB); 32 at a time 1.81; without
// staying 1.93.
template <int D>
__global__ void __launch_bounds__(2 * D, D == 256 ? 1 : 2) weight_kernel(Args g, int count) {
  NTLB_TILE_STAGES(D);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  constexpr int WAVES_N = D / 64;
  const int wm = wave / WAVES_N, wn = wave % WAVES_N;
  const int num_n = (int)((g.N + D - 1) / D), num_m = (int)((g.M + D - 1) / D), tiles = num_m * num_n;
  int chunk = -1, place = 0, lo = 0, n = 0;  // of 64 experts, a lane each: how many have more rows; its rows
  struct Tile {
    int e, lo, n, m, c;  // m, c: row and column tile
  };
  // the next tile from pid on, and its pid; count: none is left
  auto next = [&](int pid, Tile& t) {
    for (; pid < count; pid += (int)gridDim.x) {
      const int at = order(pid), rank = at / tiles, q = at - rank * tiles;
      if (rank >= g.E) continue;
      const int c = rank & ~63;
      if (c != chunk) {
        int reached = 0;
        for (int i = 0; i < c; i += 64) Rows(g, i, lane, reached);
        chunk = c;
        const Rows r(g, c, lane, reached);
        lo = r.lo;
        n = r.n;
        place = wave_place(n, lane, min(g.E - c, 64));
      }
      const int who = __builtin_ctzll(__ballot(place == (rank & 63)));
      t.e = c + who;
      t.lo = __builtin_amdgcn_readlane(lo, who);
      t.n = __builtin_amdgcn_readlane(n, who);
      const int first = q / (GROUP_W * num_n) * GROUP_W, side = min(num_m - first, GROUP_W), in = q - first * num_n;
      t.m = first + in % side;
      t.c = in / side;
      break;
    }
    return pid;
  };
  TrCopy<D> ca, cb;
  auto begin = [&](const Tile& t) {
    ca.init(Mat{g.a + (int64_t)t.lo * g.lda, g.lda, g.M, t.n}, (int64_t)t.m * D, wave, lane);
    cb.init(Mat{g.b + (int64_t)t.lo * g.ldb, g.ldb, g.N, t.n}, (int64_t)t.c * D, wave, lane);
    prime(ca, cb, 0, wave, la0, lb0);
  };
  Tile t, u;
  int pid = next((int)blockIdx.x, t);
  if (pid >= count) return;
  if (t.n > 0) begin(t);
  for (;;) {
    NTLB_ZERO_ACC(D);
    if (t.n > 0) multiply<D, true, true, true>(ca, cb, 0, (t.n + KSTEP - 1) / KSTEP, acc, wm, wn, wave, lane, la0, lb0, la1, lb1);
    pid = next(pid + (int)gridDim.x, u);
    if (pid < count && u.n > 0) begin(u);
    store_tile<D>(acc, wave, wm, wn, own_lane(), (int64_t)t.m * D, (int64_t)t.c * D, g.M, g.N, g.out + (int64_t)t.e * g.M * g.ldo, g.ldo, la1);
    if (pid >= count) break;
    t = u;
  }
}

// ---------------------------------------------------------------------------
// y where experts have few rows: bound by the weights, read once.  A workgroup takes
// 16 rows of W_e and all of e's rows (64 at a time); its four waves take
// 64-column chunks in turn, straight from memory into fragments (a lane 32 bytes of
// a row, 16 rows a fragment, the same columns of x and W), and their sums meet in LDS.
// 8 rows of as many experts, 4096 x 7168: 80 us, 5.9 TB/s; with W's loads hinted as read once
// 95, by eight waves or 32 rows of W_e no better.
// ---------------------------------------------------------------------------
constexpr int FEW_WAVES = 4;

template <int MT>
__device__ __forceinline__ void few_rows(const Args& g, const uint8_t* wp, const uint8_t* xp, int lo, int m0, int n, int64_t n0,
                                         int wave, int lane, float4* sums) {
  const int r = lane & 15, gl = lane >> 4, chunks = (int)((g.k + 63) / 64);
  const uint8_t* wr = wp + min<int64_t>(n0 + r, g.N - 1) * g.ldb + gl * 32;
  const uint8_t* xr[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) xr[i] = xp + (int64_t)(lo + min(m0 + 16 * i + r, n - 1)) * g.lda + gl * 32;
  v4f acc[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) acc[i] = (v4f){0.f, 0.f, 0.f, 0.f};
  const int whole = (int)(g.k / 64);
  auto load = [&](const uint8_t* p, int c) {
    v8i v;
    const uint4 a = *reinterpret_cast<const uint4*>(p + (int64_t)c * 128), b = *reinterpret_cast<const uint4*>(p + (int64_t)c * 128 + 16);
    v[0] = (int)a.x; v[1] = (int)a.y; v[2] = (int)a.z; v[3] = (int)a.w;
    v[4] = (int)b.x; v[5] = (int)b.y; v[6] = (int)b.z; v[7] = (int)b.w;
    return v;
  };
  auto add = [&](const v8i& w, const v8i (&x)[MT]) {
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      acc[i] = mma<0>(w, x[i], acc[i]);
      acc[i] = mma<1>(w, x[i], acc[i]);
    }
  };
  // a wave's chunks, U of them in flight
  constexpr int U = MT == 4 ? 2 : 4;
  int c = wave;
  for (; c + (U - 1) * FEW_WAVES < whole; c += U * FEW_WAVES) {
    v8i w[U], x[U][MT];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      w[u] = load(wr, c + u * FEW_WAVES);
#pragma unroll
      for (int i = 0; i < MT; ++i) x[u][i] = load(xr[i], c + u * FEW_WAVES);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) add(w[u], x[u]);
  }
  for (; c < whole; c += FEW_WAVES) {
    const v8i w = load(wr, c);
    v8i x[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) x[i] = load(xr[i], c);
    add(w, x);
  }
  if (whole < chunks && whole % FEW_WAVES == wave) {
    // the last columns: 16-byte pieces past k are taken as zero
    const int left = (int)(g.k - (int64_t)whole * 64) - gl * 16;
    auto part = [&](const uint8_t* p) {
      v8i v = {0, 0, 0, 0, 0, 0, 0, 0};
      const uint8_t* q = p + (int64_t)whole * 128;
      if (left > 0) {
        const uint4 a = *reinterpret_cast<const uint4*>(q);
        v[0] = (int)a.x; v[1] = (int)a.y; v[2] = (int)a.z; v[3] = (int)a.w;
      }
      if (left > 8) {
        const uint4 a = *reinterpret_cast<const uint4*>(q + 16);
        v[4] = (int)a.x; v[5] = (int)a.y; v[6] = (int)a.z; v[7] = (int)a.w;
      }
      return v;
    };
    const v8i w = part(wr);
    v8i x[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) x[i] = part(xr[i]);
    add(w, x);
  }
  __syncthreads();  // the sums of the rows before have been read
#pragma unroll
  for (int i = 0; i < MT; ++i) sums[(i * FEW_WAVES + wave) * 64 + lane] = make_float4(acc[i][0], acc[i][1], acc[i][2], acc[i][3]);
  __syncthreads();
  // lane: row m0 + 16 i + lane % 16, columns n0 + 4 (lane / 16) ..
  for (int i = wave; i < MT; i += FEW_WAVES) {
    float4 s = sums[i * FEW_WAVES * 64 + lane];
#pragma unroll
    for (int w = 1; w < FEW_WAVES; ++w) {
      const float4 o = sums[(i * FEW_WAVES + w) * 64 + lane];
      s.x += o.x;
      s.y += o.y;
      s.z += o.z;
      s.w += o.w;
    }
    const int m = m0 + 16 * i + r;
    const int64_t c = n0 + 4 * gl;
    if (m >= n || c >= g.N) continue;
    uint16_t* o = g.out + (int64_t)(lo + m) * g.ldo + c;
    const uint32_t a = pack_bf16(s.x, s.y), b = pack_bf16(s.z, s.w);
    if (c + 4 <= g.N) {
      *reinterpret_cast<u32x2_2*>(o) = (u32x2_2){a, b};
    } else {
      o[0] = (uint16_t)a;
      if (c + 1 < g.N) o[1] = (uint16_t)(a >> 16);
      if (c + 2 < g.N) o[2] = (uint16_t)b;
    }
  }
}

__global__ void __launch_bounds__(64 * FEW_WAVES) few_kernel(Args g, int blocks) {
  __shared__ float4 sums[4 * FEW_WAVES * 64];
  const int e = (int)blockIdx.x / blocks, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t n0 = (int64_t)((int)blockIdx.x - e * blocks) * 16;
  const int to = e < g.E ? min(g.offsets[e + 1], (int)g.R) : (int)g.R;
  if (to <= (e ? g.offsets[e] : 0)) return;  // no rows, whatever came before (8 rows of 32 experts: 83 us without, 80 with)
  int lo = 0;
  for (int c = 0; c < e; c += 64) Rows(g, c, min(lane, e - 1 - c), lo);
  const int n = to - lo;
  if (e == g.E) {  // rows behind the last expert's
    for (int i = threadIdx.x; i < n * 16; i += 64 * FEW_WAVES) {
      const int64_t c = n0 + i % 16;
      if (c < g.N) g.out[(int64_t)(lo + i / 16) * g.ldo + c] = 0;
    }
    return;
  }
  const uint8_t* wp = uniform64(g.b + (int64_t)e * g.b_expert);
  for (int m0 = 0; m0 < n; m0 += 64) {
    const int left = n - m0;
    if (left <= 16) few_rows<1>(g, wp, g.a, lo, m0, n, n0, wave, lane, sums);
    else if (left <= 32) few_rows<2>(g, wp, g.a, lo, m0, n, n0, wave, lane, sums);
    else few_rows<4>(g, wp, g.a, lo, m0, n, n0, wave, lane, sums);
  }
}

// ---------------------------------------------------------------------------
// x kept in 8 bits, and back (HBM-bound): 16 lanes a tile of 128 columns.  32768 x 7168:
// 135 us (5.2 TB/s) and 109 (6.5)
// ---------------------------------------------------------------------------
struct Keep {
  const uint8_t* x;  // bf16 rows, 16-byte pieces
  int64_t ldx;       // bytes
  int64_t tiles;
  int K;
  TileRows by;
  uint8_t* kc;
  uint8_t* ke;
};
__global__ void __launch_bounds__(256) keep_kernel(Keep g) {
  const int64_t q = ((int64_t)blockIdx.x * 256 + threadIdx.x) / 16;
  const bool on = q < g.tiles;
  const uint32_t t = (uint32_t)(on ? q : g.tiles - 1), row = g.by.row(t);
  const int c = (int)(t - row * g.by.per_row) * KEPT_TILE + (threadIdx.x & 15) * 8;
  uint4 v = make_uint4(0, 0, 0, 0);
  if (c < g.K) v = *reinterpret_cast<const uint4*>(g.x + (int64_t)row * g.ldx + 2 * c);  // the pitch holds whole pieces
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  float f[8];
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    f[i] = c + i < g.K ? ((i & 1) ? __uint_as_float(w[i >> 1] & 0xFFFF0000u) : __uint_as_float(w[i >> 1] << 16)) : 0.f;
    m = max(m, finite_bits(f[i]));
  }
  const uint32_t byte = kept_byte(tile_max<16>(m));
  if (!on) return;
  const float inv = kept_inverse(byte);
  store8_nt(g.kc + (int64_t)row * (g.by.per_row * (int64_t)KEPT_TILE) + c, kept_codes4(f[0], f[1], f[2], f[3], inv),
            kept_codes4(f[4], f[5], f[6], f[7], inv));
  if ((threadIdx.x & 15) == 0) g.ke[t] = (uint8_t)byte;
}

__global__ void __launch_bounds__(256) values_kernel(Keep g, uint8_t* out, int64_t ldo) {
  const int64_t q = ((int64_t)blockIdx.x * 256 + threadIdx.x) / 16;
  if (q >= g.tiles) return;
  const uint32_t t = (uint32_t)q, row = g.by.row(t);
  const int c = (int)(t - row * g.by.per_row) * KEPT_TILE + (threadIdx.x & 15) * 8;
  if (c >= g.K) return;
  const uint2 v = *reinterpret_cast<const uint2*>(g.kc + (int64_t)row * (g.by.per_row * (int64_t)KEPT_TILE) + c);
  const float scale = kept_scale(g.ke[t]);
  float a[4], b[4];
  kept_values4(v.x, scale, a);
  kept_values4(v.y, scale, b);
  // 4 significant bits: exact in bf16, down to its least step of 2^-133
  *reinterpret_cast<uint4*>(out + (int64_t)row * ldo + 2 * c) =
      make_uint4(pack_bf16(a[0], a[1]), pack_bf16(a[2], a[3]), pack_bf16(b[0], b[1]), pack_bf16(b[2], b[3]));
}

constexpr int64_t MAX_PITCH = 1 << 22, MAX_EXPERTS = 4096;
constexpr int64_t MAX_THREADS = ((int64_t)1 << 32) - 1;  // of a launch

static int check(const char* fn, int64_t R, int64_t E, int64_t N, int64_t K, const int32_t* offsets) {
  clear_error();
  if (R < 0 || E < 1 || N < 1 || K < 1) return fail(NTLB_EINVAL, "%s: bad shape R %lld E %lld N %lld K %lld", fn, (long long)R, (long long)E, (long long)N, (long long)K);
  if (E > MAX_EXPERTS || R > ((int64_t)1 << 30) || N > MAX_PITCH || K > MAX_PITCH) return fail(NTLB_EUNSUPPORTED, "%s: R %lld E %lld N %lld K %lld is too large", fn, (long long)R, (long long)E, (long long)N, (long long)K);
  if (!offsets || !aligned(offsets, 4)) return fail(NTLB_EINVAL, "%s: bad offsets", fn);
  return NTLB_OK;
}
// rows of whole 16-byte pieces
static bool fits(const void* p, int64_t ld, int64_t cols) {
  return p && aligned(p, 16) && ld % 8 == 0 && ld >= cols && ld <= MAX_PITCH;
}
static int bad(const char* fn, const char* what) {
  return fail(NTLB_EINVAL, "%s: %s must lie in 16-byte aligned rows of whole 16-byte pieces, at most %lld values apart", fn, what, (long long)MAX_PITCH);
}

// workgroups that stream: 16 rows of each expert's weights, and of the columns of the rows behind
static int64_t few_blocks(int64_t E, int64_t N) { return (E + 1) * cdiv(N, 16); }

// How y and dx are formed for N columns over K: by streaming the weights past few rows
// (FEW, y only), or by tiles of D, their contraction in `parts` ranges.
//
// How many rows an expert has is known to the device only; the host goes by R rows over
// the experts that can have some.
//
// In the figures rows are averages over experts of which the most popular has two to nine times
// as many; in brackets, as many rows for each.
//
// Few rows stream, where their grid fits a launch: past the weights goes x once for 16 of their rows, tiles of some
// rows take a tile's time.  Up to 2 to 32 rows an expert, by the weights' size: 768 x 1024
// of 8 experts 12 us at 32 rows and 11 by tiles [8 and 10], at 64 rows 21 and 11 [12 and 10]; 2048 x 4096
// of 8 25 us at 4 and 39 by whole tiles [24 and 39], at 16 38 and 26 by ranges [31 and 25]; 4096 x 7168 of 32
// 309 us at 2 and 306 [307 and 306], at 4 326 and 307 [322 and 307].
//
// Tiles by the rounds that they take, one workgroup of 256 tiles a compute unit or two of
// 128, a round of the latter 2/3 of the former's time: 4096 x 7168, 32 experts of 256
// rows, y 586 us by 256 tiles and 658 [455 and 582], dx 636 and 683 [498 and 619], of 64 rows y 474 and 412
// [359 and 321], dx 401 and 377 [392 and 369]; 768 x 1024, 64 experts of 256 rows, y 49 and 36 [30 and 34].
// Where the two are near each other, how the rows divide decides, which the rule cannot see: 2048 x
// 4096, 8 experts of 512, y 76 and 97 [80 and 58], dx 95 and 85 [56 and 68]; 4096 x 7168, 32 of
// 128, y 511 and 463 [374 and 367], dx 437 and 513 [416 and 413].
//
// Tiles that leave compute units idle divide the contraction where that pays: a step of
// 64 is half a us, the ranges' join 4, and their sums go out and in at 4 TB/s.  One expert,
// 4096 x 4096, 64 rows 38 us whole and 14 in 8 ranges; 2048 x 4096, 8 experts of 64 rows 43 and
// 33 in 3 ranges [39 and 29] (in 4, more workgroups than places, 42 [30]); 768 x 1024, 8 experts of 250
// rows 12 whole and 18 in 2.
struct Plan {
  bool few;
  int D, parts;
};
static Plan plan_of(int64_t R, int64_t E, int64_t N, int64_t K, bool y) {
  const int64_t live = std::min(R, E), cus = split_device_cus(), nk = cdiv(K, KSTEP);
  const bool fits = few_blocks(E, N) * 64 * FEW_WAVES <= MAX_THREADS;
  Plan p{y && fits && R <= live * std::clamp<int64_t>(400000000 / (live * N * K), 2, 32), 128, 1};
  if (p.few) return p;
  auto tiles = [&](int64_t D) {  // a last one of every expert's is half empty
    return (live == 1 ? cdiv(R, D) : std::max(live, R / D + cdiv(live, 2))) * cdiv(N, D);
  };
  const int64_t t = tiles(128);
  if (3 * cdiv(tiles(256), cus) <= 2 * cdiv(t, 2 * cus)) {
    p.D = 256;
  } else if (t < cus) {  // ranges of four steps at least, and sums of 64 MB at most
    const int64_t sums = R * cdiv(N, 4) * 16, most = std::min({(2 * cus - cus / 8) / t, nk / 4, (int64_t)16, ((int64_t)64 << 20) / sums});
    double best = 0;
    for (int n = 2; n <= most; ++n) {
      const double gain = 0.5 * (double)nk * (n - 1) / n - 4 - (double)(n * sums) * 5e-7;
      if (gain > best) {
        best = gain;
        p.parts = n;
      }
    }
  }
  return p;
}
static int64_t sums_bytes(const Plan& p, int64_t R, int64_t N) { return p.parts > 1 ? p.parts * R * cdiv(N, 4) * 16 : 0; }
// workgroups of the tiles: the last one of each expert that can have rows, and of the rows behind, too
static int64_t row_tiles(const Args& g, const Plan& p) { return (g.R / p.D + std::min<int64_t>(g.R, g.E + 1)) * cdiv(g.N, p.D) * p.parts; }

// y's or dx' tiles, and their ranges' sum
template <bool Y>
static int launch(const char* fn, Args g, const Plan& p, void* ws, int64_t ws_bytes, hipStream_t st) {
  const int64_t need = sums_bytes(p, g.R, g.N), n = row_tiles(g, p);
  if (ws_bytes < need || (need && (!ws || !aligned(ws, 16)))) return fail(NTLB_EINVAL, "%s: workspace of %lld bytes, %lld needed", fn, (long long)ws_bytes, (long long)need);
  if (n * 2 * p.D > MAX_THREADS) return fail(NTLB_EUNSUPPORTED, "%s: %lld tiles are too many", fn, (long long)n);
  g.parts = p.parts;
  g.sums = (float*)ws;
  g.lds = cdiv(g.N, 4) * 4;
  const dim3 grd((unsigned)n);
  if constexpr (Y) {
    if (p.D == 256) rows_kernel<256><<<grd, 512, 0, st>>>(g);
    else rows_kernel<128><<<grd, 256, 0, st>>>(g);
  } else {
    if (p.D == 256) inputs_kernel<256><<<grd, 512, 0, st>>>(g);
    else inputs_kernel<128><<<grd, 256, 0, st>>>(g);
  }
  if (int rc = check_launch(fn)) return rc;
  if (p.parts == 1) return NTLB_OK;
  join_kernel<<<(unsigned)cdiv(g.R * (g.lds / 4), 256), 256, 0, st>>>(g);
  return check_launch(fn);
}

}  // namespace grouped
}  // namespace ntlb

using namespace ntlb;

extern "C" int64_t ntlb_grouped_matmul_workspace_bytes(int64_t R, int64_t E, int64_t N, int64_t K, int dx) {
  if (R < 1 || E < 1 || N < 1 || K < 1) return 0;
  return dx ? grouped::sums_bytes(grouped::plan_of(R, E, K, N, false), R, K)
            : grouped::sums_bytes(grouped::plan_of(R, E, N, K, true), R, N);
}

extern "C" int ntlb_grouped_matmul(const uint16_t* x, int64_t ldx, const uint16_t* w, int64_t ldw, int64_t w_stride,
                                   const int32_t* offsets, int64_t R, int64_t E, int64_t N, int64_t K, uint16_t* y,
                                   int64_t ldy, void* workspace, int64_t ws_bytes, void* stream) {
  const char* fn = "ntlb_grouped_matmul";
  if (int rc = grouped::check(fn, R, E, N, K, offsets)) return rc;
  if (R == 0) return NTLB_OK;
  if (!grouped::fits(x, ldx, K)) return grouped::bad(fn, "x");
  if (!grouped::fits(w, ldw, K) || w_stride % 8 || w_stride < 0) return grouped::bad(fn, "w");
  if (!y || ldy < N) return fail(NTLB_EINVAL, "%s: bad y", fn);
  grouped::Args g{};
  g.a = (const uint8_t*)x; g.lda = ldx * 2; g.b = (const uint8_t*)w; g.ldb = ldw * 2; g.b_expert = w_stride * 2;
  g.offsets = offsets; g.R = R; g.E = (int)E; g.k = K; g.N = N; g.out = y; g.ldo = ldy;
  hipStream_t st = as_stream(stream);
  const grouped::Plan p = grouped::plan_of(R, E, N, K, true);
  if (!p.few) return grouped::launch<true>(fn, g, p, workspace, ws_bytes, st);
  grouped::few_kernel<<<(unsigned)grouped::few_blocks(E, N), 64 * grouped::FEW_WAVES, 0, st>>>(g, (int)cdiv(N, 16));
  return check_launch(fn);
}

extern "C" int ntlb_grouped_matmul_dx(const uint16_t* dy, int64_t lddy, const uint16_t* w, int64_t ldw, int64_t w_stride,
                                      const int32_t* offsets, int64_t R, int64_t E, int64_t N, int64_t K, uint16_t* dx,
                                      int64_t lddx, void* workspace, int64_t ws_bytes, void* stream) {
  const char* fn = "ntlb_grouped_matmul_dx";
  if (int rc = grouped::check(fn, R, E, N, K, offsets)) return rc;
  if (R == 0) return NTLB_OK;
  if (!grouped::fits(dy, lddy, N)) return grouped::bad(fn, "dy");
  if (!grouped::fits(w, ldw, K) || w_stride % 8 || w_stride < 0) return grouped::bad(fn, "w");
  if (!dx || lddx < K) return fail(NTLB_EINVAL, "%s: bad dx", fn);
  grouped::Args g{};
  g.a = (const uint8_t*)dy; g.lda = lddy * 2; g.b = (const uint8_t*)w; g.ldb = ldw * 2; g.b_expert = w_stride * 2;
  g.offsets = offsets; g.R = R; g.E = (int)E; g.k = N; g.N = K; g.out = dx; g.ldo = lddx;
  return grouped::launch<false>(fn, g, grouped::plan_of(R, E, K, N, false), workspace, ws_bytes, as_stream(stream));
}

extern "C" int ntlb_grouped_matmul_dw(const uint16_t* dy, int64_t lddy, const uint16_t* x, int64_t ldx,
                                      const int32_t* offsets, int64_t R, int64_t E, int64_t N, int64_t K, uint16_t* dw,
                                      void* stream) {
  const char* fn = "ntlb_grouped_matmul_dw";
  if (int rc = grouped::check(fn, R, E, N, K, offsets)) return rc;
  if (!dw) return fail(NTLB_EINVAL, "%s: bad dw", fn);
  if (R > 0 && !grouped::fits(dy, lddy, N)) return grouped::bad(fn, "dy");
  if (R > 0 && !grouped::fits(x, ldx, K)) return grouped::bad(fn, "x");
  grouped::Args g{};
  g.a = (const uint8_t*)dy; g.lda = lddy * 2; g.b = (const uint8_t*)x; g.ldb = ldx * 2;
  g.offsets = offsets; g.R = R; g.E = (int)E; g.M = N; g.N = K; g.out = dw; g.ldo = K;
  const int D = N > 128 && K > 128 && E * cdiv(N, 256) * cdiv(K, 256) >= split_device_cus() ? 256 : 128;
  const int64_t n = grouped::ordered_grid(E * cdiv(N, D) * cdiv(K, D));
  if (n > ((int64_t)1 << 30)) return fail(NTLB_EUNSUPPORTED, "%s: %lld tiles are too many", fn, (long long)n);  // counted in 32 bits
  hipStream_t st = as_stream(stream);
  const unsigned wgs = (unsigned)std::min<int64_t>(n, cdiv(split_device_cus(), 8) * 8 * (D == 256 ? 1 : 2));
  if (D == 256) grouped::weight_kernel<256><<<wgs, 512, 0, st>>>(g, (int)n);
  else grouped::weight_kernel<128><<<wgs, 256, 0, st>>>(g, (int)n);
  return check_launch(fn);
}

extern "C" int ntlb_kept_rows(const uint16_t* x, int64_t ldx, int64_t R, int64_t K, uint8_t* kept, uint8_t* kept_exp,
                              void* stream) {
  const char* fn = "ntlb_kept_rows";
  clear_error();
  if (R < 0 || K < 1 || K > grouped::MAX_PITCH) return fail(NTLB_EINVAL, "%s: bad shape %lld x %lld", fn, (long long)R, (long long)K);
  if (R == 0) return NTLB_OK;
  if (!grouped::fits(x, ldx, K)) return grouped::bad(fn, "x");
  if (!kept || !aligned(kept, 16) || !kept_exp) return fail(NTLB_EINVAL, "%s: bad kept codes", fn);
  const int64_t NT = cdiv(K, KEPT_TILE);
  return row_pieces(R, NT, [&](int64_t r, int64_t n) {
    grouped::Keep g{(const uint8_t*)(x + r * ldx), ldx * 2, n * NT, (int)K, TileRows(NT), kept + r * NT * KEPT_TILE, kept_exp + r * NT};
    grouped::keep_kernel<<<(unsigned)cdiv(g.tiles, 16), 256, 0, as_stream(stream)>>>(g);
    return check_launch(fn);
  });
}

extern "C" int ntlb_kept_values(const uint8_t* kept, const uint8_t* kept_exp, int64_t R, int64_t K, uint16_t* out,
                                int64_t ldo, void* stream) {
  const char* fn = "ntlb_kept_values";
  clear_error();
  if (R < 0 || K < 1 || K > grouped::MAX_PITCH) return fail(NTLB_EINVAL, "%s: bad shape %lld x %lld", fn, (long long)R, (long long)K);
  if (R == 0) return NTLB_OK;
  if (!grouped::fits(out, ldo, K)) return grouped::bad(fn, "out");
  if (!kept || !aligned(kept, 16) || !kept_exp) return fail(NTLB_EINVAL, "%s: bad kept codes", fn);
  const int64_t NT = cdiv(K, KEPT_TILE);
  return row_pieces(R, NT, [&](int64_t r, int64_t n) {
    grouped::Keep g{nullptr, 0, n * NT, (int)K, TileRows(NT), const_cast<uint8_t*>(kept) + r * NT * KEPT_TILE, const_cast<uint8_t*>(kept_exp) + r * NT};
    grouped::values_kernel<<<(unsigned)cdiv(g.tiles, 16), 256, 0, as_stream(stream)>>>(g, (uint8_t*)(out + r * ldo), ldo * 2);
    return check_launch(fn);
  });
}
