// Softmax cross entropy of a linear head, without keeping the logits:
//   z = X W^T [T, V],  loss_t = logsumexp(z_t) - z_t[y_t]
//   dz_t = u_t (softmax(z_t) - onehot(y_t)),  dX = dz W,  dW = dz^T X
// (u_t: the gradient that comes in for loss_t)
// X bf16 [T, H], W bf16 [V, H]; products of bf16 values are exact in fp32 and
// summed in fp32 on the matrix cores; statistics, exponentials and losses are
// fp32.
//
// Matrix-core bound: 2 T V H operations forward, 4 T V H for the gradients and
// 2 T V H more to form the logits again.  That saves memory, T x V values of 32 bits
// (2.1 GB at 4096 x 131072) from the forward to the backward, and costs time: at the
// rates below a logit takes 2 H / 1.33e15 s to form, one written and read 8 / 5.3e12
// s, which is as much at a width of 1000, half at 2048 and a seventh at 7168 (0.8 ms
// for 5.5 at 4096 x 131072).  Positions that are ignored are left out
// before the products: X's live rows are gathered (and padded to whole 64-column
// steps) into X', so masked positions cost nothing, hold no part in any sum and
// cannot pass on a NaN.  How many are live is known to the device only: tiles
// past them exit, and the contraction of dW ends there.
//
// Forward: 256x256 (or 128x128) tiles of z; the epilogue reduces a tile's row to
// its largest z and the sum of exp(z - largest) and picks the label's logit, and a
// second kernel joins the tiles' pairs of a row, in 64 bits.  Backward, per piece of the vocabulary (the piece's
// dz, bf16, is the only matrix of logits' size that exists): dz from the logits
// formed again, dX += dz W (fp32, in `slices` ranges of the piece where the tiles
// alone would leave compute units idle), dW = dz^T X'.  dz is rounded to bf16
// once, as the operand of its two products, which costs about what the
// rounding of the outputs does as long as the roundings are independent.  The
// large values, p - 1 at the labels, would not be if they held the factor 1 / n of
// a mean: every one of them would be off by the same part, and so the whole
// gradient.  So dz is formed without the rows' common factor (for u of its own
// for each row, their largest magnitude), which the outputs take in fp32.  Up to 64
// rows dz is two bf16 values, at no product's cost.
//
// Measured, 3891 live rows of 4096, 7168 wide, 131072 words in two pieces: logits
// and their sums 5.48 to 5.52 ms (1.33 PFLOP/s), per piece logits and dz 2.79 to
// 2.80 (1.31), dX and dW 5.45 (1.34; in launches of their own 2.83 and 2.74); the
// library's product of the forward's operands runs at 1.49.  All are held by the
// chip's power: under such a load its clock falls from 2.4 to about 1.8 GHz.  With
// all copies from the nearest cache (the same step again and again) the four would
// take 5.24, 2.63, 2.48 and 2.45 ms: the wait for memory is what is left of dX and
// dW.  Four waves of 128 x 128 instead of eight of 128 x 64 read less of LDS, but
// one wave a SIMD has no other to hide its waits: 5.79, 2.86, 3.20 and 3.05.  16
// rows of 4096 x 131072 words: 175 to 187 us, 5.7 to 6.1 TB/s of weights.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "ntlb_bf16_tile.h"
#include "ntlb_device.h"
#include "ntlb_gemm_bf16.h"
#include "ntlb_host.h"
#include "ntlb_splitk.h"

namespace ntlb {
namespace xent {

using namespace tile;

constexpr float LOG2E = 1.44269502e+00f;

constexpr int EPI_LSE = 0, EPI_DZ = 1, EPI_ACC = 2, EPI_STORE = 3;

// The gradient that comes in: du[0] for all rows, over the number of live rows
// if mean; or, `most` given, du[t] for row t, their common factor most[0], which is
// 0 only if all are.  With no live row nothing comes in: du is not read (of an empty
// batch it may be NULL).
struct Up {
  const float* du;
  const float* most;
  int mean;
  __device__ float common(int live) const {
    return live == 0 ? 0.f : most ? most[0] : du[0] * (mean ? 1.0f / (float)live : 1.0f);
  }
  __device__ float rest(int row, float c) const { return !most ? 1.0f : c == 0.f ? 0.f : du[row] / c; }
};

struct Args {
  Mat a, b;
  int64_t M, N;
  const int32_t* live;  // device: the rows in use (of A for LSE / DZ / ACC, of the contraction for STORE)
  int slices;           // ACC, and LSE and DZ by small tiles: ranges of the contraction
  int base;             // LSE, DZ by small tiles: the tiles before this one are not divided
  float4* part_z;       // LSE, DZ with ranges: their sums, [tile - base][range][16 v4f][thread]
  uint32_t* count;      // ... of each divided tile, how many are there (0 before and after)
  int group_m;          // raster: row tiles side by side
  // LSE
  float2* part;         // [column tiles][ldp] (largest, sum)
  int64_t ldp;
  float* zl;            // [M] the label's logit
  const int32_t* y;     // labels of the live rows, < 0: none
  int64_t v0;           // first column's place in the vocabulary
  // DZ
  const float2* stat;   // [M] logsumexp times log2(e): fp32 and the rest
  const int32_t* rows;
  Up up;
  int half;             // DZ: the row that the rest of row 0's values goes to, or 0
  const int32_t* n;     // STORE: the number of live rows
  // outputs
  void* out;            // DZ: bf16, ACC: fp32 [slices][..], STORE: bf16
  int64_t ldo;          // elements; DZ: of a block
  int64_t cols;         // DZ: columns to store, whole blocks
  int64_t slice;        // elements of a slice
  int add;              // ACC: add to what is there
};

// A set of logits z: the largest of them and the sum of exp(z - largest).  A row
// keeps both to the end (and its logsumexp in two parts): rounded to one number, it
// would be off by a unit of itself, and with it a confident row's loss and p - 1,
// which are far smaller.  The largest itself adds exactly 1.
template <typename T>
__device__ __forceinline__ void merge(float& ax, T& ay, float bx, T by) {
  const float hi = fmaxf(ax, bx), ref = hi == -__builtin_inff() ? 0.f : hi;
  ay = ay * (T)__builtin_amdgcn_exp2f((ax - ref) * LOG2E) + by * (T)__builtin_amdgcn_exp2f((bx - ref) * LOG2E);
  ax = hi;
}

// Where the small tiles of z are too few for the chip, a tile's contraction is
// divided among `slices` workgroups: each leaves its sums, and the last to arrive
// adds all of them, in the ranges' order, and goes on.  Nobody waits.  Only groups
// of 16 rows that hold live ones travel.
template <int MT>
__device__ __forceinline__ bool exchange(v4f (&acc)[MT][4], float4* part, uint32_t* count, int slices, int sl, int groups, int tid) {
  constexpr int THREADS = 256, PER = MT * 4 * THREADS;
  __shared__ int last;
  part += tid;
#pragma unroll
  for (int tm = 0; tm < MT; ++tm)
    if (tm < groups)
#pragma unroll
      for (int tn = 0; tn < 4; ++tn)
        part[sl * PER + (tm * 4 + tn) * THREADS] = make_float4(acc[tm][tn][0], acc[tm][tn][1], acc[tm][tn][2], acc[tm][tn][3]);
  __syncthreads();  // all waves' stores come before it, and what comes before a release it carries along
  if (tid == 0) last = __hip_atomic_fetch_add(count, 1u, __ATOMIC_RELEASE, __HIP_MEMORY_SCOPE_AGENT) == (uint32_t)(slices - 1);
  __syncthreads();
  if (!last) return false;
  if (tid == 0) __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
  __syncthreads();
#pragma unroll
  for (int tm = 0; tm < MT; ++tm)
    if (tm < groups) {
#pragma unroll
      for (int tn = 0; tn < 4; ++tn) acc[tm][tn] = (v4f){0.f, 0.f, 0.f, 0.f};
      for (int c0 = 0; c0 < slices; c0 += 4) {
        float4 v[4][4];
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int tn = 0; tn < 4; ++tn) v[c][tn] = part[min(c0 + c, slices - 1) * PER + (tm * 4 + tn) * THREADS];
#pragma unroll
        for (int c = 0; c < 4; ++c)
          if (c0 + c < slices)
#pragma unroll
            for (int tn = 0; tn < 4; ++tn) acc[tm][tn] += (v4f){v[c][tn].x, v[c][tn].y, v[c][tn].z, v[c][tn].w};
      }
    }
  if (tid == 0) atomicExch(count, 0u);  // ready for the next product
  return true;
}

// One output tile of D x D, the pid-th of its product: 256, eight waves of 128 x
// 64, one workgroup a compute unit; 128, four waves of 64 x 64, two workgroups.
// la0 ... lb1: two stages of both operands, TILE bytes each.
template <int D, bool TA, bool TB, int EPI>
__device__ __forceinline__ void head_tile(Args g, int pid, uint8_t* la0, uint8_t* lb0, uint8_t* la1, uint8_t* lb1) {
  constexpr int TM = D, TN = D, TILE = D * ROWB, WAVES_N = D / 64, MT = D / 32;
  constexpr bool SPLIT = D == 128 && (EPI == EPI_LSE || EPI == EPI_DZ), RANGES = SPLIT || EPI == EPI_ACC;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WAVES_N, wn = wave % WAVES_N;
  const int live = __builtin_amdgcn_readfirstlane(g.live[0]);
  // tiles: each XCD walks a contiguous range of a raster of group_m row tiles
  const int num_n = (int)((g.N + TN - 1) / TN);
  const int num_m_all = (int)((g.M + TM - 1) / TM);
  const int num_m = EPI == EPI_STORE ? num_m_all : (live + TM - 1) / TM;
  int sl = 0, parts = EPI == EPI_ACC ? g.slices : 1;
  if constexpr (EPI == EPI_ACC) {
    const int tiles = num_m * num_n;
    if (pid >= tiles * g.slices) return;
    // the ranges of a tile lie on different XCDs' shares, side by side in k
    const int nwg = tiles * g.slices, xcd = pid & 7, per = nwg >> 3, extra = nwg & 7;
    const int q = xcd * per + min(xcd, extra) + (pid >> 3);
    sl = q / tiles;
    pid = q - sl * tiles;
  } else {
    const int tiles = num_m * num_n, base = SPLIT ? min(g.base, tiles) : tiles;
    const bool divided = SPLIT && pid >= base;
    if (divided) parts = g.slices;
    const int first = divided ? base : 0, n = divided ? (tiles - base) * parts : base;
    pid -= first;
    if (pid >= n) return;
    const int xcd = pid & 7, per = n >> 3, extra = n & 7;
    pid = xcd * per + min(xcd, extra) + (pid >> 3);
    if (divided) {
      sl = pid % parts;
      pid /= parts;
    }
    pid += first;
  }
  const int group = pid / (g.group_m * num_n), first_m = group * g.group_m;
  const int gsize = min(num_m - first_m, g.group_m), in_group = pid - group * g.group_m * num_n;
  const int64_t m0 = (int64_t)(first_m + in_group % gsize) * TM, n0 = (int64_t)(in_group / gsize) * TN;
  if constexpr (EPI == EPI_STORE) {
    g.a.k = live;
    g.b.k = live;
  } else {
    g.M = live;
    g.a.rows = live;
  }
  const int nk = max(1, (int)((g.a.k + KSTEP - 1) / KSTEP));
  const int kb0 = RANGES ? (int)((int64_t)sl * nk / parts) : 0;
  const int kb1 = RANGES ? (int)((int64_t)(sl + 1) * nk / parts) : nk;

  // A is X' or dz, B the weight or (with A transposed) X'
  typename std::conditional<TA, BlockTrCopy<D>, BlockRowCopy<D>>::type ca;
  typename std::conditional<TA, BlockTrCopy<D>, typename std::conditional<TB, TrCopy<D>, RowCopy<D>>::type>::type cb;
  ca.init(g.a, m0, wave, lane);
  cb.init(g.b, n0, wave, lane);
  v4f acc[MT][4];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = (v4f){0.f, 0.f, 0.f, 0.f};
  multiply<D, TA, TB>(ca, cb, kb0, kb1, acc, wm, wn, wave, lane, la0, lb0, la1, lb1);
  if constexpr (SPLIT) {
    const int groups = min((int)(g.M - m0 - wm * 16 * MT + 15) / 16, MT);
    const int64_t tile = pid - g.base;
    if (parts > 1 && !exchange<MT>(acc, g.part_z + tile * parts * (MT * 4 * 256), g.count + tile, parts, sl, groups, tid)) return;
  }
  // a wave's 16 KiB of the stages for its output rows
  constexpr int PER = TILE / 16384;
  uint8_t* stage = (wave / PER == 0 ? la0 : wave / PER == 1 ? lb0 : wave / PER == 2 ? la1 : lb1) + (wave % PER) * 16384;
  // lane: rows m0 + wm*16*MT + tm*16 + lane%16, columns n0 + wn*64 + tn*16 + 4*(lane/16) + r
  const int64_t mw = m0 + wm * 16 * MT + (lane & 15), nw = n0 + wn * 64 + (lane >> 4) * 4;
  // Few waves hold columns past N or a row's label: what either asks of each value
  // stands behind a test of the whole wave
  const int cols = (int)min<int64_t>(64, g.N - (n0 + wn * 64)) - (lane >> 4) * 4;  // of N, from the lane's first
  const bool edge = g.N - (n0 + wn * 64) < 64;
  if constexpr (EPI == EPI_LSE) {
    float2* red = reinterpret_cast<float2*>(la0);  // [WAVES_N][D]
    int lab[MT];  // the label's column, from the lane's first
#pragma unroll
    for (int tm = 0; tm < MT; ++tm) lab[tm] = mw + tm * 16 < g.M ? (int)(g.y[mw + tm * 16] - nw) : -1;
#pragma unroll
    for (int tm = 0; tm < MT; ++tm) {
      if (__any(lab[tm] >= 0 && lab[tm] < 64)) {
#pragma unroll
        for (int tn = 0; tn < 4; ++tn)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (lab[tm] == tn * 16 + r) g.zl[mw + tm * 16] = acc[tm][tn][r];
      }
      if (edge) {
#pragma unroll
        for (int tn = 0; tn < 4; ++tn)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (tn * 16 + r >= cols) acc[tm][tn][r] = -__builtin_inff();
      }
      float mx = -__builtin_inff();
#pragma unroll
      for (int tn = 0; tn < 4; ++tn)
#pragma unroll
        for (int r = 0; r < 4; ++r) mx = fmaxf(mx, acc[tm][tn][r]);
      mx = fmaxf(mx, __shfl_xor(mx, 16));
      mx = fmaxf(mx, __shfl_xor(mx, 32));
      const float ref = mx == -__builtin_inff() ? 0.f : mx;
      float s = 0.f;
#pragma unroll
      for (int tn = 0; tn < 4; ++tn)
#pragma unroll
        for (int r = 0; r < 4; ++r) s += __builtin_amdgcn_exp2f((acc[tm][tn][r] - ref) * LOG2E);
      s += __shfl_xor(s, 16);
      s += __shfl_xor(s, 32);
      if (lane < 16) red[wn * D + wm * 16 * MT + tm * 16 + lane] = make_float2(mx, s);
    }
    __syncthreads();
    if (tid < D && m0 + tid < g.M) {
      float2 t = red[tid];
#pragma unroll
      for (int i = 1; i < WAVES_N; ++i) merge(t.x, t.y, red[i * D + tid].x, red[i * D + tid].y);
      g.part[(n0 / TN) * g.ldp + m0 + tid] = t;
    }
  } else if constexpr (EPI == EPI_DZ) {
    // p = 2^(z log2(e) - hi) 2^-lo, whose second factor the row's u takes: one multiply-add
    // a value (two with the largest logit taken off first: 31.1 us, this 30.2, at 1003 x 1000 x 10007)
    const float c = g.up.common(live);
    float hi[MT], lo[MT], u[MT];
    int lab[MT];
    // dz's rows up to the next 64 are read, zero past the live ones; so are whole
    // blocks, zero past the piece
#pragma unroll
    for (int tm = 0; tm < MT; ++tm) {
      const bool on = mw + tm * 16 < g.M;
      const int64_t m = on ? mw + tm * 16 : 0;
      const float2 st = g.stat[m];
      hi[tm] = on ? st.x : __builtin_inff();
      lo[tm] = on ? st.y : 0.f;
      u[tm] = on ? g.up.rest(g.rows[m], c) * __builtin_amdgcn_exp2f(-lo[tm]) : 0.f;
      lab[tm] = on ? (int)(g.y[m] - g.v0 - nw) : -1;
    }
#pragma unroll
    for (int tm = 0; tm < MT; ++tm) {
#pragma unroll
      for (int tn = 0; tn < 4; ++tn)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          acc[tm][tn][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(acc[tm][tn][r], LOG2E, -hi[tm]));
      if (__any(lab[tm] >= 0 && lab[tm] < 64)) {
        const float one = __builtin_amdgcn_exp2f(lo[tm]);  // 1, over the factor that u holds
#pragma unroll
        for (int tn = 0; tn < 4; ++tn)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (lab[tm] == tn * 16 + r) acc[tm][tn][r] -= one;
      }
      if (edge) {
#pragma unroll
        for (int tn = 0; tn < 4; ++tn)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (tn * 16 + r >= cols) acc[tm][tn][r] = 0.f;
      }
      // rows past the live ones: zero times a word's infinity is NaN, which no factor
      // of 0 takes out
      const bool past = mw + tm * 16 >= g.M;
      if (__any(past)) {
#pragma unroll
        for (int tn = 0; tn < 4; ++tn)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (past) acc[tm][tn][r] = 0.f;
      }
    }
    const int64_t block = n0 / 64 + wn;
    const bool rest = D == 128 && g.half;  // (up to 64 rows always take the small tiles)
    const int64_t end = rest ? g.half : (g.M + 63) / 64 * 64;
    uint16_t* o = (uint16_t*)g.out + block * g.ldo;
    store_bf16<MT, false>(stage, lane, m0 + wm * 16 * MT, 0, end, g.cols - block * 64, o, 64, [&](int tm, int tn, float (&v)[4]) {
#pragma unroll
      for (int r = 0; r < 4; ++r) v[r] = acc[tm][tn][r] * u[tm];
    });
    if (rest)
      store_bf16<MT, false>(stage, lane, m0 + wm * 16 * MT, 0, end, g.cols - block * 64, o + g.half * 64, 64, [&](int tm, int tn, float (&v)[4]) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float w = acc[tm][tn][r] * u[tm], hi = (float)(__bf16)w;
          v[r] = __builtin_fabsf(hi) < __builtin_inff() ? w - hi : 0.f;  // what is no number is in the first half
        }
      });
  } else if constexpr (EPI == EPI_ACC) {
    float* o = (float*)g.out + sl * g.slice;
#pragma unroll
    for (int tm = 0; tm < MT; ++tm) {
      const int64_t m = mw + tm * 16;
      if (m >= g.M) continue;
#pragma unroll
      for (int tn = 0; tn < 4; ++tn) {
        const int64_t n = nw + tn * 16;
        if (n >= g.ldo) continue;  // the pitch is a multiple of four
        v4f* q = reinterpret_cast<v4f*>(o + m * g.ldo + n);
        *q = g.add ? *q + acc[tm][tn] : acc[tm][tn];
      }
    }
  } else {
    const float c = g.up.common(g.n[0]);
    store_bf16<MT, true>(stage, lane, m0 + wm * 16 * MT, n0 + wn * 64, g.M, g.N, (uint16_t*)g.out, g.ldo, [&](int tm, int tn, float (&v)[4]) {
#pragma unroll
      for (int r = 0; r < 4; ++r) v[r] = acc[tm][tn][r] * c;
    });
  }
}

template <int D, bool TA, bool TB, int EPI>
__global__ void __launch_bounds__(2 * D, D == 256 ? 1 : 2) head_kernel(Args g) {
  NTLB_TILE_STAGES(D);
  head_tile<D, TA, TB, EPI>(g, (int)blockIdx.x, la0, lb0, la1, lb1);
}

// dX's tiles (the first nx, a multiple of 8, workgroups) and dW's in one grid
template <int D>
__global__ void __launch_bounds__(2 * D, D == 256 ? 1 : 2) gradients_kernel(Args x, Args w, int nx) {
  NTLB_TILE_STAGES(D);
  const int pid = (int)blockIdx.x;
  if (pid < nx)
    head_tile<D, false, true, EPI_ACC>(x, pid, la0, lb0, la1, lb1);
  else
    head_tile<D, true, true, EPI_STORE>(w, pid - nx, la0, lb0, la1, lb1);
}

// ---------------------------------------------------------------------------
// the live rows: pos[t] = place of row t among them (-1: ignored), rows[i] and
// y[i] (-1: not a word) of the i-th, live[0] how many, live[1] the rows of dz.  One workgroup; up to HERE
// rows each of gather_kernel's counts for itself (16 rows: 5.0 us, with this
// launch 4.7 + 4.9; 1003 rows 5.0 and 2.4 + 3.6).
// ---------------------------------------------------------------------------
constexpr int SCAN = 1024, HERE = 1024, COUNTERS = 1024;
struct Targets {
  const void* p;
  int wide;
  int64_t T, V, ignore;
  __device__ int64_t at(int64_t t) const { return t >= T ? ignore : wide ? ((const int64_t*)p)[t] : (int64_t)((const int32_t*)p)[t]; }
  __device__ int32_t word(int64_t v) const { return v >= 0 && v < V ? (int32_t)v : -1; }
};
struct Live {
  int32_t *pos, *rows, *y, *live;
};

__global__ void __launch_bounds__(SCAN) scan_kernel(Targets tg, Live o) {
  __shared__ int wsum[SCAN / 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int base = 0;
  for (int64_t t0 = 0; t0 < tg.T; t0 += SCAN) {
    const int64_t t = t0 + tid, v = tg.at(t);
    const bool on = v != tg.ignore;
    const uint64_t b = __ballot(on);
    if (lane == 0) wsum[wave] = __popcll(b);
    __syncthreads();
    int before = base, all = 0;
#pragma unroll
    for (int w = 0; w < SCAN / 64; ++w) {
      before += w < wave ? wsum[w] : 0;
      all += wsum[w];
    }
    const int at = before + __popcll(b & ((1ull << lane) - 1));
    if (t < tg.T) o.pos[t] = on ? at : -1;
    if (on) {
      o.rows[at] = (int32_t)t;
      o.y[at] = tg.word(v);
    }
    base += all;
    __syncthreads();
  }
  if (tid == 0) o.live[0] = o.live[1] = base;
}

// eight values of a row of H from column c, zero past H; rows begin anywhere
__device__ __forceinline__ uint4 piece_of(const uint16_t* row, int64_t c, int64_t H) {
  if (c + 8 <= H) {
    const u32x4_2 v = *reinterpret_cast<const u32x4_2*>(row + c);
    return make_uint4(v[0], v[1], v[2], v[3]);
  }
  uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (c + i < H) w[i >> 1] |= (uint32_t)row[c + i] << (16 * (i & 1));
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// rows of any pitch into rows of whole 16-byte pieces, zero past H: HBM-bound
// (42508 rows of 345: 14.3 us, 4.1 TB/s).  A workgroup takes `per` rows.
__global__ void __launch_bounds__(256) pad_kernel(const uint16_t* x, int64_t ldx, int64_t R, int64_t H, uint16_t* out,
                                                  int64_t ldo, int per) {
  const int pieces = (int)(ldo / 8);
  const int64_t r0 = (int64_t)blockIdx.x * per;
  const int n = (int)min<int64_t>(per, R - r0) * pieces;
#pragma unroll 4
  for (int i = threadIdx.x; i < n; i += 256) {
    const int r = i / pieces, c = i - r * pieces;
    reinterpret_cast<uint4*>(out + (r0 + r) * ldo)[c] = piece_of(x + (r0 + r) * ldx, (int64_t)c * 8, H);
  }
}

// X': 16-byte pieces of the live rows of X into blocks of 64 columns, zero past
// H and, by the last 63 workgroups, in the rows up to the next 64; with `half`, twice,
// `half` rows on again.  Also what the other kernels expect
// set: zl (NaN until a tile finds the label), a zero loss for the ignored rows and
// the counters of the ranges.
template <bool COUNT>
__global__ void __launch_bounds__(256) gather_kernel(const uint16_t* x, int64_t ldx, int64_t H, Targets tg,
                                                     Live o, uint16_t* xp, int64_t hk, int64_t block, float* zl, float* loss,
                                                     uint32_t* count, int half) {
  const int64_t t = blockIdx.x;
  if (t == 0 && count)
    for (int i = threadIdx.x; i < COUNTERS; i += 256) count[i] = 0;
  const bool past = t >= tg.T;
  int at, n;
  if constexpr (COUNT) {
    __shared__ int2 red[4];
    const int64_t v = tg.at(t);
    int2 c = make_int2(0, 0);
    for (int i = threadIdx.x; i < tg.T; i += 256) {
      const bool on = tg.at(i) != tg.ignore;
      c.x += on && i < t;
      c.y += on;
    }
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      c.x += __shfl_xor(c.x, d);
      c.y += __shfl_xor(c.y, d);
    }
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = c;
    __syncthreads();
    at = red[0].x + red[1].x + red[2].x + red[3].x;
    n = red[0].y + red[1].y + red[2].y + red[3].y;
    const bool on = v != tg.ignore;
    if (threadIdx.x == 0) {
      if (!past) o.pos[t] = on ? at : -1;
      if (on) {
        o.rows[at] = (int32_t)t;
        o.y[at] = tg.word(v);
      }
      if (t == 0) {
        o.live[0] = n;
        o.live[1] = half && n ? half + n : n;
      }
    }
    if (!on) at = -1;
  } else {
    n = o.live[0];
    at = past ? -1 : o.pos[t];
  }
  if (past) at = n + (int)(t - tg.T);
  if (past && at >= (half ? half : (n + 63) / 64 * 64)) return;
  if (at < 0) {
    if (threadIdx.x == 0 && loss) loss[t] = 0.f;
    return;
  }
  if (threadIdx.x == 0 && !past) zl[at] = __builtin_nanf("");
  const uint16_t* src = x + t * ldx;
  for (int64_t c = threadIdx.x; c < hk / 8; c += blockDim.x) {
    const uint4 v = past ? make_uint4(0, 0, 0, 0) : piece_of(src, c * 8, H);
    uint4* o = reinterpret_cast<uint4*>(xp + (c >> 3) * block + (int64_t)at * 64 + (c & 7) * 8);
    o[0] = v;
    if (half) o[half * 8] = v;
  }
}

// The live rows' pairs joined, and their losses, by R rows and Q walkers; TOTAL: of
// all rows, in one workgroup, and then their sum or mean in a fixed order (0 where
// none is live).  Sums are 64 bits here: of a confident row's, each addition to the
// 1 of its largest logit would otherwise round what the others add.
template <int R, int Q, bool TOTAL>
__global__ void __launch_bounds__(R * Q) join_kernel(const float2* part, int64_t ldp, int64_t parts, const float* zl,
                                                     const int32_t* rows, const int32_t* live, int mean, float2* stat,
                                                     float* each, float* loss) {
  constexpr int WAVES = R * Q / 64;
  __shared__ float red_top[WAVES][R];
  __shared__ double red_sum[WAVES][R];
  __shared__ float losses[R];
  const int tid = threadIdx.x, r = tid % R, q = tid / R, n = live[0];
  const int64_t m = (int64_t)blockIdx.x * R + r;
  const bool on = m < n;
  float top = -__builtin_inff();
  double sum = 0.0;
  if (on)
#pragma unroll 4
    for (int64_t i = q; i < parts; i += Q) merge<double>(top, sum, part[i * ldp + m].x, part[i * ldp + m].y);
#pragma unroll
  for (int d = R; d < 64; d *= 2) merge<double>(top, sum, __shfl_xor(top, d), __shfl_xor(sum, d));
  if ((tid & 63) < R) {
    red_top[tid >> 6][r] = top;
    red_sum[tid >> 6][r] = sum;
  }
  __syncthreads();
  if (q == 0 && on) {
#pragma unroll
    for (int i = 1; i < WAVES; ++i) merge<double>(top, sum, red_top[i][r], red_sum[i][r]);
    const float z = zl[m], log_sum = log1pf((float)(sum - 1.0)), l = log_sum + (top - z);
    const double all = (double)top * LOG2E + (double)log_sum * 1.4426950408889634;
    const float hi = (float)all;
    stat[m] = z != z ? make_float2(z, z) : make_float2(hi, (float)(all - hi));  // no such word, or its logit is NaN: so is all of the row
    if constexpr (TOTAL) {
      losses[r] = l;
    } else {
      each[m] = l;
      if (loss) loss[rows[m]] = l;
    }
  }
  if constexpr (TOTAL) {
    __syncthreads();
    if (tid < 64) {
      float s = tid < n ? losses[tid % R] : 0.f;
#pragma unroll
      for (int d = 1; d < 64; d *= 2) s += __shfl_xor(s, d);
      if (tid == 0) loss[0] = mean ? s / (float)max(n, 1) : s;
    }
  }
}

// the sum or mean of more rows' losses, in a fixed order; 0 where none is live.  A
// launch of its own, 2 us: the join's last workgroup cannot know that it is the
// last without a fence in each, 15 us for 4096 rows.
__global__ void __launch_bounds__(1024) total_kernel(const float* each, const int32_t* live, int mean, float* loss) {
  __shared__ float red[16];
  const int n = live[0];
  float s = 0.f;
  for (int i = threadIdx.x; i < n; i += 1024) s += each[i];
#pragma unroll
  for (int d = 1; d < 64; d *= 2) s += __shfl_xor(s, d);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    float t = 0.f;
    for (int i = 0; i < 16; ++i) t += red[i];
    loss[0] = mean ? t / (float)max(n, 1) : t;
  }
}

// the largest finite |du| of the live rows, if `most` is given (1 where the finite ones
// are 0 but others are not finite: those have to reach dz), and the counters of the
// ranges cleared, if there are any
__global__ void __launch_bounds__(1024) most_kernel(const float* du, const int32_t* rows, const int32_t* live, float* most,
                                                    uint32_t* count) {
  __shared__ uint32_t red[16];
  if (count) count[threadIdx.x] = 0;
  if (!most) return;
  uint32_t m = 0;
  int wild = 0;
  for (int i = threadIdx.x; i < live[0]; i += 1024) {
    const uint32_t a = abs_bits(du[rows[i]]);
    m = a < 0x7F800000u ? max(m, a) : m;
    wild |= a >= 0x7F800000u;
  }
  m = wave_max_u32(m);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = m;
  wild = __syncthreads_or(wild);
  if (threadIdx.x == 0) {
    for (int i = 1; i < 16; ++i) m = max(m, red[i]);
    most[0] = m == 0 && wild ? 1.0f : __uint_as_float(m);
  }
}

// dX rows: the slices summed in order, bf16; zero for the ignored rows
__global__ void __launch_bounds__(256) scatter_kernel(const float* acc, int64_t ldp, int64_t slice, int slices, int half, Up up,
                                                      const int32_t* live, const int32_t* pos, int64_t H, uint16_t* dx,
                                                      int64_t ldx) {
  const int64_t t = blockIdx.x;
  const int at = pos[t];
  const float f = up.common(live[0]);
  for (int64_t c = (int64_t)threadIdx.x * 4; c < H; c += blockDim.x * 4) {
    v4f v = {0.f, 0.f, 0.f, 0.f};
    if (at >= 0) {
#pragma unroll 4
      for (int s = 0; s < slices; ++s) v += *reinterpret_cast<const v4f*>(acc + s * slice + (int64_t)at * ldp + c);
      if (half)
#pragma unroll 4
        for (int s = 0; s < slices; ++s) v += *reinterpret_cast<const v4f*>(acc + s * slice + (int64_t)(half + at) * ldp + c);
      v *= f;
    }
    uint16_t* o = dx + t * ldx + c;
    if (c + 4 <= H) {
      *reinterpret_cast<u32x2_2*>(o) = (u32x2_2){pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3])};
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (c + i < H) o[i] = f32_to_bf16_bits(v[i]);
    }
  }
}

// Up to 64 rows, whose tiles and steps have room for it, dz's rounding to bf16 is
// not left out: row `half` + i holds what row i's values lack, beside X' row i
// again, and both products sum the two.  (Of few values the gradients would
// otherwise be off by up to 1.9 times their own rounding; of many it is 1.4 times.)
static int half_of(int64_t T) { return T <= 32 ? 32 : T <= 64 ? 64 : 0; }
// rows of dz as dX's product has them
static int64_t dz_rows(int64_t T) { return half_of(T) + T; }
// elements of a block of X' or dz: 64 columns of the rows, whole 64 of them
static int64_t block_of(int64_t T) { return half_of(T) ? 2 * half_of(T) * 64 : cdiv(T, 64) * 64 * 64; }

// what the forward leaves for the backward
struct State {
  int64_t hk, block;  // columns of X', whole blocks; elements of one
  int64_t xp, pos, rows, y, stat, live, bytes;
};
static State state_of(int64_t T, int64_t H) {
  State s;
  s.hk = cdiv(H, 64) * 64;
  s.block = block_of(T);
  auto up = [](int64_t v) { return cdiv(v, 256) * 256; };
  s.xp = 0;
  s.pos = up(s.hk / 64 * s.block * 2);
  s.rows = s.pos + up(T * 4);
  s.y = s.rows + up(T * 4);
  s.stat = s.y + up(T * 4);
  s.live = s.stat + up(T * 8);
  s.bytes = s.live + 256;
  return s;
}

// relative times of a K step: 256 x 256 tiles, one 128 x 128 tile alone on a
// compute unit, two side by side.  A forward by 128 and by 256, us: 600 rows, 1000
// wide, 10007 words 22 and 30; 1003 rows 37 and 31; 1024 rows, 2048 wide, 32768
// words 145 and 118; 2048 rows, 1024 wide, 4096 words 20 and 30; 4096 rows, 4096
// wide, 16384 words 570 and 440.
constexpr double BIG_STEP = 1.0, LONE_STEP = 0.5, PAIR_STEP = 0.68;

// The tile of a product of M x N over `steps` K steps: the one whose rounds of
// workgroups (one or two to a compute unit) take less time
static int tile_for(int64_t M, int64_t N) {
  const int64_t cus = split_device_cus();
  const double big = (double)cdiv(cdiv(M, 256) * cdiv(N, 256), cus) * BIG_STEP;
  const int64_t small = cdiv(M, 128) * cdiv(N, 128);
  const double little = small <= cus ? LONE_STEP : (double)cdiv(small, 2 * cus) * PAIR_STEP;
  return little < big ? 128 : 256;
}

// The parts of a D-tiled product's contraction of `steps`: ranges that fill the
// last round of workgroups, at least 16 steps each; each range costs about four
// steps more (its fp32 tile read, written and summed)
static int ranges_for(int D, int64_t M, int64_t N, int64_t steps) {
  const int64_t tiles = cdiv(M, D) * cdiv(N, D), room = split_device_cus() * (D == 128 ? 2 : 1);
  int best_n = 1;
  double best = 1e30;
  for (int n = 1; n <= 16 && (n == 1 || steps / n >= 16); ++n) {
    const double t = (double)cdiv(tiles * n, room) * ((double)steps / n + 4);
    if (t < best * 0.98) {
      best = t;
      best_n = n;
    }
  }
  return best_n;
}

// one product
template <bool TA, bool TB, int EPI>
static void launch_head(int D, const Args& g, hipStream_t st) {
  const int64_t tiles = cdiv(g.M, D) * cdiv(g.N, D), base = std::min<int64_t>(g.base, tiles);
  const unsigned n = (unsigned)(EPI == EPI_ACC ? tiles * g.slices : EPI == EPI_STORE ? tiles : base + (tiles - base) * g.slices);
  if (D == 256)
    head_kernel<256, TA, TB, EPI><<<n, 512, 0, st>>>(g);
  else
    head_kernel<128, TA, TB, EPI><<<n, 256, 0, st>>>(g);
}

static void launch_pair(int D, const Args& x, const Args& w, hipStream_t st) {
  const int64_t nx = cdiv(cdiv(x.M, D) * cdiv(x.N, D) * x.slices, 8) * 8, nw = cdiv(w.M, D) * cdiv(w.N, D);
  if (D == 256)
    gradients_kernel<256><<<(unsigned)(nx + nw), 512, 0, st>>>(x, w, (int)nx);
  else
    gradients_kernel<128><<<(unsigned)(nx + nw), 256, 0, st>>>(x, w, (int)nx);
}

// dX's and dW's products in one launch, where the tiles of one fill the rounds
// that the other leaves open: the tile and dX's ranges of least time.  That of a
// step, of an item's beginning and end in steps, of the memory's part and of
// adding a range's values are fitted to 17 shapes by both tiles and 1 to 16 ranges
// (off by 12%; the choice is within 13% of the best, 4% on average).  us of the
// choice, and of two launches with tiles of their own: 1003 rows, 1000 wide,
// 10007 words 52 and 65; 64, 1024, 32000 34 and 48; 600, 768, 50257 98 and 145;
// 2048, 2048, 32768 430 and 466; 4096, 4096, 16384 819 and 870.
struct Pair {
  int tile, slices;
};
static Pair pair_of(int64_t T, int64_t H, int64_t cols) {
  const int64_t cus = split_device_cus();
  const double memory = 4.0 * (double)cols * (double)(H + T) / 5.14e6;  // W, dW; dz twice
  Pair best{256, 1};
  double t_best = 1e30;
  for (int D = 256; D >= 128; D /= 2) {
    const double step = D == 256 ? 1.33 : 0.83, over_x = D == 256 ? 10.6 : 5.1, over_w = D == 256 ? 3.9 : 5.1;
    const int64_t steps = cdiv(cols, KSTEP), nw = cdiv(cols, D) * cdiv(H, D);
    const double tw = step * ((double)cdiv(T, KSTEP) + over_w);
    for (int n = 1; n <= 16 && (n == 1 || steps / n >= 8); ++n) {
      const int64_t nx = cdiv(T, D) * cdiv(H, D) * n, room = cus * (D == 128 && nx + nw > cus ? 2 : 1), x = nx % room;
      const double tx = step * ((double)steps / n + over_x);
      // dX's whole rounds, then the rest of it beside dW
      double t = (double)(nx / room) * tx - 8;
      if (x == 0)
        t += (double)cdiv(nw, room) * tw;
      else if ((double)(room - x) * (int64_t)(tx / tw) >= (double)nw)
        t += tx;
      else
        t += std::max(tx, ((double)x * tx + (double)nw * tw) / (double)room + 0.5 * tw);
      const double a = t * t, b = memory * memory;
      t = std::sqrt(std::sqrt(a * a + b * b)) + 1.45e-6 * (double)T * (double)(H * n);
      if (t < t_best) {
        t_best = t;
        best = {D, n};
      }
    }
  }
  return best;
}

// The logits of `cols` words by small tiles: what the tiles past the last whole
// round (two workgroups to a compute unit) are divided into, if that leaves the
// chip room: the ranges of least time, in us 0.63 a step, and for more than one
// range 1.34 for each 128 rows of one, which the last to arrive reads, and 0.029
// (twice that with 128 rows) a workgroup, whose release all share: fitted to 14
// shapes by 1 to 16 ranges, off by 5%.  Forward by one range and by the choice: 3
// rows, 6413 wide, 265 words 71 us and 17; 5, 4208, 2904 48 and 19; 1, 7168, 4096
// 75 and 25; 1000, 7168, 1000 81 and 45; 16, 4096, 16384 46 and 34; 1000, 1024,
// 500, by one, 18 (by two 19); 54 tiles past the first 512: 4, 3600, 72400 145 and 113.
struct Ranges {
  int base = 0, n = 1;  // tiles that are not divided, ranges of the others
  int64_t tiles = 0;    // that are
  int64_t bytes() const { return n < 2 ? 0 : COUNTERS * 4 + tiles * n * 65536; }
};
static Ranges logit_ranges(int64_t T, int64_t H, int64_t cols) {
  Ranges best;
  if (tile_for(T, cols) != 128) return best;
  const int64_t room = 2 * split_device_cus(), all = cdiv(T, 128) * cdiv(cols, 128), tiles = all % room, steps = cdiv(H, KSTEP);
  if (tiles == 0 || tiles > COUNTERS || all - tiles > (1 << 30)) return best;
  const double rows = (double)cdiv(std::min<int64_t>(T, 128), 16) / 8;
  double t_best = 0.63 * (double)steps;
  for (int n = 2; n <= std::min<int64_t>(16, steps) && tiles * n <= room; ++n) {
    const double t = 0.63 * (double)steps / n + 1.34 * n * rows + 0.029 * (double)(tiles * n) * (1 + rows);
    if (t < t_best) {
      t_best = t;
      best = {(int)(all - tiles), n, tiles};
    }
  }
  return best;
}

// forward workspace: the pairs, the label logits, the rows' losses, the ranges' sums
static int64_t forward_parts(int64_t T, int64_t V) { return cdiv(V, tile_for(T, V)); }
static int64_t forward_sums(int64_t T, int64_t V) { return cdiv(forward_parts(T, V) * T * 8, 256) * 256 + 2 * cdiv(T * 4, 256) * 256; }
static int64_t forward_ws(int64_t T, int64_t H, int64_t V) { return forward_sums(T, V) + logit_ranges(T, H, V).bytes(); }

// backward: pieces of the vocabulary, tiles, ranges of the dX product, workspace
struct Plan {
  int64_t piece, block;  // words of a piece, elements of a block of dz
  int dz_tile, dx_tile, dw_tile, slices;
  Pair pair;  // where both gradients are wanted
  Ranges ranges;  // of the whole pieces' logits
  int64_t dz, acc, most, sums, bytes;
};
constexpr int64_t DZ_BYTES = (int64_t)512 << 20;
static Plan plan_of(int64_t T, int64_t H, int64_t V) {
  Plan p;
  const int64_t hk = cdiv(H, 64) * 64;
  const int64_t words = std::min<int64_t>(1 << 20, std::max<int64_t>(256, DZ_BYTES / (T * 2) / 256 * 256));
  p.piece = cdiv(cdiv(V, cdiv(V, words)), 256) * 256;
  const int64_t cols = std::min(p.piece, V);
  p.block = block_of(T);
  p.dz_tile = tile_for(T, cols);
  p.dw_tile = tile_for(cols, H);
  // dX: ranges can fill the chip with either tile; the small one where the large one's are too short
  const int64_t steps = cdiv(cols, KSTEP);
  p.dx_tile = cdiv(T, 256) * cdiv(H, 256) * std::max<int64_t>(1, steps / 16) < split_device_cus() || T <= 128 ? 128 : 256;
  p.slices = ranges_for(p.dx_tile, T, H, steps);
  p.pair = pair_of(T, H, cols);
  p.dz = cdiv(cols, 64) * p.block * 2;
  p.acc = dz_rows(T) * hk * 4 * std::max(p.slices, p.pair.slices);
  p.most = p.dz + p.acc;
  p.ranges = logit_ranges(T, H, cols);
  p.sums = p.most + 256;
  p.bytes = p.sums + p.ranges.bytes();
  return p;
}

// every product's grid, of up to 512 threads a tile and 16 ranges, below 2^32 threads
static bool grids_fit(int64_t T, int64_t H, int64_t V) {
  auto tiles = [](int64_t a, int64_t b) { return cdiv(a, 128) * cdiv(b, 128); };
  const int64_t most = 1 << 23;  // of 256 threads: 128 x 128, or four of 512
  return tiles(T, V) <= most && tiles(V, H) <= most && tiles(T, H) <= most / 16;
}

static int check(const char* fn, const void* w, int64_t T, int64_t H, int64_t V, int64_t ldw) {
  if (T < 0 || H < 1 || V < 1) return fail(NTLB_EINVAL, "%s: bad shape T %lld H %lld V %lld", fn, (long long)T, (long long)H, (long long)V);
  if (T > (1 << 22) || V > (1 << 30) || H > (1 << 20) || !grids_fit(T, H, V)) return fail(NTLB_EUNSUPPORTED, "%s: T %lld H %lld V %lld is too large", fn, (long long)T, (long long)H, (long long)V);
  if (!w || !aligned(w, 16) || ldw < H || ldw % 8 || ldw > (1 << 22)) return fail(NTLB_EINVAL, "%s: the weight needs 16-byte rows of at least H values", fn);
  return NTLB_OK;
}

}  // namespace xent
}  // namespace ntlb

using namespace ntlb;

extern "C" int ntlb_pad_rows(const uint16_t* x, int64_t ldx, int64_t R, int64_t H, uint16_t* out, int64_t ldo, void* stream) {
  const char* fn = "ntlb_pad_rows";
  clear_error();
  if (R < 0 || H < 1 || ldx < 0 || ldo < H || ldo % 8) return fail(NTLB_EINVAL, "%s: bad shape R %lld H %lld ldx %lld ldo %lld", fn, (long long)R, (long long)H, (long long)ldx, (long long)ldo);
  if (ldo > (1 << 22) || R > ((int64_t)1 << 31) - 1) return fail(NTLB_EUNSUPPORTED, "%s: R %lld ldo %lld is too large", fn, (long long)R, (long long)ldo);
  if (R == 0) return NTLB_OK;
  if (!x || !out || !aligned(out, 16)) return fail(NTLB_EINVAL, "%s: bad pointer", fn);
  // few rows: one each to a thousand workgroups (1003 x 345: 9.2 us by 46 rows a workgroup)
  const int per = (int)std::max<int64_t>(1, std::min(2048 / (ldo / 8), R / 1024));
  xent::pad_kernel<<<(unsigned)cdiv(R, per), 256, 0, as_stream(stream)>>>(x, ldx, R, H, out, ldo, per);
  return check_launch(fn);
}

// An empty batch leaves the state of one row, none of it live, and its dW (zero) goes
// through the same product
extern "C" int64_t ntlb_linear_xent_state_bytes(int64_t T, int64_t H) { return T < 0 || H < 1 ? 0 : xent::state_of(std::max<int64_t>(T, 1), H).bytes; }

extern "C" int64_t ntlb_linear_xent_workspace_bytes(int64_t T, int64_t H, int64_t V, int backward) {
  if (T < 0 || H < 1 || V < 1) return 0;
  if (backward) return xent::plan_of(std::max<int64_t>(T, 1), H, V).bytes;
  return T > 0 ? xent::forward_ws(T, H, V) : 0;
}

extern "C" int ntlb_linear_xent_forward(const uint16_t* x, int64_t ldx, const uint16_t* w, int64_t ldw,
                                        const void* targets, int targets64, int64_t T, int64_t H, int64_t V,
                                        int64_t ignore_index, int reduction, float* loss, void* state, void* workspace,
                                        int64_t ws_bytes, void* stream) {
  const char* fn = "ntlb_linear_xent_forward";
  clear_error();
  if (int rc = xent::check(fn, w, T, H, V, ldw)) return rc;
  if (reduction < 0 || reduction > 2) return fail(NTLB_EINVAL, "%s: bad reduction %d", fn, reduction);
  if (!loss || !state || !aligned(state, 256)) return fail(NTLB_EINVAL, "%s: NULL pointer", fn);
  if (T > 0 && (!x || !targets || (ldx != 0 && ldx < H))) return fail(NTLB_EINVAL, "%s: bad hidden or targets", fn);
  const int64_t need = T > 0 ? xent::forward_ws(T, H, V) : 0;
  if (ws_bytes < need || (need && (!workspace || !aligned(workspace, 16)))) return fail(NTLB_EINVAL, "%s: workspace of %lld bytes, %lld needed", fn, (long long)ws_bytes, (long long)need);
  hipStream_t st = as_stream(stream);
  const xent::State s = xent::state_of(std::max<int64_t>(T, 1), H);
  uint8_t* sp = (uint8_t*)state;
  const xent::Targets tg{targets, targets64, T, V, ignore_index};
  const xent::Live o{(int32_t*)(sp + s.pos), (int32_t*)(sp + s.rows), (int32_t*)(sp + s.y), (int32_t*)(sp + s.live)};
  float2* stat = (float2*)(sp + s.stat);
  uint16_t* xp = (uint16_t*)(sp + s.xp);
  const int64_t parts = T > 0 ? xent::forward_parts(T, V) : 0;
  float2* part = (float2*)workspace;
  float* zl = T > 0 ? (float*)((uint8_t*)workspace + cdiv(parts * T * 8, 256) * 256) : nullptr;
  float* each = T > 0 ? zl + cdiv(T * 4, 256) * 64 : nullptr;
  const xent::Ranges ranges = T > 0 ? xent::logit_ranges(T, H, V) : xent::Ranges{};
  uint32_t* count = ranges.n > 1 ? (uint32_t*)((uint8_t*)workspace + xent::forward_sums(T, V)) : nullptr;
  float* rows_loss = reduction == 0 ? loss : nullptr;
  if (T > xent::HERE) {
    xent::scan_kernel<<<1, xent::SCAN, 0, st>>>(tg, o);
    xent::gather_kernel<false><<<(unsigned)T + 63, 256, 0, st>>>(x, ldx, H, tg, o, xp, s.hk, s.block, zl, rows_loss, count, xent::half_of(T));
  } else {
    xent::gather_kernel<true><<<(unsigned)T + 63, 256, 0, st>>>(x, ldx, H, tg, o, xp, s.hk, s.block, zl, rows_loss, count, xent::half_of(T));
  }
  if (T > 0) {
    xent::Args g{};
    g.a = {(const uint8_t*)xp, s.block * 2, T, s.hk};
    g.b = {(const uint8_t*)w, ldw * 2, V, H};
    g.M = T; g.N = V; g.live = o.live; g.group_m = 8; g.part = part; g.ldp = T; g.zl = zl; g.y = o.y;
    g.slices = ranges.n; g.base = ranges.base; g.count = count; g.part_z = count ? (float4*)(count + xent::COUNTERS) : nullptr;
    xent::launch_head<false, false, xent::EPI_LSE>(xent::tile_for(T, V), g, st);
  }
  const int mean = reduction == 2;
  // up to 64 rows one workgroup does it all; many pairs of few rows: more walkers to
  // a row (16 rows of 1024 pairs: 5.6 us, by 16 walkers 27; 4096 rows of 256: 8.5 and 6.7)
  if (reduction != 0 && T <= 16)
    xent::join_kernel<16, 64, true><<<1, 1024, 0, st>>>(part, T, parts, zl, o.rows, o.live, mean, stat, nullptr, loss);
  else if (reduction != 0 && T <= 64 && parts <= 256)
    xent::join_kernel<64, 16, true><<<1, 1024, 0, st>>>(part, T, parts, zl, o.rows, o.live, mean, stat, nullptr, loss);
  else if (T > 0) {
    if (parts > 128 && T <= 1024)
      xent::join_kernel<4, 256, false><<<(unsigned)cdiv(T, 4), 1024, 0, st>>>(part, T, parts, zl, o.rows, o.live, mean, stat, each, rows_loss);
    else
      xent::join_kernel<16, 16, false><<<(unsigned)cdiv(T, 16), 256, 0, st>>>(part, T, parts, zl, o.rows, o.live, mean, stat, each, rows_loss);
    if (reduction != 0) xent::total_kernel<<<1, 1024, 0, st>>>(each, o.live, mean, loss);
  }
  return check_launch(fn);
}

extern "C" int ntlb_linear_xent_backward(const void* state, const uint16_t* w, int64_t ldw, int64_t T, int64_t H,
                                         int64_t V, int reduction, const float* dloss, uint16_t* dx, int64_t lddx,
                                         uint16_t* dw, int64_t lddw, void* workspace, int64_t ws_bytes, void* stream) {
  const char* fn = "ntlb_linear_xent_backward";
  clear_error();
  if (int rc = xent::check(fn, w, T, H, V, ldw)) return rc;
  if (reduction < 0 || reduction > 2) return fail(NTLB_EINVAL, "%s: bad reduction %d", fn, reduction);
  if (!state || !aligned(state, 256) || (T > 0 && !dloss)) return fail(NTLB_EINVAL, "%s: NULL pointer", fn);
  if ((dx && lddx < H) || (dw && lddw < H)) return fail(NTLB_EINVAL, "%s: a gradient's pitch is below H", fn);
  if ((T == 0 || !dx) && !dw) return NTLB_OK;
  const int64_t Tn = std::max<int64_t>(T, 1);
  const xent::Plan p = xent::plan_of(Tn, H, V);
  if (ws_bytes < p.bytes || !workspace || !aligned(workspace, 16)) return fail(NTLB_EINVAL, "%s: workspace of %lld bytes, %lld needed", fn, (long long)ws_bytes, (long long)p.bytes);
  hipStream_t st = as_stream(stream);
  const xent::State s = xent::state_of(Tn, H);
  const uint8_t* sp = (const uint8_t*)state;
  const int32_t* live = (const int32_t*)(sp + s.live);
  uint16_t* dz = (uint16_t*)workspace;
  float* acc = (float*)((uint8_t*)workspace + p.dz);
  float* most = reduction == 0 ? (float*)((uint8_t*)workspace + p.most) : nullptr;
  const xent::Up up{dloss, most, reduction == 2};
  const bool both = dx && dw && T > 0;
  const int slices = both ? p.pair.slices : p.slices;
  uint32_t* count = p.ranges.n > 1 ? (uint32_t*)((uint8_t*)workspace + p.sums) : nullptr;
  if (most || count) xent::most_kernel<<<1, xent::COUNTERS, 0, st>>>(dloss, (const int32_t*)(sp + s.rows), live, most, count);
  for (int64_t v0 = 0; v0 < V; v0 += p.piece) {
    const int64_t n = std::min(p.piece, V - v0), np = cdiv(n, 64) * 64;
    const uint8_t* wp = (const uint8_t*)(w + v0 * ldw);
    xent::Args g{};
    g.live = live; g.group_m = 8;
    g.a = {sp + s.xp, s.block * 2, Tn, s.hk};
    g.b = {wp, ldw * 2, n, H};
    g.M = T; g.N = n; g.y = (const int32_t*)(sp + s.y); g.v0 = v0; g.stat = (const float2*)(sp + s.stat);
    g.rows = (const int32_t*)(sp + s.rows); g.up = up;
    g.out = dz; g.ldo = p.block; g.cols = np;
    // (the last piece may have fewer tiles than the others' base, or fewer past it)
    g.half = xent::half_of(T);
    g.slices = p.ranges.n; g.base = p.ranges.base; g.count = count;
    g.part_z = count ? (float4*)(count + xent::COUNTERS) : nullptr;
    if (T > 0) xent::launch_head<false, false, xent::EPI_DZ>(p.dz_tile, g, st);
    xent::Args x{}, q{};
    x.live = live + 1; x.group_m = 8; x.slices = slices;
    x.a = {(const uint8_t*)dz, p.block * 2, Tn, np};
    x.b = {wp, ldw * 2, H, n};
    x.M = xent::dz_rows(T); x.N = H; x.out = acc; x.ldo = s.hk; x.slice = x.M * s.hk; x.add = v0 > 0;
    q.live = live + 1; q.n = live; q.group_m = 8;
    q.a = {(const uint8_t*)dz, p.block * 2, np, Tn};
    q.b = {sp + s.xp, s.block * 2, s.hk, Tn};
    q.M = n; q.N = H; q.out = dw + v0 * lddw; q.ldo = lddw;
    q.up = up;
    if (both)
      xent::launch_pair(p.pair.tile, x, q, st);
    else if (dw)
      xent::launch_head<true, true, xent::EPI_STORE>(p.dw_tile, q, st);
    else if (dx)
      xent::launch_head<false, true, xent::EPI_ACC>(p.dx_tile, x, st);
  }
  if (dx && T > 0)
    xent::scatter_kernel<<<(unsigned)T, 256, 0, st>>>(acc, s.hk, xent::dz_rows(T) * s.hk, slices, xent::half_of(T), up, live, (const int32_t*)(sp + s.pos),
                                                     H, dx, lddx);
  return check_launch(fn);
}
