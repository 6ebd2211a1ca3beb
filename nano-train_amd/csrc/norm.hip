// Layer norm of the rows of x [T, H], forward and backward:
//   m = mean(x), r = 1 / sqrt(mean((x - m)^2) + eps), xh = (x - m) r
//   y = xh w + b
//   t = dy w,  dx = r (t - mean(t) - xh mean(t xh))
//   dw = sum over rows of dy xh,  db = sum over rows of dy
// All sums and statistics are fp32; y and dx are rounded once to x's type, dw
// and db once to the weights'.
//
// HBM-bound: x in, y out; x and dy in, dx out.  A row is read once and stays in
// registers: RT threads (one wave to 16) hold VPT 16-byte vectors each, and a
// workgroup walks rows with the weights, and in the backward the column sums
// dw and db, in registers, the next row's loads in flight while this one is
// reduced.  The variance is the mean of (x - m)^2 over the registers, a second
// reduction, because E[x^2] - m^2 cancels for rows far off centre.  The
// backward takes m and r from the forward (8 bytes a row) and so needs one
// reduction, of two sums.  Each workgroup writes one row of partial dw and db,
// which a second kernel sums in a fixed order: the result does not depend on
// how the workgroups are scheduled.
// Measured (a large copy runs at 5.3 TB/s): 8192 x 7168 bf16 forward 38.6 us (6.1
// TB/s), backward 70.0 (5.0) and 4.7 for dw and db's sums; 65536 x 512 fp16
// forward 23.8 us (5.7), backward 34.8 (5.8) and 3.9; one row of 7168 3.2 us, the
// launch and the latency of one pass.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "ntlb_device.h"
#include "ntlb_host.h"
#include "ntlb_splitk.h"

namespace ntlb {
namespace norm {

typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
// rows of an odd pitch start at any element: the vector accesses carry the
// element's alignment, not 16 bytes
typedef uint32_t u32x4_2 __attribute__((ext_vector_type(4), aligned(2)));

template <int DT>
struct El {
  static constexpr int bytes = DT == DT_F32 ? 4 : 2;
  static constexpr int n = 16 / bytes;  // elements of a vector
};

struct Raw {
  uint32_t w[4];
};

// Unpacked values are not kept across a reduction (their registers cost more
// than unpacking again): the raw vector is a new value once `sum` is there
__device__ __forceinline__ void renew(Raw& r, float sum) {
  asm("" : "+v"(r.w[0]), "+v"(r.w[1]), "+v"(r.w[2]), "+v"(r.w[3]) : "v"(sum));
}

// How a row divides into vectors of n elements: WHOLE: H is a multiple of n;
// RAGGED: the last vector of a row begins at H - n and shares elements with the
// one before it; TINY: H < n.  A thread with no vector of its own takes the last
// one again.  So every access is unconditional and in bounds, and a shared
// element is computed alike by those that hold it (who may all store it); only
// sums must count it once.  (A branch around a load or store would make the
// compiler wait for everything in flight.)
constexpr int WHOLE = 0, RAGGED = 1, TINY = 2;

template <int DT, int MODE>
struct Span {
  static constexpr int N = El<DT>::n;
  int c;      // first column
  int first;  // first element of its own
  int end;    // TINY: elements in the row
  __device__ __forceinline__ Span(int vec, int H) {
    const int c0 = vec * N;
    if constexpr (MODE == TINY) {
      c = 0;
      first = vec == 0 ? 0 : N;
      end = H;
    } else {
      c = min(c0, H - N);
      first = min(c0 - c, N);
      end = N;
    }
  }
  __device__ __forceinline__ bool own(int i) const {
    if constexpr (MODE == WHOLE) return first == 0;
    if constexpr (MODE == RAGGED) return i >= first;
    return first == 0 && i < end;
  }
};

template <int DT, int MODE>
__device__ __forceinline__ Raw load_vec(const void* row, const Span<DT, MODE>& s) {
  Raw r;
  if constexpr (MODE != TINY) {
    const u32x4_2 v = *reinterpret_cast<const u32x4_2*>((const uint8_t*)row + (uint32_t)s.c * El<DT>::bytes);
    r.w[0] = v[0]; r.w[1] = v[1]; r.w[2] = v[2]; r.w[3] = v[3];
  } else {
    r = {{0, 0, 0, 0}};
#pragma unroll
    for (int i = 0; i < El<DT>::n; ++i)
      if (i < s.end) {
        if constexpr (DT == DT_F32)
          r.w[i] = ((const uint32_t*)row)[i];
        else
          r.w[i >> 1] |= (uint32_t)((const uint16_t*)row)[i] << (16 * (i & 1));
      }
  }
  return r;
}

template <int DT>
__device__ __forceinline__ void unpack(const Raw& r, float (&f)[El<DT>::n]) {
#pragma unroll
  for (int i = 0; i < El<DT>::n; ++i) {
    if constexpr (DT == DT_F32)
      f[i] = __uint_as_float(r.w[i]);
    else if constexpr (DT == DT_BF16)
      f[i] = (i & 1) ? __uint_as_float(r.w[i >> 1] & 0xFFFF0000u) : __uint_as_float(r.w[i >> 1] << 16);
    else
      f[i] = __half2float(__ushort_as_half((uint16_t)(r.w[i >> 1] >> (16 * (i & 1)))));
  }
}

template <int DT, int MODE>
__device__ __forceinline__ void store_vec(void* row, const Span<DT, MODE>& s, const float (&f)[El<DT>::n]) {
  uint32_t w[4];
  if constexpr (DT == DT_F32) {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __float_as_uint(f[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (DT == DT_BF16) {
        const v2bf p = {(__bf16)f[2 * i], (__bf16)f[2 * i + 1]};
        w[i] = __builtin_bit_cast(uint32_t, p);
      } else {
        w[i] = (uint32_t)__half_as_ushort(f32_to_f16(f[2 * i])) |
               ((uint32_t)__half_as_ushort(f32_to_f16(f[2 * i + 1])) << 16);
      }
    }
  }
  if constexpr (MODE != TINY) {
    const u32x4_2 v = {w[0], w[1], w[2], w[3]};
    // streamed: not read again here (8192 x 7168 bf16 forward: 47 us without the hint, 44 with it)
    __builtin_nontemporal_store(v, reinterpret_cast<u32x4_2*>((uint8_t*)row + (uint32_t)s.c * El<DT>::bytes));
  } else {
#pragma unroll
    for (int i = 0; i < El<DT>::n; ++i)
      if (s.own(i)) {
        if constexpr (DT == DT_F32)
          ((uint32_t*)row)[i] = w[i];
        else
          ((uint16_t*)row)[i] = (uint16_t)(w[i >> 1] >> (16 * (i & 1)));
      }
  }
}

// sum over the 64 lanes, in every lane
__device__ __forceinline__ float wave_sum(float v) {
  v += __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(v), 0xB1, 0xF, 0xF, false));
  v += __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(v), 0x4E, 0xF, 0xF, false));
  v += __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(v), 0x141, 0xF, 0xF, false));
  v += __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(v), 0x140, 0xF, 0xF, false));
  v += __shfl_xor(v, 16);
  v += __shfl_xor(v, 32);
  return v;
}

// N sums over the RT threads of a row; slot: LDS for RT / 64 waves, not the one
// of the reduction before (its reads may still run on)
template <int RT, int N>
__device__ __forceinline__ void row_sum(float (&v)[N], float* slot) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = wave_sum(v[i]);
  if constexpr (RT > 64) {
    constexpr int NW = RT / 64;
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) slot[(threadIdx.x >> 6) * N + i] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float s = slot[i];
#pragma unroll
      for (int w = 1; w < NW; ++w) s += slot[w * N + i];
      v[i] = s;
    }
  }
}

struct Args {
  const void* x;
  int64_t ldx;  // in bytes, as the others
  const void* w;
  const void* b;
  int w_dtype;
  int64_t T;
  int H;
  float eps;
  void* y;  // y, or dx
  int64_t ldy;
  float* mean;
  float* rstd;
  const void* dy;
  int64_t lddy;
  float* part;  // [2][workgroups][H]: dw, db
};

// the weights of a thread's vectors as floats (w NULL: `none`), there before
// anything else is issued: the kernel's one branch on types, outside its loop
template <int WDT, int DT, int RT, int VPT, int MODE>
__device__ __forceinline__ void load_weights_of(const void* w, int t, int H, float (&f)[VPT][El<DT>::n]) {
  constexpr int N = El<DT>::n, M = El<WDT>::n;
#pragma unroll
  for (int v = 0; v < VPT; ++v) {
    const Span<DT, MODE> s(t + v * RT, H);
    if constexpr (MODE == TINY || M > N) {
#pragma unroll
      for (int i = 0; i < N; ++i) f[v][i] = load_elem(w, WDT, min(s.c + i, H - 1));
    } else {
#pragma unroll
      for (int h = 0; h < N / M; ++h) {
        Span<WDT, MODE> q(0, H);
        q.c = s.c + h * M;
        float u[M];
        unpack<WDT>(load_vec<WDT, MODE>(w, q), u);
#pragma unroll
        for (int i = 0; i < M; ++i) f[v][h * M + i] = u[i];
      }
    }
  }
}
template <int DT, int RT, int VPT, int MODE>
__device__ __forceinline__ void load_weights(const void* w, int dt, int t, int H, float none,
                                             float (&f)[VPT][El<DT>::n]) {
  if (!w) {
#pragma unroll
    for (int v = 0; v < VPT; ++v)
#pragma unroll
      for (int i = 0; i < El<DT>::n; ++i) f[v][i] = none;
  } else if (dt == DT_F32) {
    load_weights_of<DT_F32, DT, RT, VPT, MODE>(w, t, H, f);
  } else if (dt == DT_BF16) {
    load_weights_of<DT_BF16, DT, RT, VPT, MODE>(w, t, H, f);
  } else {
    load_weights_of<DT_F16, DT, RT, VPT, MODE>(w, t, H, f);
  }
#pragma unroll
  for (int v = 0; v < VPT; ++v)
#pragma unroll
    for (int i = 0; i < El<DT>::n; ++i) asm volatile("" : "+v"(f[v][i]));
}

template <int RT>
constexpr int block_threads() { return RT == 64 ? 256 : RT; }  // one-wave rows share no barrier

template <int DT, int RT, int VPT, int MODE>
__global__ void __launch_bounds__(block_threads<RT>()) forward_kernel(Args g) {
  constexpr int N = El<DT>::n, ROWS = block_threads<RT>() / RT;
  __shared__ float red[2][RT / 64];
  const int t = threadIdx.x % RT, H = g.H;
  const int64_t stride = (int64_t)gridDim.x * ROWS;
  // one row per wave or more waves: scalar, so that row addresses are
  int64_t row = (int64_t)blockIdx.x * ROWS + __builtin_amdgcn_readfirstlane(threadIdx.x / RT);
  const float inv = 1.0f / (float)H;
  float w[VPT][N], b[VPT][N];
  load_weights<DT, RT, VPT, MODE>(g.w, g.w_dtype, t, H, 1.0f, w);
  load_weights<DT, RT, VPT, MODE>(g.b, g.w_dtype, t, H, 0.0f, b);
  Raw nx[VPT];
  auto fetch = [&](int64_t r) {
    const uint8_t* p = (const uint8_t*)g.x + r * g.ldx;
#pragma unroll
    for (int v = 0; v < VPT; ++v) nx[v] = load_vec(p, Span<DT, MODE>(t + v * RT, H));
  };
  if (row < g.T) fetch(row);
  for (; row < g.T; row += stride) {
    Raw x[VPT];
#pragma unroll
    for (int v = 0; v < VPT; ++v) x[v] = nx[v];
    fetch(min<int64_t>(row + stride, g.T - 1));  // past the end: the last row again
    float s[1] = {0.f};
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      const Span<DT, MODE> sp(t + v * RT, H);
      float f[N];
      unpack<DT>(x[v], f);
#pragma unroll
      for (int i = 0; i < N; ++i) s[0] += sp.own(i) ? f[i] : 0.f;
    }
    row_sum<RT, 1>(s, red[0]);
    const float m = s[0] * inv;
    float q[1] = {0.f};
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      const Span<DT, MODE> sp(t + v * RT, H);
      float f[N];
      renew(x[v], m);
      unpack<DT>(x[v], f);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float d = sp.own(i) ? f[i] - m : 0.f;
        q[0] += d * d;
      }
    }
    row_sum<RT, 1>(q, red[1]);
    const float r = 1.0f / sqrtf(q[0] * inv + g.eps);
    uint8_t* yp = (uint8_t*)g.y + row * g.ldy;
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      float f[N];
      renew(x[v], r);
      unpack<DT>(x[v], f);
#pragma unroll
      for (int i = 0; i < N; ++i) f[i] = (f[i] - m) * r * w[v][i] + b[v][i];
      store_vec(yp, Span<DT, MODE>(t + v * RT, H), f);
    }
    if (g.mean && t == 0) {
      g.mean[row] = m;
      g.rstd[row] = r;
    }
  }
}

// DX: dx is wanted; DW: the partial sums of dw and db are
template <int DT, int RT, int VPT, int MODE, bool DX, bool DW>
__global__ void __launch_bounds__(block_threads<RT>()) backward_kernel(Args g) {
  constexpr int N = El<DT>::n, BT = block_threads<RT>(), ROWS = BT / RT;
  __shared__ float red[2][RT / 64 * 2];
  const int t = threadIdx.x % RT, H = g.H;
  const int64_t stride = (int64_t)gridDim.x * ROWS;
  // one row per wave or more waves: scalar, so that row addresses are
  int64_t row = (int64_t)blockIdx.x * ROWS + __builtin_amdgcn_readfirstlane(threadIdx.x / RT);
  const float inv = 1.0f / (float)H;
  float w[VPT][N], aw[VPT][N], ab[VPT][N];
  if constexpr (DX) load_weights<DT, RT, VPT, MODE>(g.w, g.w_dtype, t, H, 1.0f, w);
#pragma unroll
  for (int v = 0; v < VPT; ++v)
#pragma unroll
    for (int i = 0; i < N; ++i) aw[v][i] = ab[v][i] = 0.f;
  Raw nx[VPT], nd[VPT];
  float nm = 0.f, nr = 0.f;
  auto fetch = [&](int64_t r) {
    const uint8_t* p = (const uint8_t*)g.x + r * g.ldx;
    const uint8_t* d = (const uint8_t*)g.dy + r * g.lddy;
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      nx[v] = load_vec(p, Span<DT, MODE>(t + v * RT, H));
      nd[v] = load_vec(d, Span<DT, MODE>(t + v * RT, H));
    }
    nm = g.mean[r];
    nr = g.rstd[r];
  };
  // eight vectors a thread leave no registers for a row in flight beside this one
  constexpr bool AHEAD = VPT < 8;
  if (AHEAD && row < g.T) fetch(row);
#pragma unroll 1
  for (int buf = 0; row < g.T; row += stride, buf ^= 1) {
    if (!AHEAD) fetch(row);
    Raw x[VPT], d[VPT];
    const float m = nm, r = nr;
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      x[v] = nx[v];
      d[v] = nd[v];
    }
    if (AHEAD) fetch(min<int64_t>(row + stride, g.T - 1));  // past the end: the last row again
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      float f[N], e[N];
      const Span<DT, MODE> sp(t + v * RT, H);
      unpack<DT>(x[v], f);
      unpack<DT>(d[v], e);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float xh = (f[i] - m) * r;
        e[i] = sp.own(i) ? e[i] : 0.f;
        if constexpr (DW) {
          aw[v][i] += e[i] * xh;
          ab[v][i] += e[i];
        }
        if constexpr (DX) {
          const float u = e[i] * w[v][i];
          s[0] += u;
          s[1] += u * xh;
        }
      }
      if constexpr (DW) {  // added here and now: dy and xh are not kept for it
#pragma unroll
        for (int i = 0; i < N; ++i) asm volatile("" : "+v"(aw[v][i]), "+v"(ab[v][i]));
      }
    }
    if constexpr (DX) {
      row_sum<RT, 2>(s, red[buf]);
      const float s0 = s[0] * inv, s1 = s[1] * inv;
      uint8_t* dp = (uint8_t*)g.y + row * g.ldy;
#pragma unroll
      for (int v = 0; v < VPT; ++v) {
        float f[N], e[N];
        renew(x[v], s0);
        renew(d[v], s0);
        unpack<DT>(x[v], f);
        unpack<DT>(d[v], e);
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const float xh = (f[i] - m) * r;
          f[i] = r * (e[i] * w[v][i] - s0 - xh * s1);
        }
        store_vec(dp, Span<DT, MODE>(t + v * RT, H), f);
      }
    }
  }
  if constexpr (DW) {
    float* pw = g.part + (int64_t)blockIdx.x * H;
    float* pb = pw + (int64_t)gridDim.x * H;
    if constexpr (ROWS == 1) {
#pragma unroll
      for (int v = 0; v < VPT; ++v) {
        const Span<DT, MODE> sp(t + v * RT, H);
#pragma unroll
        for (int i = 0; i < N; ++i)
          if (sp.own(i)) {
            pw[sp.c + i] = aw[v][i];
            pb[sp.c + i] = ab[v][i];
          }
      }
    } else {
      // the workgroup's row walkers, summed in their order
      constexpr int W = RT * VPT * N;
      __shared__ float sum[ROWS][W];
      for (int k = 0; k < 2; ++k) {
        __syncthreads();
#pragma unroll
        for (int v = 0; v < VPT; ++v) {
          const Span<DT, MODE> sp(t + v * RT, H);
#pragma unroll
          for (int i = 0; i < N; ++i)
            if (sp.own(i)) sum[threadIdx.x / RT][sp.c + i] = k ? ab[v][i] : aw[v][i];
        }
        __syncthreads();
        for (int c = threadIdx.x; c < H; c += BT) {
          float a = sum[0][c];
#pragma unroll
          for (int q = 1; q < ROWS; ++q) a += sum[q][c];
          (k ? pb : pw)[c] = a;
        }
      }
    }
  }
}

// dw / db (blockIdx.y) of 32 columns, two a thread, so that a partial row's piece
// is a whole line: 64 walkers down the P partial rows, their sums added in a fixed
// tree (256 rows of 7168: 4.6 us, by 16 columns, one a thread, 6.8)
constexpr int FIN_COLS = 32, FIN_WALK = 64;
__global__ void __launch_bounds__(FIN_COLS / 2 * FIN_WALK) finish_kernel(const float* part, int P, int H, void* dw, void* db,
                                                                          int w_dtype) {
  typedef float f2 __attribute__((ext_vector_type(2), aligned(4)));
  constexpr int PAIRS = FIN_COLS / 2;
  __shared__ f2 sum[FIN_WALK / 4][PAIRS];
  const int c = blockIdx.x * FIN_COLS + threadIdx.x % PAIRS * 2, q = threadIdx.x / PAIRS;
  const float* p = part + (int64_t)blockIdx.y * P * H;
  f2 a = {0.f, 0.f};
  if (c + 1 < H) {
#pragma unroll 4
    for (int r = q; r < P; r += FIN_WALK) a += *reinterpret_cast<const f2*>(p + (int64_t)r * H + c);
  } else if (c < H) {
    for (int r = q; r < P; r += FIN_WALK) a[0] += p[(int64_t)r * H + c];
  }
#pragma unroll
  for (int d = PAIRS; d < 64; d *= 2) a += (f2){__shfl_xor(a[0], d), __shfl_xor(a[1], d)};
  if ((threadIdx.x & 63) < PAIRS) sum[threadIdx.x >> 6][threadIdx.x % PAIRS] = a;
  __syncthreads();
  void* out = blockIdx.y ? db : dw;
  if (q == 0 && c < H && out) {
#pragma unroll
    for (int k = 1; k < FIN_WALK / 4; ++k) a += sum[k][threadIdx.x];
    store_elem(out, w_dtype, c, a[0]);
    if (c + 1 < H) store_elem(out, w_dtype, c + 1, a[1]);
  }
}

constexpr int MAX_H = 16384;

// Threads and vectors each for a row of nv vectors of 16 bytes, and workgroups
// per compute unit.  The forward is fastest with four vectors a thread (few
// waves to reduce over, enough loads in flight), the backward, which holds
// three times the registers, with one.  us at 8192 x 7168 bf16 (896 vectors),
// threads x vectors x workgroups: forward 256x4x3 43, 512x2x2 44, 1024x1x2 47;
// backward 1024x1x1 78, 512x2x1 84, 256x4x2 91.  At 16384 x 2048: forward 64x4 22,
// 256x1 23; backward 256x1x2 46, 64x4 46.  Few workgroups keep the partial rows of dw and db
// few: 1024x1x2 took 100.
struct Shape {
  int rt, vpt, per_cu;
};
static Shape forward_shape(int64_t nv) {
  if (nv <= 64) return {64, 1, 4};
  if (nv <= 128) return {64, 2, 4};
  if (nv <= 256) return {64, 4, 4};
  if (nv <= 512) return {128, 4, 8};
  if (nv <= 1024) return {256, 4, 3};
  if (nv <= 2048) return {512, 4, 2};
  return {512, 8, 1};
}
static Shape backward_shape(int64_t nv) {
  if (nv <= 64) return {64, 1, 2};
  if (nv <= 128) return {128, 1, 4};
  if (nv <= 256) return {256, 1, 2};
  if (nv <= 512) return {512, 1, 1};
  if (nv <= 1024) return {1024, 1, 1};
  if (nv <= 2048) return {512, 4, 1};
  return {512, 8, 1};
}
static int64_t vectors(int dt, int64_t H) { return cdiv(H * dtype_size(dt), 16); }
static int64_t groups(const Shape& s, int64_t T) {
  return std::max<int64_t>(1, std::min(cdiv(T, s.rt == 64 ? 4 : 1), (int64_t)split_device_cus() * s.per_cu));
}

template <int DT, int RT, int VPT, int MODE>
static void launch_forward(const Args& g, int64_t n, hipStream_t st) {
  forward_kernel<DT, RT, VPT, MODE><<<(unsigned)n, block_threads<RT>(), 0, st>>>(g);
}
template <int DT, int RT, int VPT, int MODE>
static void launch_backward(const Args& g, int64_t n, bool dx, bool dw, hipStream_t st) {
  const dim3 grd((unsigned)n), blk(block_threads<RT>());
  if (dx && dw)
    backward_kernel<DT, RT, VPT, MODE, true, true><<<grd, blk, 0, st>>>(g);
  else if (dx)
    backward_kernel<DT, RT, VPT, MODE, true, false><<<grd, blk, 0, st>>>(g);
  else
    backward_kernel<DT, RT, VPT, MODE, false, true><<<grd, blk, 0, st>>>(g);
}

struct Forward {
  const Args& g;
  int64_t n;
  hipStream_t st;
  template <int DT, int RT, int VPT, int MODE>
  void run() const { launch_forward<DT, RT, VPT, MODE>(g, n, st); }
  template <int DT, int MODE>
  bool shaped(const Shape& s) const {
#define NTLB_CASE(RT, VPT) \
  if (s.rt == RT && s.vpt == VPT) return run<DT, RT, VPT, MODE>(), true;
    NTLB_CASE(64, 1) NTLB_CASE(64, 2) NTLB_CASE(64, 4) NTLB_CASE(128, 4) NTLB_CASE(256, 4) NTLB_CASE(512, 4)
    if constexpr (DT == DT_F32) NTLB_CASE(512, 8)
    return false;
  }
};
struct Backward {
  const Args& g;
  int64_t n;
  bool dx, dw;
  hipStream_t st;
  template <int DT, int RT, int VPT, int MODE>
  void run() const { launch_backward<DT, RT, VPT, MODE>(g, n, dx, dw, st); }
  template <int DT, int MODE>
  bool shaped(const Shape& s) const {
    NTLB_CASE(64, 1) NTLB_CASE(128, 1) NTLB_CASE(256, 1) NTLB_CASE(512, 1) NTLB_CASE(1024, 1) NTLB_CASE(512, 4)
    if constexpr (DT == DT_F32) NTLB_CASE(512, 8)
#undef NTLB_CASE
    return false;
  }
};
// the kernel of a type, a width and a shape; false if there is none
template <int DT, typename F>
static bool dispatch_dt(const Shape& s, int H, const F& f) {
  if (H < El<DT>::n) return f.template run<DT, 64, 1, TINY>(), true;
  return H % El<DT>::n ? f.template shaped<DT, RAGGED>(s) : f.template shaped<DT, WHOLE>(s);
}
template <typename F>
static bool dispatch(int dt, const Shape& s, int64_t H, const F& f) {
  if (dt == NTLB_F32) return dispatch_dt<DT_F32>(s, (int)H, f);
  if (dt == NTLB_BF16) return dispatch_dt<DT_BF16>(s, (int)H, f);
  return dispatch_dt<DT_F16>(s, (int)H, f);
}

static int check(const char* fn, const void* x, int dt, int64_t T, int64_t H, int64_t ldx, int wdt) {
  if (!valid_dtype(dt) || !valid_dtype(wdt)) return fail(NTLB_EINVAL, "%s: bad dtype %d / %d", fn, dt, wdt);
  if (T < 0 || H < 1) return fail(NTLB_EINVAL, "%s: bad shape %lld x %lld", fn, (long long)T, (long long)H);
  if (H > MAX_H) return fail(NTLB_EUNSUPPORTED, "%s: rows of %lld elements (at most %d)", fn, (long long)H, MAX_H);
  if (T > 0 && !x) return fail(NTLB_EINVAL, "%s: NULL x", fn);
  // rows may repeat (pitch 0) in an input, not overlap in part
  if (ldx != 0 && ldx < H) return fail(NTLB_EINVAL, "%s: row pitch %lld below %lld", fn, (long long)ldx, (long long)H);
  return NTLB_OK;
}

}  // namespace norm
}  // namespace ntlb

using namespace ntlb;

extern "C" int ntlb_layer_norm_forward(const void* x, int x_dtype, int64_t T, int64_t H, int64_t ldx, const void* w,
                                       const void* b, int w_dtype, float eps, void* y, int64_t ldy, float* mean,
                                       float* rstd, void* stream) {
  const char* fn = "ntlb_layer_norm_forward";
  clear_error();
  if (int rc = norm::check(fn, x, x_dtype, T, H, ldx, w_dtype)) return rc;
  if (!(eps >= 0.0f)) return fail(NTLB_EINVAL, "%s: eps must not be negative", fn);
  if ((mean == nullptr) != (rstd == nullptr)) return fail(NTLB_EINVAL, "%s: mean and rstd go together", fn);
  if (T == 0) return NTLB_OK;
  if (!y || ldy < H) return fail(NTLB_EINVAL, "%s: bad y", fn);
  const int64_t e = dtype_size(x_dtype);
  norm::Args g{};
  g.x = x; g.ldx = ldx * e; g.w = w; g.b = b; g.w_dtype = w_dtype; g.T = T; g.H = (int)H; g.eps = eps;
  g.y = y; g.ldy = ldy * e; g.mean = mean; g.rstd = rstd;
  const norm::Shape s = norm::forward_shape(norm::vectors(x_dtype, H));
  const int64_t n = norm::groups(s, T);
  hipStream_t st = as_stream(stream);
  if (!norm::dispatch(x_dtype, s, H, norm::Forward{g, n, st})) return fail(NTLB_EUNSUPPORTED, "%s: no kernel for %lld columns", fn, (long long)H);
  return check_launch(fn);
}

extern "C" int64_t ntlb_layer_norm_workspace_bytes(int x_dtype, int64_t T, int64_t H) {
  if (!valid_dtype(x_dtype) || T < 1 || H < 1 || H > norm::MAX_H) return 0;
  return norm::groups(norm::backward_shape(norm::vectors(x_dtype, H)), T) * H * 8;
}

extern "C" int ntlb_layer_norm_backward(const void* x, int x_dtype, int64_t T, int64_t H, int64_t ldx, const void* dy,
                                        int64_t lddy, const float* mean, const float* rstd, const void* w, int w_dtype,
                                        void* dx, int64_t lddx, void* dw, void* db, void* workspace, int64_t ws_bytes,
                                        void* stream) {
  const char* fn = "ntlb_layer_norm_backward";
  clear_error();
  if (int rc = norm::check(fn, x, x_dtype, T, H, ldx, w_dtype)) return rc;
  if (T > 0 && (!dy || !mean || !rstd)) return fail(NTLB_EINVAL, "%s: NULL pointer", fn);
  if (lddy != 0 && lddy < H) return fail(NTLB_EINVAL, "%s: dy's row pitch %lld below %lld", fn, (long long)lddy, (long long)H);
  if (dx && lddx < H) return fail(NTLB_EINVAL, "%s: dx's row pitch %lld below %lld", fn, (long long)lddx, (long long)H);
  const bool sums = dw || db;
  if (!dx && !sums) return NTLB_OK;
  const norm::Shape s = norm::backward_shape(norm::vectors(x_dtype, H));
  const int64_t n = T > 0 ? norm::groups(s, T) : 0;
  if (sums && n * H * 8 > ws_bytes) return fail(NTLB_EINVAL, "%s: workspace of %lld bytes, %lld needed", fn, (long long)ws_bytes, (long long)(n * H * 8));
  if (sums && n && (!workspace || !aligned(workspace, 4))) return fail(NTLB_EINVAL, "%s: bad workspace", fn);
  const int64_t e = dtype_size(x_dtype);
  norm::Args g{};
  g.x = x; g.ldx = ldx * e; g.w = w; g.w_dtype = w_dtype; g.T = T; g.H = (int)H;
  g.y = dx; g.ldy = lddx * e; g.mean = const_cast<float*>(mean); g.rstd = const_cast<float*>(rstd);
  g.dy = dy; g.lddy = lddy * e; g.part = (float*)workspace;
  hipStream_t st = as_stream(stream);
  if (T > 0) {
    if (!norm::dispatch(x_dtype, s, H, norm::Backward{g, n, dx != nullptr, sums, st})) return fail(NTLB_EUNSUPPORTED, "%s: no kernel for %lld columns", fn, (long long)H);
    if (int rc = check_launch(fn)) return rc;
  }
  if (sums) {
    const dim3 grd((unsigned)cdiv(H, norm::FIN_COLS), 2), blk(norm::FIN_COLS / 2 * norm::FIN_WALK);
    norm::finish_kernel<<<grd, blk, 0, st>>>((const float*)workspace, (int)n, (int)H, dw, db, w_dtype);
    return check_launch(fn);
  }
  return NTLB_OK;
}
