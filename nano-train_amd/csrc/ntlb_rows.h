// What the kernels over whole rows share (norm.hip, rms.hip, rms_bwd.hip): a row in
// registers as 16-byte vectors, its reductions, the weights beside it, and the sums
// of weight gradients over workgroups.
#pragma once

#include <hip/hip_runtime.h>

#include "ntlb_device.h"

namespace ntlb {
namespace rows {

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

// STREAM: read once and not again, a hint to the caches (8192 x 7168 bf16, rms norm: forward 101
// and 99 us, backward 77 and 75)
template <bool STREAM = false, int DT, int MODE>
__device__ __forceinline__ Raw load_vec(const void* row, const Span<DT, MODE>& s) {
  Raw r;
  if constexpr (MODE != TINY) {
    const u32x4_2* p = reinterpret_cast<const u32x4_2*>((const uint8_t*)row + (uint32_t)s.c * El<DT>::bytes);
    const u32x4_2 v = STREAM ? __builtin_nontemporal_load(p) : *p;
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

template <int DT>
__device__ __forceinline__ Raw pack(const float (&f)[El<DT>::n]) {
  Raw r;
  if constexpr (DT == DT_F32) {
#pragma unroll
    for (int i = 0; i < 4; ++i) r.w[i] = __float_as_uint(f[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (DT == DT_BF16) {
        const v2bf p = {(__bf16)f[2 * i], (__bf16)f[2 * i + 1]};
        r.w[i] = __builtin_bit_cast(uint32_t, p);
      } else {
        r.w[i] = (uint32_t)__half_as_ushort(f32_to_f16(f[2 * i])) |
                 ((uint32_t)__half_as_ushort(f32_to_f16(f[2 * i + 1])) << 16);
      }
    }
  }
  return r;
}

template <int DT, int MODE>
__device__ __forceinline__ void store_raw(void* row, const Span<DT, MODE>& s, const Raw& r) {
  if constexpr (MODE != TINY) {
    const u32x4_2 v = {r.w[0], r.w[1], r.w[2], r.w[3]};
    // streamed: not read again here (8192 x 7168 bf16 forward: 47 us without the hint, 44 with it)
    __builtin_nontemporal_store(v, reinterpret_cast<u32x4_2*>((uint8_t*)row + (uint32_t)s.c * El<DT>::bytes));
  } else {
#pragma unroll
    for (int i = 0; i < El<DT>::n; ++i)
      if (s.own(i)) {
        if constexpr (DT == DT_F32)
          ((uint32_t*)row)[i] = r.w[i];
        else
          ((uint16_t*)row)[i] = (uint16_t)(r.w[i >> 1] >> (16 * (i & 1)));
      }
  }
}
template <int DT, int MODE>
__device__ __forceinline__ void store_vec(void* row, const Span<DT, MODE>& s, const float (&f)[El<DT>::n]) {
  store_raw<DT, MODE>(row, s, pack<DT>(f));
}

// sum over each L lanes, in every lane
template <int L = 64>
__device__ __forceinline__ float wave_sum(float v) {
  static_assert(L == 16 || L == 32 || L == 64, "lanes of a row");
  v += __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(v), 0xB1, 0xF, 0xF, false));
  v += __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(v), 0x4E, 0xF, 0xF, false));
  v += __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(v), 0x141, 0xF, 0xF, false));
  v += __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(v), 0x140, 0xF, 0xF, false));
  if constexpr (L >= 32) v += __shfl_xor(v, 16);
  if constexpr (L == 64) v += __shfl_xor(v, 32);
  return v;
}

// N sums over the RT threads of a row; slot: LDS for RT / 64 waves, not the one
// of the reduction before (its reads may still run on)
template <int RT, int N>
__device__ __forceinline__ void row_sum(float (&v)[N], float* slot) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = wave_sum<(RT < 64 ? RT : 64)>(v[i]);
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
        unpack<WDT>(load_vec(w, q), u);
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
constexpr int block_threads() { return RT <= 64 ? 256 : RT; }  // rows of one wave or less share no barrier
// which of a workgroup's rows a thread has, uniform in the wave where it is
template <int RT>
__device__ __forceinline__ int row_of_block() {
  const int r = threadIdx.x / RT;
  return RT >= 64 ? __builtin_amdgcn_readfirstlane(r) : r;
}

// dw / db (blockIdx.y) of 32 columns, two a thread, so that a partial row's piece
// is a whole line: 64 walkers down the P partial rows, their sums added in a fixed
// tree (256 rows of 7168: 4.6 us, by 16 columns, one a thread, 6.8)
constexpr int FIN_COLS = 32, FIN_WALK = 64;
static __global__ void __launch_bounds__(FIN_COLS / 2 * FIN_WALK) finish_kernel(const float* part, int P, int H, void* dw, void* db,
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

}  // namespace rows
}  // namespace ntlb
