// SwiGLU of a product's output x [T, 2I] that holds gate and up, forward and backward:
//   h = g sig(g) u,  dg = dh u sig(g) (1 + g (1 - sig(g))),  du = dh g sig(g)
// gate and up are the halves of a row, or lie in alternating blocks of columns (a
// multiple of 128).  fp32 inside, one rounding to x's type.  (torch's F.silu(g) * u in
// 16 bits rounds twice, which swiglu_backward of moe_bwd.hip follows.)  For the
// backward x stays as it is, or gate and up are kept in 8 bits (ntlb_kept.h), in
// tiles of 128 of h's columns: codes [T][gate, up][NT 128], a byte each tile
// [T][gate, up][NT].
//
// With t = exp(-|g|) sigmoid and its complement are 1 / (1 + t) and t / (1 + t), the
// former at g's own side: neither overflows nor cancels.  Of a gate below -87.3 t is
// under the normal numbers of fp32 (and of the exponential's unit, which gives 0), while its
// product with g, u and dh may be any number: t is the square of exp(-|g| / 2), and a
// sigmoid below 1/2 is held as two factors, the second multiplied last.  So results are
// right down to g = -174, where the root ends too; below it they are 0.
//
// HBM-bound.  16 lanes (fp32: 32) take a tile, a lane 16 bytes of gate and of up, so
// that a tile's scale is a reduction within the wave and nothing is read twice.  32768 x
// 2048 bf16: 66 us (6.1 TB/s), keeping codes 93 (5.8), backward 106 (6.3), from codes
// 86 (6.2).  Codes as 16-byte stores, two lanes' exchanged: slower.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "ntlb_device.h"
#include "ntlb_host.h"
#include "ntlb_kept.h"
#include "ntlb_rows.h"

namespace ntlb {
namespace swiglu {

using namespace rows;

constexpr int THREADS = 256;

struct Args {
  const void* x;
  int64_t ldx;  // in bytes, as the others
  int64_t tiles;  // T NT
  int I, NT, block;
  TileRows by;  // of NT tiles
  void* h;
  int64_t ldh;
  uint8_t* kc;
  uint8_t* ke;
  const void* dh;
  int64_t lddh;
  void* dx;
  int64_t lddx;
};

// sig(g) = near far, far being 1 or t's root; rest = 1 - sig(g).
// For 16-bit results the exponential's argument is rounded once (|g| 2^-24 of the
// result) and the reciprocal is the unit's own (2^-23); fp32 takes the exact ones.
struct Sigmoid {
  float near, far, rest;
};
template <int DT>
__device__ __forceinline__ Sigmoid sigmoid(float g) {
  float root, a;
  if constexpr (DT == DT_F32) {
    root = expf(-0.5f * __builtin_fabsf(g));
    a = 1.0f / (1.0f + root * root);
  } else {
    root = __builtin_amdgcn_exp2f(-__builtin_fabsf(g) * 7.21347511e-01f);
    a = __builtin_amdgcn_rcpf(1.0f + root * root);
  }
  const float b = root * a;
  return g >= 0.f ? Sigmoid{a, 1.0f, root * b} : Sigmoid{b, root, a};  // NaN: all three
}

// N values from column c of a row, those past the I of its part zero
template <int DT, bool WHOLE_>
__device__ __forceinline__ void load_part(const uint8_t* p, int n, float (&f)[El<DT>::n]) {
  constexpr int N = El<DT>::n;
  if (WHOLE_ || n >= N) {
    Span<DT, WHOLE> s(0, N);
    unpack<DT>(load_vec<true>(p, s), f);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = i < n ? load_elem(p, DT, i) : 0.f;
  }
}
template <int DT, bool WHOLE_>
__device__ __forceinline__ void store_part(uint8_t* p, int n, const float (&f)[El<DT>::n]) {
  constexpr int N = El<DT>::n;
  if (WHOLE_ || n >= N) {
    Span<DT, WHOLE> s(0, N);
    store_vec(p, s, f);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < n) store_elem(p, DT, i, f[i]);
  }
}

// where a lane's columns are
struct At {
  int64_t row, tile;  // tile: of all rows
  int c, col, n;      // column of h, of gate in x, values that there are
  bool on;
  template <int N>
  __device__ __forceinline__ void init(const Args& g) {
    constexpr int LANES = 128 / N;
    tile = ((int64_t)blockIdx.x * THREADS + threadIdx.x) / LANES;
    on = tile < g.tiles;
    if (!on) tile = g.tiles - 1;  // its lanes walk along and write nothing
    const uint32_t q = (uint32_t)tile, r = g.by.row(q);
    row = r;
    c = (int)(q - r * (uint32_t)g.NT) * 128 + (int)(threadIdx.x % LANES) * N;
    n = min(max(g.I - c, 0), N);
    const int b = c / g.block;
    col = b * 2 * g.block + (c - b * g.block);
  }
};

template <int DT, bool W, bool KEEP>
__global__ void __launch_bounds__(THREADS) forward_kernel(Args g) {
  constexpr int N = El<DT>::n, LANES = 128 / N, E = El<DT>::bytes;
  At at;
  at.init<N>(g);
  const int n = at.on ? at.n : 0;
  const uint8_t* p = (const uint8_t*)g.x + at.row * g.ldx + (int64_t)at.col * E;
  float a[N] = {}, u[N] = {};
  if (n > 0) {
    load_part<DT, W>(p, n, a);
    load_part<DT, W>(p + (int64_t)g.block * E, n, u);
    float f[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const Sigmoid s = sigmoid<DT>(a[i]);
      f[i] = a[i] * s.near * u[i] * s.far;
    }
    store_part<DT, W>((uint8_t*)g.h + at.row * g.ldh + (int64_t)at.c * E, n, f);
  }
  if constexpr (KEEP) {
    uint32_t ma = 0, mu = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      ma = max(ma, finite_bits(a[i]));
      mu = max(mu, finite_bits(u[i]));
    }
    const uint32_t ba = kept_byte(tile_max<LANES>(ma)), bu = kept_byte(tile_max<LANES>(mu));
    if (!at.on) return;
    const float ia = kept_inverse(ba), iu = kept_inverse(bu);
    uint8_t* ca = g.kc + at.row * (2 * 128 * (int64_t)g.NT) + at.c;
    uint8_t* cu = ca + 128 * (int64_t)g.NT;
    const uint32_t a0 = kept_codes4(a[0], a[1], a[2], a[3], ia), u0 = kept_codes4(u[0], u[1], u[2], u[3], iu);
    if constexpr (N == 8) {
      store8_nt(ca, a0, kept_codes4(a[4 % N], a[5 % N], a[6 % N], a[7 % N], ia));
      store8_nt(cu, u0, kept_codes4(u[4 % N], u[5 % N], u[6 % N], u[7 % N], iu));
    } else {
      *reinterpret_cast<uint32_t*>(ca) = a0;
      *reinterpret_cast<uint32_t*>(cu) = u0;
    }
    if (threadIdx.x % LANES == 0) {
      uint8_t* e = g.ke + at.row * (2 * (int64_t)g.NT) + at.c / 128;
      e[0] = (uint8_t)ba;
      e[g.NT] = (uint8_t)bu;
    }
  }
}

template <int N>
__device__ __forceinline__ void load_codes(const uint8_t* p, float scale, float (&f)[N]) {
  uint32_t w[2];
  if constexpr (N == 8) {
    typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
    const u32x2 v = __builtin_nontemporal_load(reinterpret_cast<const u32x2*>(p));
    w[0] = v[0];
    w[1] = v[1];
  } else {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  }
#pragma unroll
  for (int h = 0; h < N / 4; ++h) {
    float v[4];
    kept_values4(w[h], scale, v);
#pragma unroll
    for (int i = 0; i < 4; ++i) f[4 * h + i] = v[i];
  }
}

template <int DT, bool W, bool KEEP>
__global__ void __launch_bounds__(THREADS) backward_kernel(Args g) {
  constexpr int N = El<DT>::n, E = El<DT>::bytes;
  At at;
  at.init<N>(g);
  const int n = at.n;
  if (!at.on || n == 0) return;
  float a[N], u[N], d[N];
  load_part<DT, W>((const uint8_t*)g.dh + at.row * g.lddh + (int64_t)at.c * E, n, d);
  if constexpr (KEEP) {
    const uint8_t* e = g.ke + at.row * (2 * (int64_t)g.NT) + at.c / 128;
    const uint8_t* p = g.kc + at.row * (2 * 128 * (int64_t)g.NT) + at.c;
    load_codes<N>(p, kept_scale(e[0]), a);
    load_codes<N>(p + 128 * (int64_t)g.NT, kept_scale(e[g.NT]), u);
  } else {
    const uint8_t* p = (const uint8_t*)g.x + at.row * g.ldx + (int64_t)at.col * E;
    load_part<DT, W>(p, n, a);
    load_part<DT, W>(p + (int64_t)g.block * E, n, u);
  }
  float da[N], du[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const Sigmoid s = sigmoid<DT>(a[i]);
    da[i] = d[i] * u[i] * (s.near * (1.0f + a[i] * s.rest)) * s.far;
    du[i] = d[i] * (a[i] * s.near) * s.far;
  }
  uint8_t* o = (uint8_t*)g.dx + at.row * g.lddx + (int64_t)at.col * E;
  store_part<DT, W>(o, n, da);
  store_part<DT, W>(o + (int64_t)g.block * E, n, du);
}

template <int DT, bool W>
static void launch_of(const Args& g, bool backward, hipStream_t st) {
  const unsigned n = (unsigned)cdiv(g.tiles * (128 / El<DT>::n), THREADS);
  if (backward) {
    if (g.kc) backward_kernel<DT, W, true><<<n, THREADS, 0, st>>>(g);
    else backward_kernel<DT, W, false><<<n, THREADS, 0, st>>>(g);
  } else {
    if (g.kc) forward_kernel<DT, W, true><<<n, THREADS, 0, st>>>(g);
    else forward_kernel<DT, W, false><<<n, THREADS, 0, st>>>(g);
  }
}
template <int DT>
static void launch_dt(const Args& g, bool backward, hipStream_t st) {
  g.I % El<DT>::n ? launch_of<DT, false>(g, backward, st) : launch_of<DT, true>(g, backward, st);
}
static int run(const char* fn, const Args& all, int dt, int64_t T, bool backward, void* stream) {
  const int64_t e = dtype_size(dt);
  return row_pieces(T, all.NT, [&](int64_t t, int64_t n) {
    Args g = all;
    g.ldx *= e; g.ldh *= e; g.lddh *= e; g.lddx *= e;
    g.tiles = n * g.NT;
    if (g.x) g.x = (const uint8_t*)g.x + t * g.ldx;
    if (g.h) g.h = (uint8_t*)g.h + t * g.ldh;
    if (g.dh) g.dh = (const uint8_t*)g.dh + t * g.lddh;
    if (g.dx) g.dx = (uint8_t*)g.dx + t * g.lddx;
    if (g.kc) g.kc += t * 2 * 128 * g.NT;
    if (g.ke) g.ke += t * 2 * g.NT;
    if (dt == NTLB_F32) launch_dt<DT_F32>(g, backward, as_stream(stream));
    else if (dt == NTLB_BF16) launch_dt<DT_BF16>(g, backward, as_stream(stream));
    else launch_dt<DT_F16>(g, backward, as_stream(stream));
    return check_launch(fn);
  });
}
static int begin(const char* fn, Args& g, int dt, int64_t T, int64_t I, int64_t block, const uint8_t* kept,
                 const uint8_t* kept_exp) {
  clear_error();
  if (!valid_dtype(dt)) return fail(NTLB_EINVAL, "%s: bad dtype %d", fn, dt);
  if (T < 0 || I < 1) return fail(NTLB_EINVAL, "%s: bad shape %lld x %lld", fn, (long long)T, (long long)I);
  if (I > ((int64_t)1 << 28)) return fail(NTLB_EUNSUPPORTED, "%s: rows of %lld columns", fn, (long long)I);
  if (block < 0 || (block && (block % 128 || I % block))) return fail(NTLB_EINVAL, "%s: blocks of %lld columns: 0, or a multiple of 128 that divides %lld", fn, (long long)block, (long long)I);
  if ((kept == nullptr) != (kept_exp == nullptr)) return fail(NTLB_EINVAL, "%s: kept codes and their exponents go together", fn);
  if (kept && !aligned(kept, 16)) return fail(NTLB_EINVAL, "%s: kept codes must be 16-byte aligned", fn);
  g = Args{};
  g.I = (int)I; g.NT = (int)cdiv(I, 128); g.by = TileRows(g.NT); g.block = (int)(block ? block : I);
  g.kc = const_cast<uint8_t*>(kept); g.ke = const_cast<uint8_t*>(kept_exp);
  return NTLB_OK;
}

}  // namespace swiglu
}  // namespace ntlb

using namespace ntlb;

extern "C" int ntlb_swiglu_rows(const void* x, int dtype, int64_t T, int64_t I, int64_t ldx, int64_t block, void* h,
                                int64_t ldh, uint8_t* kept, uint8_t* kept_exp, void* stream) {
  const char* fn = "ntlb_swiglu_rows";
  swiglu::Args g;
  if (int rc = swiglu::begin(fn, g, dtype, T, I, block, kept, kept_exp)) return rc;
  if (T == 0) return NTLB_OK;
  if (!x || (ldx != 0 && ldx < 2 * I)) return fail(NTLB_EINVAL, "%s: bad x", fn);
  if (!h || ldh < I) return fail(NTLB_EINVAL, "%s: bad h", fn);
  g.x = x; g.ldx = ldx; g.h = h; g.ldh = ldh;
  return swiglu::run(fn, g, dtype, T, false, stream);
}

extern "C" int ntlb_swiglu_rows_backward(const void* x, int dtype, int64_t T, int64_t I, int64_t ldx, int64_t block,
                                         const uint8_t* kept, const uint8_t* kept_exp, const void* dh, int64_t lddh,
                                         void* dx, int64_t lddx, void* stream) {
  const char* fn = "ntlb_swiglu_rows_backward";
  swiglu::Args g;
  if (int rc = swiglu::begin(fn, g, dtype, T, I, block, kept, kept_exp)) return rc;
  if (T == 0) return NTLB_OK;
  if ((x == nullptr) == (kept == nullptr)) return fail(NTLB_EINVAL, "%s: x, or kept codes and their exponents", fn);
  if (x && ldx != 0 && ldx < 2 * I) return fail(NTLB_EINVAL, "%s: bad x", fn);
  if (!dh || (lddh != 0 && lddh < I)) return fail(NTLB_EINVAL, "%s: bad dh", fn);
  if (!dx || lddx < 2 * I) return fail(NTLB_EINVAL, "%s: bad dx", fn);
  g.x = x; g.ldx = ldx; g.dh = dh; g.lddh = lddh; g.dx = dx; g.lddx = lddx;
  return swiglu::run(fn, g, dtype, T, true, stream);
}
