// Root-mean-square norm, backward.  With xh = s r (r from the forward, s as stored or
// as 8 bits kept it) and t = dy w:
//   ds = r (t - xh mean(t xh)) + what comes in for s,  dw = sum over rows of dy xh
// ds is the gradient of x and of the residual.
//
// HBM-bound: s (or one byte a value), dy and s's gradient in, ds out, a row in
// registers as in the forward; one reduction a row.  dw's column sums stay in
// registers over a workgroup's rows and go out as one partial row, which a second
// kernel sums in a fixed order (8192 x 7168 bf16 with s's gradient: 81 us, 5.8 TB/s; s of 8
// bits 75; the sum 5)
#include <hip/hip_runtime.h>

#include <algorithm>

#include "ntlb_device.h"
#include "ntlb_host.h"
#include "ntlb_kept.h"
#include "ntlb_rms.h"
#include "ntlb_splitk.h"

namespace ntlb {
namespace rms {

struct Backward {
  const void* s;  // or kept codes and exponents
  int64_t lds;    // in bytes, as the others
  const uint8_t* ke;
  const void* dy;
  int64_t lddy;
  const void* ds;
  int64_t ldds;
  const float* rstd;
  const void* w;
  int w_dtype;
  int64_t T;
  int H;
  void* dx;
  int64_t lddx;
  float* part;  // [workgroups][H]
};

// s of a vector as it is read: values, or codes and the exponents of the two tiles
// that a ragged row's last vector may touch
template <int DT, int MODE, bool KEEP>
struct Held {
  static constexpr int N = El<DT>::n;
  Raw r;
  uint32_t ea, eb;
  __device__ __forceinline__ void load(const Backward& g, int64_t row, const Span<DT, MODE>& sp) {
    const uint8_t* p = (const uint8_t*)g.s + row * g.lds;
    if constexpr (!KEEP) {
      r = load_vec<true>(p, sp);
    } else {
      const uint8_t* e = g.ke + row * (g.lds / KEPT_TILE);
      r.w[2] = r.w[3] = 0;
      if constexpr (MODE == WHOLE) {
        if constexpr (N == 8) {
          const uint2 v = *reinterpret_cast<const uint2*>(p + sp.c);
          r.w[0] = v.x;
          r.w[1] = v.y;
        } else {
          r.w[0] = *reinterpret_cast<const uint32_t*>(p + sp.c);
          r.w[1] = 0;
        }
        ea = eb = e[sp.c / KEPT_TILE];
      } else if constexpr (MODE == RAGGED) {
        typedef uint32_t u32_1 __attribute__((aligned(1)));
        r.w[0] = *reinterpret_cast<const u32_1*>(p + sp.c);
        r.w[1] = N == 8 ? *reinterpret_cast<const u32_1*>(p + sp.c + 4) : 0u;
        ea = e[sp.c / KEPT_TILE];
        eb = e[(sp.c + N - 1) / KEPT_TILE];
      } else {
        r.w[0] = *reinterpret_cast<const uint32_t*>(p);  // a row has 128 codes
        r.w[1] = N == 8 ? *reinterpret_cast<const uint32_t*>(p + 4) : 0u;
        ea = eb = e[0];
      }
    }
  }
  __device__ __forceinline__ void values(const Span<DT, MODE>& sp, float (&f)[N]) const {
    if constexpr (!KEEP) {
      unpack<DT>(r, f);
    } else {
      const float a = kept_scale(ea), b = kept_scale(eb);
      const int edge = KEPT_TILE - sp.c % KEPT_TILE;  // the first element of the next tile
#pragma unroll
      for (int h = 0; h < N / 4; ++h) {
        float v[4];
        kept_values4(r.w[h], 1.0f, v);
#pragma unroll
        for (int i = 0; i < 4; ++i) f[4 * h + i] = v[i] * (MODE == RAGGED && 4 * h + i >= edge ? b : a);
      }
    }
  }
};

template <int DT, int RT, int VPT, int MODE, bool DS, bool KEEP>
__global__ void __launch_bounds__(block_threads<RT>()) backward_kernel(Backward g) {
  constexpr int N = El<DT>::n, BT = block_threads<RT>(), ROWS = BT / RT;
  __shared__ float red[2][RT > 64 ? RT / 64 : 1];
  const int t = threadIdx.x % RT, H = g.H;
  const int64_t stride = (int64_t)gridDim.x * ROWS;
  int64_t row = (int64_t)blockIdx.x * ROWS + row_of_block<RT>();
  const float inv = 1.0f / (float)H;
  float w[VPT][N], aw[VPT][N];
  load_weights<DT, RT, VPT, MODE>(g.w, g.w_dtype, t, H, 1.0f, w);
#pragma unroll
  for (int v = 0; v < VPT; ++v)
#pragma unroll
    for (int i = 0; i < N; ++i) aw[v][i] = 0.f;
  Held<DT, MODE, KEEP> nx[VPT];
  Raw nd[VPT], ns[VPT];
  float nr = 0.f;
  auto fetch = [&](int64_t r) {
    const uint8_t* d = (const uint8_t*)g.dy + r * g.lddy;
    const uint8_t* q = (const uint8_t*)g.ds + r * g.ldds;
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      const Span<DT, MODE> sp(t + v * RT, H);
      nx[v].load(g, r, sp);
      nd[v] = load_vec<true>(d, sp);
      if constexpr (DS) ns[v] = load_vec<true>(q, sp);
    }
    nr = g.rstd[r];
  };
  // eight vectors a thread leave no registers for a row in flight beside this one
  constexpr bool AHEAD = VPT < 8;
  if (AHEAD && row < g.T) fetch(row);
#pragma unroll 1
  for (int buf = 0; row < g.T; row += stride, buf ^= 1) {
    if (!AHEAD) fetch(row);
    Held<DT, MODE, KEEP> x[VPT];
    Raw d[VPT], q[VPT];
    const float r = nr;
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      x[v] = nx[v];
      d[v] = nd[v];
      if constexpr (DS) q[v] = ns[v];
    }
    if (AHEAD) fetch(min<int64_t>(row + stride, g.T - 1));  // past the end: the last row again
    float s[1] = {0.f};
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      float f[N], e[N];
      const Span<DT, MODE> sp(t + v * RT, H);
      x[v].values(sp, f);
      unpack<DT>(d[v], e);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float xh = f[i] * r, de = sp.own(i) ? e[i] : 0.f;
        aw[v][i] += de * xh;
        s[0] += de * w[v][i] * xh;
      }
      // added here and now: dy and xh are not kept for it
#pragma unroll
      for (int i = 0; i < N; ++i) asm volatile("" : "+v"(aw[v][i]));
    }
    row_sum<RT, 1>(s, red[buf]);
    const float m = s[0] * inv;
    uint8_t* dp = (uint8_t*)g.dx + row * g.lddx;
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      float f[N], e[N];
      const Span<DT, MODE> sp(t + v * RT, H);
      renew(x[v].r, m);
      renew(d[v], m);
      x[v].values(sp, f);
      unpack<DT>(d[v], e);
#pragma unroll
      for (int i = 0; i < N; ++i) f[i] = r * (e[i] * w[v][i] - f[i] * r * m);
      if constexpr (DS) {
        unpack<DT>(q[v], e);
#pragma unroll
        for (int i = 0; i < N; ++i) f[i] += e[i];
      }
      store_vec(dp, sp, f);
    }
  }
  float* pw = g.part + (int64_t)blockIdx.x * H;
  if constexpr (ROWS == 1) {
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      const Span<DT, MODE> sp(t + v * RT, H);
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (sp.own(i)) pw[sp.c + i] = aw[v][i];
    }
  } else {
    // the workgroup's row walkers, summed in their order
    constexpr int W = RT * VPT * N;
    __shared__ float sum[ROWS][W];
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      const Span<DT, MODE> sp(t + v * RT, H);
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (sp.own(i)) sum[threadIdx.x / RT][sp.c + i] = aw[v][i];
    }
    __syncthreads();
    for (int c = threadIdx.x; c < H; c += BT) {
      float a = sum[0][c];
#pragma unroll
      for (int q = 1; q < ROWS; ++q) a += sum[q][c];
      pw[c] = a;
    }
  }
}

// Threads and vectors a row, and workgroups a compute unit, as layer norm's backward but for
// rows of 513 to 1024 vectors (8192 x 7168 bf16 with a residual, s kept: 512 x 2 75 us, 256 x
// 4 79, 1024 x 1 81) and of up to 32, which share a wave (262144 x 64 bf16 29 us, by a wave a
// row 110)
struct Shape {
  int rt, vpt, per_cu;
};
static Shape shape_of(int dt, int64_t H) {
  const int64_t nv = cdiv(H * dtype_size(dt), 16);
  if (nv <= 16 && dt != NTLB_F32) return {16, 1, 4};
  if (nv <= 32) return {32, 1, 4};
  if (nv <= 64) return {64, 1, 2};
  if (nv <= 128) return {128, 1, 4};
  if (nv <= 256) return {256, 1, 2};
  if (nv <= 512) return {512, 1, 1};
  if (nv <= 1024) return {512, 2, 1};
  if (nv <= 2048) return {512, 4, 1};
  return {512, 8, 1};
}
static int64_t groups(const Shape& s, int64_t T) {
  return std::max<int64_t>(1, std::min(cdiv(T, s.rt <= 64 ? 256 / s.rt : 1), (int64_t)split_device_cus() * s.per_cu));
}

template <int DT, int MODE, bool DS, bool KEEP>
static bool launch(const Shape& s, const Backward& g, int64_t n, hipStream_t st) {
#define NTLB_CASE(RT, VPT)                                                                                            \
  if (s.rt == RT && s.vpt == VPT)                                                                                     \
    return backward_kernel<DT, RT, VPT, MODE, DS, KEEP><<<(unsigned)n, block_threads<RT>(), 0, st>>>(g), true;
  if constexpr (DT != DT_F32) NTLB_CASE(16, 1)
  if constexpr (DT == DT_F32 || MODE != TINY) NTLB_CASE(32, 1)
  if constexpr (MODE != TINY) {
    NTLB_CASE(64, 1) NTLB_CASE(128, 1) NTLB_CASE(256, 1) NTLB_CASE(512, 1) NTLB_CASE(512, 2) NTLB_CASE(512, 4)
    if constexpr (DT == DT_F32) NTLB_CASE(512, 8)
  }
#undef NTLB_CASE
  return false;
}
template <int DT, int MODE>
static bool pick(const Shape& s, const Backward& g, int64_t n, hipStream_t st) {
  if (g.ds) return g.ke ? launch<DT, MODE, true, true>(s, g, n, st) : launch<DT, MODE, true, false>(s, g, n, st);
  return g.ke ? launch<DT, MODE, false, true>(s, g, n, st) : launch<DT, MODE, false, false>(s, g, n, st);
}
template <int DT>
static bool pick_mode(const Shape& s, const Backward& g, int64_t n, hipStream_t st) {
  if (g.H < El<DT>::n) return pick<DT, TINY>(s, g, n, st);
  return g.H % El<DT>::n ? pick<DT, RAGGED>(s, g, n, st) : pick<DT, WHOLE>(s, g, n, st);
}

}  // namespace rms
}  // namespace ntlb

using namespace ntlb;

extern "C" int64_t ntlb_rms_norm_workspace_bytes(int x_dtype, int64_t T, int64_t H) {
  if (!valid_dtype(x_dtype) || T < 1 || H < 1 || H > rms::MAX_H) return 0;
  return rms::groups(rms::shape_of(x_dtype, H), T) * H * 4;
}

extern "C" int ntlb_rms_norm_backward(const void* s, int dtype, int64_t T, int64_t H, int64_t lds, const uint8_t* kept,
                                      const uint8_t* kept_exp, const void* dy, int64_t lddy, const void* ds,
                                      int64_t ldds, const float* rstd, const void* w, int w_dtype, void* dx,
                                      int64_t lddx, void* dw, void* workspace, int64_t ws_bytes, void* stream) {
  const char* fn = "ntlb_rms_norm_backward";
  clear_error();
  if ((kept == nullptr) != (kept_exp == nullptr) || (kept && s)) return fail(NTLB_EINVAL, "%s: s, or kept codes and their exponents", fn);
  const int64_t ldk = cdiv(H, KEPT_TILE) * KEPT_TILE;
  if (int rc = rms::check(fn, kept ? kept : s, dtype, T, H, kept ? ldk : lds, w_dtype)) return rc;
  if (kept && !aligned(kept, 16)) return fail(NTLB_EINVAL, "%s: kept codes must be 16-byte aligned", fn);
  if (T > 0 && (!dy || !rstd || !dx)) return fail(NTLB_EINVAL, "%s: NULL pointer", fn);
  if (lddy != 0 && lddy < H) return fail(NTLB_EINVAL, "%s: dy's row pitch %lld below %lld", fn, (long long)lddy, (long long)H);
  if (ds && ldds != 0 && ldds < H) return fail(NTLB_EINVAL, "%s: ds' row pitch %lld below %lld", fn, (long long)ldds, (long long)H);
  if (dx && lddx < H) return fail(NTLB_EINVAL, "%s: dx' row pitch %lld below %lld", fn, (long long)lddx, (long long)H);
  const rms::Shape sh = rms::shape_of(dtype, H);
  const int64_t n = T > 0 ? rms::groups(sh, T) : 0, need = n * H * 4;
  if (need > ws_bytes || (need && (!workspace || !aligned(workspace, 4)))) return fail(NTLB_EINVAL, "%s: workspace of %lld bytes, %lld needed", fn, (long long)ws_bytes, (long long)need);
  hipStream_t st = as_stream(stream);
  if (T > 0) {
    const int64_t e = dtype_size(dtype);
    rms::Backward g{};
    g.s = kept ? kept : s; g.lds = kept ? ldk : lds * e; g.ke = kept_exp; g.dy = dy; g.lddy = lddy * e; g.ds = ds; g.ldds = ldds * e;
    g.rstd = rstd; g.w = w; g.w_dtype = w_dtype; g.T = T; g.H = (int)H; g.dx = dx; g.lddx = lddx * e; g.part = (float*)workspace;
    const bool ok = dtype == NTLB_F32 ? rms::pick_mode<DT_F32>(sh, g, n, st)
                    : dtype == NTLB_BF16 ? rms::pick_mode<DT_BF16>(sh, g, n, st)
                                         : rms::pick_mode<DT_F16>(sh, g, n, st);
    if (!ok) return fail(NTLB_EUNSUPPORTED, "%s: no kernel for %lld columns", fn, (long long)H);
    if (int rc = check_launch(fn)) return rc;
  }
  if (dw) {
    const dim3 grd((unsigned)cdiv(H, rms::FIN_COLS), 1), blk(rms::FIN_COLS / 2 * rms::FIN_WALK);
    rms::finish_kernel<<<grd, blk, 0, st>>>((const float*)workspace, (int)n, (int)H, dw, nullptr, w_dtype);
    return check_launch(fn);
  }
  return NTLB_OK;
}
