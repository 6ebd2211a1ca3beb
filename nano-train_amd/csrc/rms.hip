// Root-mean-square norm of rows of s = x + residual [T, H], forward:
//   s = x + res (rounded to x's type; x itself without a residual)
//   r = 1 / sqrt(mean(s^2) + eps),  y = s r w
// y in x's type, or in 8 bits with a scale for each 128 columns, amax / 448 (int grid
// 127) as quant_tile_1x128 has it.  A code is y over its scale, in which r is no part:
// it is s w 448 / max|s w|, one division rounded once.  Values of 16 bits meet ties
// often (a value in 10,000 lies in the middle of two codes), and those are then
// decided as by exact arithmetic; with y rounded first they fell to either side.
// Optionally s is kept in 8 bits for
// the backward (ntlb_kept.h), which then needs no s.  The norm is that of the s
// that is stored.
//
// HBM-bound: a row is read once, stays in registers (ntlb_rows.h) and is written
// once (8192 x 7168 bf16 with a residual: 85 us, 5.5 TB/s; with codes kept 99; to codes 80).  To
// codes without a residual the arithmetic takes as long (49 us, 3.6 TB/s).  Statistics
// are fp32.  A tile of 128 columns lies in 16 (fp32: 32) lanes
// next to each other, so its largest magnitude is a reduction within the wave.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "ntlb_device.h"
#include "ntlb_host.h"
#include "ntlb_kept.h"
#include "ntlb_quant8.h"
#include "ntlb_rms.h"
#include "ntlb_splitk.h"

namespace ntlb {
namespace rms {

constexpr int OUT_VALUES = 0, OUT_KEEP = 1, OUT_CODES = 2;

// N codes (low bytes first in lo, then hi) of vector c0 / N of a row of `cols`
// stored columns; `first` of them belong to the vector before (RAGGED)
template <int N, int MODE>
__device__ __forceinline__ void store_codes(uint8_t* row, int c0, int cols, int first, uint32_t lo, uint32_t hi) {
  uint64_t v = ((uint64_t)hi << 32) | lo;
  if constexpr (MODE == RAGGED) v = first < N ? v >> (8 * first) : 0;
  if (c0 >= cols) return;
  if constexpr (N == 8)
    store8_nt(row + c0, (uint32_t)v, (uint32_t)(v >> 32));
  else
    *reinterpret_cast<uint32_t*>(row + c0) = (uint32_t)v;
}

template <int DT, int RT, int VPT, int MODE, bool RES, int OUT>
__global__ void __launch_bounds__(block_threads<RT>()) forward_kernel(Forward g) {
  constexpr int N = El<DT>::n, ROWS = block_threads<RT>() / RT, LANES = 128 / N;
  static_assert(RT >= LANES, "a tile of 128 columns is one row's");
  __shared__ float red[2][RT > 64 ? RT / 64 : 1];
  const int t = threadIdx.x % RT, H = g.H;
  const int64_t stride = (int64_t)gridDim.x * ROWS;
  int64_t row = (int64_t)blockIdx.x * ROWS + row_of_block<RT>();
  const float inv = 1.0f / (float)H;
  float w[VPT][N];
  load_weights<DT, RT, VPT, MODE>(g.w, g.w_dtype, t, H, 1.0f, w);
  Raw nx[VPT], nr[VPT];
  auto fetch = [&](int64_t r) {
    const uint8_t* p = (const uint8_t*)g.x + r * g.ldx;
    const uint8_t* q = (const uint8_t*)g.res + r * g.ldr;
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      const Span<DT, MODE> sp(t + v * RT, H);
      nx[v] = load_vec<true>(p, sp);
      if constexpr (RES) nr[v] = load_vec<true>(q, sp);
    }
  };
  if (row < g.T) fetch(row);
  for (int buf = 0; row < g.T; row += stride, buf ^= 1) {
    Raw x[VPT];
    if constexpr (RES) {
      uint8_t* sr = (uint8_t*)g.s + row * g.lds;
#pragma unroll
      for (int v = 0; v < VPT; ++v) {
        float a[N], b[N];
        unpack<DT>(nx[v], a);
        unpack<DT>(nr[v], b);
#pragma unroll
        for (int i = 0; i < N; ++i) a[i] += b[i];
        x[v] = pack<DT>(a);
      }
#pragma unroll
      for (int v = 0; v < VPT; ++v) store_raw<DT, MODE>(sr, Span<DT, MODE>(t + v * RT, H), x[v]);
    } else {
#pragma unroll
      for (int v = 0; v < VPT; ++v) x[v] = nx[v];
    }
    fetch(min<int64_t>(row + stride, g.T - 1));  // past the end: the last row again
    float q[1] = {0.f};
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      const Span<DT, MODE> sp(t + v * RT, H);
      float f[N];
      unpack<DT>(x[v], f);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float d = sp.own(i) ? f[i] : 0.f;
        q[0] += d * d;
      }
    }
    row_sum<RT, 1>(q, red[buf]);
    const float r = 1.0f / sqrtf(q[0] * inv + g.eps);
    if (OUT != OUT_CODES && g.rstd && t == 0) g.rstd[row] = r;
    // r = r1 r2, r2 a power of two
    const uint32_t rbits = __float_as_uint(r);
    const bool usual = rbits >= 0x00800000u && rbits < 0x7F800000u;
    const float r2 = __uint_as_float(rbits & 0x7F800000u), r1 = __uint_as_float((rbits & 0x007FFFFFu) | 0x3F800000u);
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
      const int c0 = (t + v * RT) * N;
      // a wave past the row's last tile has no codes (8192 x 5120 bf16: 57 us with their
      // arithmetic, 41 without)
      if (OUT != OUT_VALUES && VPT > 1 && __builtin_amdgcn_readfirstlane(c0) >= (OUT == OUT_KEEP ? (int)g.ldk : (int)g.ldy)) continue;
      const Span<DT, MODE> sp(t + v * RT, H);
      float f[N];
      renew(x[v], r);
      unpack<DT>(x[v], f);
      if constexpr (OUT == OUT_KEEP) {
        float k[N];
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) {
          k[i] = sp.own(i) ? f[i] : 0.f;
          m = max(m, finite_bits(k[i]));
        }
        const uint32_t byte = kept_byte(tile_max<LANES>(m));
        const float kinv = kept_inverse(byte);
        const uint32_t lo = kept_codes4(k[0], k[1], k[2], k[3], kinv);
        const uint32_t hi = N == 8 ? kept_codes4(k[4 % N], k[5 % N], k[6 % N], k[7 % N], kinv) : 0u;
        store_codes<N, MODE>(g.kc + row * g.ldk, c0, (int)g.ldk, sp.first, lo, hi);
        if (t % LANES == 0 && c0 < H) g.ke[row * (g.ldk / KEPT_TILE) + c0 / KEPT_TILE] = (uint8_t)byte;
      }
      if constexpr (OUT != OUT_CODES) {
#pragma unroll
        for (int i = 0; i < N; ++i) f[i] = f[i] * r * w[v][i];
        store_vec((uint8_t*)g.y + row * g.ldy, sp, f);
      } else {
        // of p = s w 2^e, exact but for the weight's factor; r itself enters the scale only
        float p[N];
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) {
          p[i] = sp.own(i) ? f[i] * r2 * w[v][i] : 0.f;
          m = max(m, abs_bits(p[i]));
        }
        m = tile_max<LANES>(m);
        float div = __uint_as_float(m), scale = div * r1 / g.qmax;
        if (usual && m >= 0x1A000000u && m <= 0x71800000u) {  // 2^-75 .. 2^100
#pragma unroll
          for (int i = 0; i < N; ++i) p[i] *= g.qmax;
        } else {  // zeros, what is not finite, magnitudes that products might not hold: y and its scale as they are
          m = 0;
#pragma unroll
          for (int i = 0; i < N; ++i) {
            p[i] = sp.own(i) ? f[i] * r * w[v][i] : 0.f;
            m = max(m, abs_bits(p[i]));
          }
          m = tile_max<LANES>(m);
          div = scale = scale_from_amax_bits(m, g.qmax, SCALE_AFTER_DIVIDE);
        }
        const float rs = fast_div_ok<false>(m) ? 1.0f / div : 1.0f;
        uint32_t rb[N] = {}, lo, hi;
        float qv[N];
        if (g.grid == GRID_E4M3)
          quant8_tile_rs<GRID_E4M3, false, false, N>(p, m, div, rs, g.qmax, rb, lo, hi, qv);
        else
          quant8_tile_rs<GRID_INT, false, false, N>(p, m, div, rs, g.qmax, rb, lo, hi, qv);
        store_codes<N, MODE>((uint8_t*)g.y + row * g.ldy, c0, (int)g.ldy, sp.first, lo, hi);
        if (t % LANES == 0 && c0 < H) g.scales[row * g.s_row + (int64_t)(c0 / 128) * g.s_col] = scale;
        if (m > 0x7F800000u && g.nan_rows) g.nan_rows[row] = 1;
      }
    }
  }
}

// Threads and vectors a row, and workgroups a compute unit, as layer norm's forward; rows of up
// to 16 or 32 vectors share a wave (262144 x 64 bf16 16 us, by a wave a row 55; codes 27, 167)
struct Shape {
  int rt, vpt, per_cu;
};
static Shape shape_of(int dt, int64_t nv) {
  if (nv <= 16 && dt != NTLB_F32) return {16, 1, 8};
  if (nv <= 32) return {32, 1, 8};
  if (nv <= 64) return {64, 1, 4};
  if (nv <= 128) return {64, 2, 4};
  if (nv <= 256) return {64, 4, 4};
  if (nv <= 512) return {128, 4, 8};
  if (nv <= 1024) return {256, 4, 3};
  if (nv <= 2048) return {512, 4, 2};
  return {512, 8, 1};
}

template <int DT, int MODE, bool RES, int OUT>
static bool launch(const Shape& s, const Forward& g, int64_t n, hipStream_t st) {
#define NTLB_CASE(RT, VPT)                                                                                            \
  if (s.rt == RT && s.vpt == VPT)                                                                                     \
    return forward_kernel<DT, RT, VPT, MODE, RES, OUT><<<(unsigned)n, block_threads<RT>(), 0, st>>>(g), true;
  if constexpr (DT != DT_F32) NTLB_CASE(16, 1)
  if constexpr (DT == DT_F32 || MODE != TINY) NTLB_CASE(32, 1)
  if constexpr (MODE != TINY) {
    NTLB_CASE(64, 1) NTLB_CASE(64, 2) NTLB_CASE(64, 4) NTLB_CASE(128, 4) NTLB_CASE(256, 4) NTLB_CASE(512, 4)
    if constexpr (DT == DT_F32) NTLB_CASE(512, 8)
  }
#undef NTLB_CASE
  return false;
}
template <int DT, int MODE>
static bool pick(const Shape& s, const Forward& g, int64_t n, int out, hipStream_t st) {
  if (g.res) {
    if (out == OUT_VALUES) return launch<DT, MODE, true, OUT_VALUES>(s, g, n, st);
    if (out == OUT_KEEP) return launch<DT, MODE, true, OUT_KEEP>(s, g, n, st);
    return launch<DT, MODE, true, OUT_CODES>(s, g, n, st);
  }
  if (out == OUT_VALUES) return launch<DT, MODE, false, OUT_VALUES>(s, g, n, st);
  if (out == OUT_KEEP) return launch<DT, MODE, false, OUT_KEEP>(s, g, n, st);
  return launch<DT, MODE, false, OUT_CODES>(s, g, n, st);
}
template <int DT>
static bool pick_mode(const Shape& s, const Forward& g, int64_t n, int out, hipStream_t st) {
  if (g.H < El<DT>::n) return pick<DT, TINY>(s, g, n, out, st);
  return g.H % El<DT>::n ? pick<DT, RAGGED>(s, g, n, out, st) : pick<DT, WHOLE>(s, g, n, out, st);
}
static int run(const char* fn, int dt, const Forward& g, int out, void* stream) {
  const int64_t nv = cdiv((int64_t)g.H * dtype_size(dt), 16);
  const Shape s = shape_of(dt, nv);
  const int64_t n = std::max<int64_t>(1, std::min(cdiv(g.T, s.rt <= 64 ? 256 / s.rt : 1), (int64_t)split_device_cus() * s.per_cu));
  hipStream_t st = as_stream(stream);
  const bool ok = dt == NTLB_F32 ? pick_mode<DT_F32>(s, g, n, out, st)
                  : dt == NTLB_BF16 ? pick_mode<DT_BF16>(s, g, n, out, st)
                                    : pick_mode<DT_F16>(s, g, n, out, st);
  if (!ok) return fail(NTLB_EUNSUPPORTED, "%s: no kernel for %d columns", fn, g.H);
  return check_launch(fn);
}

int check(const char* fn, const void* x, int dt, int64_t T, int64_t H, int64_t ldx, int wdt) {
  if (!valid_dtype(dt) || !valid_dtype(wdt)) return fail(NTLB_EINVAL, "%s: bad dtype %d / %d", fn, dt, wdt);
  if (T < 0 || H < 1) return fail(NTLB_EINVAL, "%s: bad shape %lld x %lld", fn, (long long)T, (long long)H);
  if (H > MAX_H) return fail(NTLB_EUNSUPPORTED, "%s: rows of %lld elements (at most %d)", fn, (long long)H, MAX_H);
  if (T > 0 && !x) return fail(NTLB_EINVAL, "%s: NULL x", fn);
  // rows may repeat (pitch 0) in an input, not overlap in part
  if (ldx != 0 && ldx < H) return fail(NTLB_EINVAL, "%s: row pitch %lld below %lld", fn, (long long)ldx, (long long)H);
  return NTLB_OK;
}
// the arguments both forwards share
static int begin(const char* fn, Forward& g, const void* x, int dt, int64_t T, int64_t H, int64_t ldx, const void* res,
                 int64_t ldr, const void* w, int wdt, float eps, void* s, int64_t lds) {
  clear_error();
  if (int rc = check(fn, x, dt, T, H, ldx, wdt)) return rc;
  if (!(eps >= 0.0f)) return fail(NTLB_EINVAL, "%s: eps must not be negative", fn);
  if (res && ldr != 0 && ldr < H) return fail(NTLB_EINVAL, "%s: the residual's row pitch %lld below %lld", fn, (long long)ldr, (long long)H);
  if (T > 0 && (res == nullptr) != (s == nullptr)) return fail(NTLB_EINVAL, "%s: a residual and its sum go together", fn);
  if (s && lds < H) return fail(NTLB_EINVAL, "%s: the sum's row pitch %lld below %lld", fn, (long long)lds, (long long)H);
  const int64_t e = dtype_size(dt);
  g = Forward{};
  g.x = x; g.ldx = ldx * e; g.res = res; g.ldr = ldr * e; g.w = w; g.w_dtype = wdt; g.T = T; g.H = (int)H; g.eps = eps;
  g.s = s; g.lds = lds * e;
  return NTLB_OK;
}

}  // namespace rms
}  // namespace ntlb

using namespace ntlb;

extern "C" int ntlb_rms_norm_forward(const void* x, int x_dtype, int64_t T, int64_t H, int64_t ldx, const void* res,
                                     int64_t ldr, const void* w, int w_dtype, float eps, void* s, int64_t lds, void* y,
                                     int64_t ldy, float* rstd, uint8_t* kept, uint8_t* kept_exp, void* stream) {
  const char* fn = "ntlb_rms_norm_forward";
  rms::Forward g;
  if (int rc = rms::begin(fn, g, x, x_dtype, T, H, ldx, res, ldr, w, w_dtype, eps, s, lds)) return rc;
  if ((kept == nullptr) != (kept_exp == nullptr)) return fail(NTLB_EINVAL, "%s: kept codes and their exponents go together", fn);
  if (T == 0) return NTLB_OK;
  if (!y || ldy < H) return fail(NTLB_EINVAL, "%s: bad y", fn);
  if (kept && !aligned(kept, 16)) return fail(NTLB_EINVAL, "%s: kept codes must be 16-byte aligned", fn);
  g.y = y; g.ldy = ldy * dtype_size(x_dtype); g.rstd = rstd; g.kc = kept; g.ke = kept_exp; g.ldk = cdiv(H, KEPT_TILE) * KEPT_TILE;
  return rms::run(fn, x_dtype, g, kept ? rms::OUT_KEEP : rms::OUT_VALUES, stream);
}

extern "C" int ntlb_rms_norm_quant(const void* x, int x_dtype, int64_t T, int64_t H, int64_t ldx, const void* res,
                                   int64_t ldr, const void* w, int w_dtype, float eps, void* s, int64_t lds, int grid,
                                   uint8_t* codes, int64_t ldc, float* scales, int64_t s_row, int64_t s_col,
                                   int32_t* nan_rows, void* stream) {
  const char* fn = "ntlb_rms_norm_quant";
  rms::Forward g;
  if (int rc = rms::begin(fn, g, x, x_dtype, T, H, ldx, res, ldr, w, w_dtype, eps, s, lds)) return rc;
  if (grid != GRID_INT && grid != GRID_E4M3) return fail(NTLB_EINVAL, "%s: bad grid %d", fn, grid);
  if (T == 0) return NTLB_OK;
  if (!codes || !aligned(codes, 16) || ldc != cdiv(H, 128) * 128) return fail(NTLB_EINVAL, "%s: codes must be 16-byte aligned rows of %lld bytes", fn, (long long)(cdiv(H, 128) * 128));
  if (!scales || s_row < 1 || s_col < 1) return fail(NTLB_EINVAL, "%s: bad scales", fn);
  g.y = codes; g.ldy = ldc; g.grid = grid; g.qmax = grid == GRID_E4M3 ? 448.0f : 127.0f;
  g.scales = scales; g.s_row = s_row; g.s_col = s_col; g.nan_rows = nan_rows;
  return rms::run(fn, x_dtype, g, rms::OUT_CODES, stream);
}
