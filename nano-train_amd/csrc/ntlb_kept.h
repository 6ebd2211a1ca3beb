// Activations kept for the backward in 8 bits: the values of a row's tile (128
// columns, the last one shorter) over a power of two, as e4m3.
//   2^k: the smallest power with |x| <= 448 2^k over the tile's finite values, k >=
//   -126; one byte, k + 127, a tile.
// A scale of amax / 448 would use the range no better: e4m3 values are spaced by
// their own exponent, so a scale matters only to what falls below its normal numbers
// (2^-14 of the tile's largest value and less).  A power of two costs a quarter of
// the memory, and x 2^-k is exact, so a code is one rounding of x, at most 2^-4 of
// it.  Infinities and NaN are kept as NaN and take no part in the tile's largest.
#pragma once

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "ntlb_device.h"

namespace ntlb {

constexpr int KEPT_TILE = 128;

// Tiles of rows counted in one row after another, `per_row` a row: which row a tile is of, by a
// product (q / per_row = q mul >> (31 + l), exact for q < 2^31, where 2^l >= per_row).
struct TileRows {
  uint32_t per_row, mul, shift;
  __host__ TileRows(int64_t n = 1) : per_row((uint32_t)n), mul(0), shift(0) {
    int l = 0;
    while (((int64_t)1 << l) < n) ++l;
    if (n == 1) return;
    mul = (uint32_t)(((uint64_t)1 << (31 + l)) / (uint64_t)n + 1);
    shift = (uint32_t)(l - 1);
  }
  __device__ __forceinline__ uint32_t row(uint32_t tile) const { return per_row == 1 ? tile : __umulhi(tile, mul) >> shift; }
};
// Launches over tiles take at most this many: a tile has up to 32 threads, and a launch's
// are counted in 32 bits, 2^32 of them no longer.  f(first row, rows) for each piece of T rows.
constexpr int64_t MAX_TILES = (int64_t)1 << 26;
template <typename F>
inline int row_pieces(int64_t T, int64_t per_row, F f) {
  const int64_t step = std::max<int64_t>(1, MAX_TILES / per_row);
  for (int64_t t = 0; t < T; t += step)
    if (int rc = f(t, std::min(step, T - t))) return rc;
  return 0;
}

// The byte of a tile whose largest finite magnitude has these bits (1.75 2^8 = 448)
__device__ __forceinline__ uint32_t kept_byte(uint32_t amax_bits) {
  const int e = (int)(amax_bits >> 23) - 8 + ((amax_bits & 0x7FFFFFu) > 0x600000u);
  return (uint32_t)max(e, 1);
}
__device__ __forceinline__ float kept_scale(uint32_t byte) { return __uint_as_float(byte << 23); }
__device__ __forceinline__ float kept_inverse(uint32_t byte) { return __uint_as_float((254u - byte) << 23); }
__device__ __forceinline__ uint32_t finite_bits(float v) {
  const uint32_t b = abs_bits(v);
  return b < 0x7F800000u ? b : 0u;
}

// the codes of four values, first one in the lowest byte
__device__ __forceinline__ uint32_t kept_codes4(float a, float b, float c, float d, float inv) {
  uint32_t w = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(a * inv, b * inv, 0, false);
  w = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c * inv, d * inv, (int)w, true);
  const uint32_t bad = (abs_bits(a) >= 0x7F800000u ? 0x7Fu : 0u) | (abs_bits(b) >= 0x7F800000u ? 0x7F00u : 0u) |
                       (abs_bits(c) >= 0x7F800000u ? 0x7F0000u : 0u) | (abs_bits(d) >= 0x7F800000u ? 0x7F000000u : 0u);
  return w | bad;  // 0x7F and 0xFF are NaN
}

// the values of four codes
__device__ __forceinline__ void kept_values4(uint32_t w, float scale, float (&v)[4]) {
  typedef float f2 __attribute__((ext_vector_type(2)));
  const f2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
  v[0] = lo[0] * scale;
  v[1] = lo[1] * scale;
  v[2] = hi[0] * scale;
  v[3] = hi[1] * scale;
}

// the largest over the 16 or 32 neighbouring lanes that hold a tile
template <int LANES>
__device__ __forceinline__ uint32_t tile_max(uint32_t v) {
  static_assert(LANES == 16 || LANES == 32, "lanes of a tile");
  v = row16_max_u32(v);
  if constexpr (LANES == 32) v = max(v, (uint32_t)__shfl_xor((int)v, 16));
  return v;
}

}  // namespace ntlb
