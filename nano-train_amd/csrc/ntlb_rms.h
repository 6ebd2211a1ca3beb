// Root-mean-square norm: what its forward (rms.hip) and backward (rms_bwd.hip) share.
#pragma once

#include <hip/hip_runtime.h>

#include "ntlb_rows.h"

namespace ntlb {
namespace rms {

using namespace rows;

constexpr int MAX_H = 16384;

struct Forward {
  const void* x;
  int64_t ldx;  // in bytes, as the others
  const void* res;
  int64_t ldr;
  const void* w;
  int w_dtype;
  int64_t T;
  int H;
  float eps;
  void* s;
  int64_t lds;
  void* y;  // values or codes
  int64_t ldy;
  float* rstd;
  uint8_t* kc;  // kept codes, rows of ldk bytes, and their bytes of exponents, ldk / 128 a row
  uint8_t* ke;
  int64_t ldk;
  int grid;  // codes
  float qmax;
  float* scales;
  int64_t s_row, s_col;
  int32_t* nan_rows;
};

int check(const char* fn, const void* x, int dt, int64_t T, int64_t H, int64_t ldx, int wdt);

}  // namespace rms
}  // namespace ntlb
