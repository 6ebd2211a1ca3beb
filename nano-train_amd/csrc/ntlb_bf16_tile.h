// A bf16 product's output tile of 256 x 256 or 128 x 128: copies of its operands
// global -> LDS, fragments from there, the K loop, and the store of rows (xent.hip,
// grouped.hip).
#pragma once

#include <hip/hip_runtime.h>

#include <type_traits>

#include "ntlb_device.h"

namespace ntlb {
namespace tile {

typedef int v8i __attribute__((ext_vector_type(8)));
typedef int v4i __attribute__((ext_vector_type(4)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) void* lds_ptr_t;
typedef __attribute__((address_space(3))) v4s* lds_v4s_ptr;

// the user's rows begin at any element
typedef uint32_t u32x4_2 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x2_2 __attribute__((ext_vector_type(2), aligned(2)));

constexpr int ROWB = 128, KSTEP = 64;  // bytes and values of a row's K step

// LDS stages and fragments as in gemm_dq.hip: row-major [256][128 bytes] with
// 16-byte chunks XOR-swizzled by row, or [64 contraction rows][256] as stored,
// read transposed
__device__ __forceinline__ int sw_perm(int r) { return (r & 7) ^ ((r >> 3) & 1); }
__device__ __forceinline__ int sw(int r, int c) { return r * ROWB + ((c ^ sw_perm(r)) << 4); }
__device__ __forceinline__ int tr_perm(int k) { return (2 * (k & 3)) ^ (8 * ((k >> 4) & 1)); }

// Where a lane's part of a fragment of 16 operand rows from row0 lies in a
// stage.  By rows: row0 + lane % 16, bytes 32 g .. of its K step (g = lane / 16),
// the swizzle the same for all row0.  Transposed: contraction rows 16 g + 4 h + j;
// row0's chunk is XORed into the address.
template <bool TR, int D>
struct FragAt {
  uint32_t lo, hi;
  __device__ __forceinline__ explicit FragAt(int row0, int lane) {
    const int g = lane >> 4;
    if constexpr (!TR) {
      const int r = row0 + (lane & 15);
      lo = sw(r, 2 * g);
      hi = sw(r, 2 * g + 1);
    } else {
      const int j = (lane >> 2) & 3, q = lane & 3, k = 16 * g + j;
      lo = k * (2 * D) + ((((row0 >> 3) + (q >> 1)) ^ tr_perm(k)) << 4) + (q & 1) * 8;
    }
  }
  // the address is formed again in every step: hoisted for all row groups, they
  // would take more registers than there are
  __device__ __forceinline__ void renew() {
    if constexpr (TR) asm volatile("" : "+v"(lo));
  }
  // likewise where the stages are many: a sum for each of them would be kept
  __device__ __forceinline__ void anew() {
    if constexpr (TR) asm volatile("" : "+v"(lo));
    else asm volatile("" : "+v"(lo), "+v"(hi));
  }
};
// the fragment `group` groups of 16 rows on
template <bool TR, int D>
__device__ __forceinline__ v8i frag(const uint8_t* tile, const FragAt<TR, D>& at, int group) {
  v8i f;
  if constexpr (!TR) {
    const uint4 lo = *reinterpret_cast<const uint4*>(tile + at.lo + group * 16 * ROWB);
    const uint4 hi = *reinterpret_cast<const uint4*>(tile + at.hi + group * 16 * ROWB);
    f[0] = (int)lo.x; f[1] = (int)lo.y; f[2] = (int)lo.z; f[3] = (int)lo.w;
    f[4] = (int)hi.x; f[5] = (int)hi.y; f[6] = (int)hi.z; f[7] = (int)hi.w;
  } else {
    const uint8_t* p = tile + (at.lo ^ (uint32_t)(group << 5));
#pragma unroll
    for (int h = 0; h < 4; ++h) {
      const v4s v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s_ptr)(p + h * (8 * D)));
      f[2 * h] = (int)(((uint32_t)(uint16_t)v[1] << 16) | (uint16_t)v[0]);
      f[2 * h + 1] = (int)(((uint32_t)(uint16_t)v[3] << 16) | (uint16_t)v[2]);
    }
  }
  return f;
}

// half a fragment pair's K step: 32 of its 64 contraction values
template <int HALF>
__device__ __forceinline__ v4f mma(const v8i& p, const v8i& q, v4f acc) {
  const v4i a = {p[4 * HALF], p[4 * HALF + 1], p[4 * HALF + 2], p[4 * HALF + 3]};
  const v4i b = {q[4 * HALF], q[4 * HALF + 1], q[4 * HALF + 2], q[4 * HALF + 3]};
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), acc, 0, 0, 0);
}

// the lane, counted anew: not a value that is kept in a register from before
__device__ __forceinline__ int own_lane() {
  int lane = (int)__builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u));
  asm volatile("" : "+v"(lane));
  return lane;
}

// the workgroup's barrier alone: what must have landed is waited for before it
__device__ __forceinline__ void barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  const v2bf p = {(__bf16)a, (__bf16)b};
  return __builtin_bit_cast(uint32_t, p);
}

// One operand, bf16: rows by contraction ([rows, k]) or, transposed, the other
// way ([k, rows]).  The user's weight lies by rows, 16-byte aligned, whole 16-byte
// rows; what lies at or past rows or k reads zero.  The kernels' own X' and dz lie
// in blocks: 64 columns of all rows, 128 bytes a row, one block after another, so
// that the step of a tile is one run of 32 KiB (or, transposed, a run of 8 KiB of
// each of four blocks) and not 256 rows a pitch apart.
struct Mat {
  const uint8_t* p;
  int64_t pitch;  // bytes: of a row, or of a block
  int64_t rows;   // of the operand
  int64_t k;      // contraction
};

// Copies of one K step of a tile of D rows, global -> LDS: four of 1 KiB for each
// of the D / 32 waves.  Resources begin at the tile (rows) or at the K step (transposed), so
// offsets stay small whatever the matrix's size.
// All of a resource is scalar: counts are 32 bits, since comparing 64 would be
// the vector unit's work and the resource be taken to differ among the lanes.
template <int D>
struct RowCopy {
  static constexpr int NW = D / 32;
  __amdgpu_buffer_rsrc_t rs;
  uint32_t off, pitch;
  int k, col;  // columns; the first one of the lane's chunk in a step
  uint32_t at, o;
  __device__ __forceinline__ void init(const Mat& m, int64_t r0, int wave, int lane) {
    const int xr = wave * 8 + (lane >> 3), c = (lane & 7) ^ sw_perm(xr);
    pitch = (uint32_t)m.pitch;
    k = (int)m.k;
    col = c * 8;
    off = (uint32_t)xr * pitch + c * 16;
    const int rows = max(0, min((int)(m.rows - r0), D));
    const uint32_t last = min(pitch, (uint32_t)(k * 2 + 15) / 16 * 16);
    const int bytes = rows > 0 ? (int)((uint32_t)(rows - 1) * pitch + last) : 0;
    rs = __builtin_amdgcn_make_buffer_rsrc((void*)uniform64(m.p + r0 * m.pitch), (short)0,
                                           __builtin_amdgcn_readfirstlane(bytes), 0x00020000);
  }
  // step kt's copies: columns past k read zero
  __device__ __forceinline__ void set(int kt) {
    at = (uint32_t)kt * ROWB;
    o = col < k - kt * KSTEP ? off : 0x80000000u;
  }
  __device__ __forceinline__ void issue(uint8_t* stage, int wave, int j) const {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_ptr_t)(stage + (wave + NW * j) * 1024), 16, o,
                                             at + (uint32_t)j * (8 * NW) * pitch, 0, 0);
  }
};

// The same for steps that are set once each, in their order: what lies past the
// columns is taken out of the lanes' offsets for good, which saves two registers
template <int D>
struct RowWalk {
  __amdgpu_buffer_rsrc_t rs;
  uint32_t off, pitch, at;
  int k, wave;
  __device__ __forceinline__ void init(const Mat& m, int64_t r0, int w, int lane) {
    RowCopy<D> c;
    c.init(m, r0, w, lane);
    rs = c.rs;
    off = c.off;
    pitch = c.pitch;
    k = __builtin_amdgcn_readfirstlane(c.k);
    wave = w;
  }
  __device__ __forceinline__ void set(int kt) {
    at = (uint32_t)kt * ROWB;
    const int rem = k - kt * KSTEP;
    if (rem < KSTEP) {
      const int lane = own_lane(), col = ((lane & 7) ^ sw_perm(wave * 8 + (lane >> 3))) * 8;
      off = col < rem ? off : 0x80000000u;
    }
  }
  __device__ __forceinline__ void issue(uint8_t* stage, int w, int j) const {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_ptr_t)(stage + (w + RowCopy<D>::NW * j) * 1024), 16, off,
                                             at + (uint32_t)j * (8 * RowCopy<D>::NW) * pitch, 0, 0);
  }
};

template <int D>
struct TrCopy {
  const uint8_t* p;
  uint32_t pitch, last, off;
  int k;
  __amdgpu_buffer_rsrc_t rs;
  // the first of the rows of a wave's copy j (two of 512 bytes or four of 256):
  // bit 4, which the swizzle looks at, is the wave's, so its lanes' offsets serve all j
  __device__ static int row0(int wave, int j) {
    return (D == 256 ? 2 * (wave & 3) + 16 * (wave >> 2) + 8 * (j & 1) : 8 * (wave >> 1) + 16 * (wave & 1) + 4 * (j & 1)) +
           32 * (j >> 1);
  }
  __device__ __forceinline__ void init(const Mat& m, int64_t r0, int wave, int lane) {
    const int R = row0(wave, 0) + lane / (D / 8), c = lane % (D / 8) ^ tr_perm(R);
    p = uniform64(m.p + r0 * 2);
    pitch = (uint32_t)m.pitch;
    k = __builtin_amdgcn_readfirstlane((int)m.k);
    // the last stored row ends with the operand's rows, 16 bytes rounded up
    last = min(pitch, (uint32_t)(m.rows * 2 + 15) / 16 * 16) - (uint32_t)(r0 * 2);
    off = (uint32_t)R * pitch + 16 * c;
  }
  // step kt's resource, from its first row's first column of the tile: 64 pitches
  // where a 65th row holds their end, else to the end of the last row (a tile that
  // overhangs its rows reads into the next stored row)
  __device__ __forceinline__ void set(int kt) {
    const int rem = k - kt * KSTEP;
    const uint32_t bytes = rem <= 0 ? 0 : rem > KSTEP ? KSTEP * pitch : (uint32_t)(rem - 1) * pitch + last;
    rs = __builtin_amdgcn_make_buffer_rsrc((void*)uniform64(p + (int64_t)kt * KSTEP * pitch), (short)0,
                                           __builtin_amdgcn_readfirstlane((int)bytes), 0x00020000);
  }
  __device__ __forceinline__ void issue(uint8_t* stage, int wave, int j) const {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_ptr_t)(stage + row0(wave, j) * (2 * D)), 16, off,
                                             (uint32_t)(row0(0, j)) * pitch, 0, 0);
  }
};

// by rows, in blocks of the contraction
template <int D>
struct BlockRowCopy {
  static constexpr int NW = D / 32;
  const uint8_t* p;
  int64_t pitch;
  int bytes;
  uint32_t off;
  __amdgpu_buffer_rsrc_t rs;
  __device__ __forceinline__ void init(const Mat& m, int64_t r0, int wave, int lane) {
    const int xr = wave * 8 + (lane >> 3), c = (lane & 7) ^ sw_perm(xr);
    p = uniform64(m.p + r0 * ROWB);
    pitch = m.pitch;
    bytes = __builtin_amdgcn_readfirstlane(max(0, min((int)(m.rows - r0), D)) * ROWB);
    off = (uint32_t)(xr * ROWB + c * 16);
  }
  __device__ __forceinline__ void set(int kt) {
    rs = __builtin_amdgcn_make_buffer_rsrc((void*)uniform64(p + kt * pitch), (short)0, bytes, 0x00020000);
  }
  __device__ __forceinline__ void issue(uint8_t* stage, int wave, int j) const {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_ptr_t)(stage + (wave + NW * j) * 1024), 16, off, j * (8 * NW * ROWB), 0, 0);
  }
};

// transposed, in blocks of the operand's rows: the contraction's rows up to the
// next 64 are there, zero
template <int D>
struct BlockTrCopy {
  const uint8_t* p;
  uint32_t bytes, off;
  __amdgpu_buffer_rsrc_t rs;
  __device__ __forceinline__ void init(const Mat& m, int64_t r0, int wave, int lane) {
    const int R = TrCopy<D>::row0(wave, 0) + lane / (D / 8), c = lane % (D / 8) ^ tr_perm(R);
    p = uniform64(m.p + (r0 / 64) * m.pitch);
    const int blocks = min((int)((m.rows - r0 + 63) / 64), D / 64);
    bytes = __builtin_amdgcn_readfirstlane(m.k > 0 && blocks > 0 ? (uint32_t)blocks * (uint32_t)m.pitch : 0);
    off = (uint32_t)(c >> 3) * (uint32_t)m.pitch + (uint32_t)(R * ROWB + (c & 7) * 16);
  }
  __device__ __forceinline__ void set(int kt) {
    const uint32_t at = (uint32_t)kt * (KSTEP * ROWB);
    rs = __builtin_amdgcn_make_buffer_rsrc((void*)uniform64(p + at), (short)0,
                                           __builtin_amdgcn_readfirstlane((int)(bytes > at ? bytes - at : 0)), 0x00020000);
  }
  __device__ __forceinline__ void issue(uint8_t* stage, int wave, int j) const {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_ptr_t)(stage + TrCopy<D>::row0(wave, j) * (2 * D)), 16, off,
                                             TrCopy<D>::row0(0, j) * ROWB, 0, 0);
  }
};

// A wave's 16 MT x 64 output rows as bf16, 32 rows at a time through 4 KiB of LDS
// (16-byte chunks XOR-swizzled by row, so that neither side's lanes share banks) to
// stores of whole 128-byte lines.  value(tm, tn, v): the lane's four of a block.
template <int MT, bool NTS, typename F>
__device__ __forceinline__ void store_bf16(uint8_t* stage, int lane, int64_t m0, int64_t n0, int64_t M, int64_t N,
                                           uint16_t* out, int64_t ldo, F value) {
  constexpr int PITCH = 64 * 2;
  // whole tiles' stores without a branch of their own: 56 of them for each compute unit take 28 us less
  const bool full = m0 + 16 * MT <= M && n0 + 64 <= N;
#pragma unroll
  for (int part = 0; part < MT / 2; ++part) {
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int tn = 0; tn < 4; ++tn) {
        float v[4];
        value(part * 2 + t, tn, v);
        *reinterpret_cast<uint2*>(stage + (t * 16 + (lane & 15)) * PITCH + (((tn * 2 + (lane >> 5)) ^ (lane & 7)) << 4) + ((lane >> 4) & 1) * 8) =
            make_uint2(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]));
      }
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0): the wave's rows are written
    __builtin_amdgcn_wave_barrier();
    auto at = [&](int j) {  // the place of the lane's 16 bytes in quarter j
      const int row = (lane >> 3) + 8 * j;
      return m0 + part * 32 + row;
    };
    if (full) {
      uint4 q[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) q[j] = *reinterpret_cast<const uint4*>(stage + ((lane >> 3) + 8 * j) * PITCH + (((lane & 7) ^ (lane >> 3)) << 4));
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const u32x4_2 v = {q[j].x, q[j].y, q[j].z, q[j].w};
        u32x4_2* o = reinterpret_cast<u32x4_2*>(out + at(j) * ldo + n0 + (lane & 7) * 8);
        if constexpr (NTS)
          __builtin_nontemporal_store(v, o);
        else
          *o = v;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int c = lane & 7;
        const int64_t m = at(j), n = n0 + c * 8;
        const uint4 q = *reinterpret_cast<const uint4*>(stage + ((lane >> 3) + 8 * j) * PITCH + ((c ^ (lane >> 3)) << 4));
        if (m >= M || n >= N) continue;
        uint16_t* o = out + m * ldo + n;
        if (n + 8 <= N) {
          const u32x4_2 v = {q.x, q.y, q.z, q.w};
          if constexpr (NTS)
            __builtin_nontemporal_store(v, reinterpret_cast<u32x4_2*>(o));
          else
            *reinterpret_cast<u32x4_2*>(o) = v;
        } else {
          const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (n + i < N) o[i] = (uint16_t)(w[i >> 1] >> (16 * (i & 1)));
        }
      }
    }
    __builtin_amdgcn_s_waitcnt(0xC07F);  // read before the next rows overwrite them
    __builtin_amdgcn_wave_barrier();
  }
}

// the copies of step kt into a stage
template <typename CA, typename CB>
__device__ __forceinline__ void prime(CA& ca, CB& cb, int kt, int wave, uint8_t* la, uint8_t* lb) {
  ca.set(kt);
  cb.set(kt);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    ca.issue(la, wave, j);
    cb.issue(lb, wave, j);
  }
}

// acc += the product of K steps kb0 .. kb1 - 1 of a tile of D x D (256: eight waves
// of 128 x 64, one workgroup a compute unit; 128: four of 64 x 64, two workgroups),
// wave (wm, wn) of it.  la0 ... lb1: two stages of both operands, D * ROWB bytes
// each, which nothing reads or writes any more afterwards.  PRIMED: prime() has been
// called for step kb0 and the first stage.  idle: the wave's rows lie behind the
// operand's last one; it copies its share and multiplies nothing, which leaves the matrix
// cores and their power to the others (256 rows of 32 experts, 4096 x 7168: 325 us and so 315;
// 4096 rows 568 and 542; dx of 32768 1773 and 1748).
template <int D, bool TA, bool TB, bool PRIMED = false, typename CA, typename CB>
__device__ __forceinline__ void multiply(CA& ca, CB& cb, int kb0, int kb1, v4f (&acc)[D / 32][4], int wm, int wn, int wave,
                                         int lane, uint8_t* la0, uint8_t* lb0, uint8_t* la1, uint8_t* lb1,
                                         bool idle = false) {
  constexpr int MT = D / 32;
  if (idle && kb0 < kb1) {  // the copies and barriers of the loop below
    if constexpr (!PRIMED) prime(ca, cb, kb0, wave, la0, lb0);
    __builtin_amdgcn_s_waitcnt(0);
    barrier();
#pragma unroll 1
    for (int kt = kb0; kt < kb1; ++kt) {
      const bool odd = (kt - kb0) & 1;
      const int kn = min(kt + 1, kb1 - 1);
      ca.set(kn);
      cb.set(kn);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        ca.issue(odd ? la0 : la1, wave, j);
        cb.issue(odd ? lb0 : lb1, wave, j);
      }
      __builtin_amdgcn_s_waitcnt(0);
      barrier();
    }
    return;
  }
  // K loop.  A step's fragments stream through registers, A's two row groups
  // ahead.  The one barrier of a step stands after its last LDS read, before the
  // products of its last two row groups: those cover the first reads of the next
  // step, and the copies of the step after it, into the stage just read, have a
  // whole step's time to land.  So an iteration is: the last two row groups of
  // step kt - 1 (of zeros, at first), the others of step kt, the barrier.
  if (kb0 < kb1) {
    auto copy = [&](uint8_t* na, uint8_t* nb, int j) {
      ca.issue(na, wave, j);
      cb.issue(nb, wave, j);
    };
    auto rows = [&](int tm, const v8i (&bf)[4], const v8i& a) {
      // one operand by rows, one transposed: the products before the other wave's
      // reads (4096 x 7168 over 65536: 2.85 ms, without 3.10; of two operands read
      // alike 4096 x 65536 over 7168 5.48 and 5.41 ms, 65536 x 7168 over 4096 2.89 and 2.69)
      if (TB && !TA) __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int tn = 0; tn < 4; ++tn) acc[tm][tn] = mma<0>(bf[tn], a, acc[tm][tn]);
#pragma unroll
      for (int tn = 0; tn < 4; ++tn) acc[tm][tn] = mma<1>(bf[tn], a, acc[tm][tn]);
      asm volatile("" : "+v"(acc[tm][0]), "+v"(acc[tm][1]), "+v"(acc[tm][2]), "+v"(acc[tm][3])::"memory");
      if (TB && !TA) __builtin_amdgcn_s_setprio(0);
    };
    if constexpr (!PRIMED) prime(ca, cb, kb0, wave, la0, lb0);
    v8i b0[4], b1[4], af[4];
    FragAt<TA, D> fa(wm * 16 * MT, lane);
    FragAt<TB, D> fb(wn * 64, lane);
#pragma unroll
    for (int i = 0; i < 4; ++i) b1[i] = af[i] = (v8i){0, 0, 0, 0, 0, 0, 0, 0};
    __builtin_amdgcn_s_waitcnt(0);
    barrier();
    auto step = [&](auto bufc, int kt, const v8i (&bo)[4], v8i (&bf)[4]) {
      constexpr int BUF = decltype(bufc)::value;
      const uint8_t* ta = BUF ? la1 : la0;
      const uint8_t* tb = BUF ? lb1 : lb0;
      uint8_t* oa = BUF ? la0 : la1;
      uint8_t* ob = BUF ? lb0 : lb1;
      const int kn = min(kt + 1, kb1 - 1);  // the last step copies itself into the idle stage
      fa.renew();
      fb.renew();
      ca.set(kn);
      cb.set(kn);
#pragma unroll
      for (int tn = 0; tn < 4; ++tn) bf[tn] = frag(tb, fb, tn);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        af[i] = frag(ta, fa, i);
        copy(oa, ob, 2 * i);
        copy(oa, ob, 2 * i + 1);
        rows(MT - 2 + i, bo, af[2 + i]);
      }
#pragma unroll
      for (int tm = 0; tm < MT - 2; ++tm) {
        af[(tm + 2) & 3] = frag(ta, fa, tm + 2);
        rows(tm, bf, af[tm & 3]);
      }
      __builtin_amdgcn_s_waitcnt(0);  // this wave's reads of the stage and its copies into the other are done
      barrier();
    };
    int kt = kb0;
    for (; kt + 2 <= kb1; kt += 2) {
      step(std::integral_constant<int, 0>(), kt, b1, b0);
      step(std::integral_constant<int, 1>(), kt + 1, b0, b1);
    }
    if (kt < kb1) {
      step(std::integral_constant<int, 0>(), kt, b1, b0);
#pragma unroll
      for (int i = 0; i < 4; ++i) b1[i] = b0[i];
    }
    rows(MT - 2, b1, af[2]);
    rows(MT - 1, b1, af[3]);
    // no wave reads the stages any more, and none copies into them
  }
}

// The same of two operands by rows with the copies of A (FAR_B: of B) two steps ahead,
// for what comes from far: three stages of it, two of the other (5 D ROWB bytes).  A
// step's copies of the near one are issued first, so that at its end a wave waits for
// those of the next step only.
// (32768 x 7168 by 4096 rows: 1507 us with both one step ahead, 1404 so; with B's two
// ahead too, its stage freed by a second barrier after its fragments are read, 1501.)
// prime_ahead() has been called for step k0; k0 < k1.  Afterwards nothing reads or
// writes the stages.  idle: as above.
struct Stages {
  uint8_t *far0, *far1, *far2, *near0, *near1;  // of the operand two steps ahead, of the other
  template <int I>
  __device__ __forceinline__ uint8_t* far() const { return I == 0 ? far0 : I == 1 ? far1 : far2; }
  template <int I>
  __device__ __forceinline__ uint8_t* near() const { return I == 0 ? near0 : near1; }
};
template <bool FAR_B = false, typename CA, typename CB>
__device__ __forceinline__ void prime_ahead(CA& ca, CB& cb, int k0, int wave, const Stages& st) {
  prime(ca, cb, k0, wave, FAR_B ? st.near0 : st.far0, FAR_B ? st.far0 : st.near0);
  if constexpr (FAR_B) cb.set(k0 + 1);
  else ca.set(k0 + 1);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if constexpr (FAR_B) cb.issue(st.far1, wave, j);
    else ca.issue(st.far1, wave, j);
  }
}
template <int D, bool FAR_B = false, typename CA, typename CB>
__device__ __forceinline__ void multiply_ahead(CA& ca, CB& cb, int k0, int k1, v4f (&acc)[D / 32][4], int wm, int wn, int wave, int lane,
                                               const Stages& st, bool idle) {
  constexpr int MT = D / 32;
  constexpr int NONE = 0x0070, FOUR = 0x0074;  // s_waitcnt: lgkmcnt(0) with vmcnt(0), vmcnt(4)
  if (idle) {  // the copies and barriers of the loop below
    __builtin_amdgcn_s_waitcnt(FOUR);
    barrier();
    uint8_t *f0 = st.far2, *f1 = st.far0, *f2 = st.far1, *n0 = st.near1, *n1 = st.near0;
#pragma unroll 1
    for (int kt = k0; kt < k1; ++kt) {
      ca.set(kt + (FAR_B ? 1 : 2));
      cb.set(kt + (FAR_B ? 2 : 1));
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (FAR_B) ca.issue(n0, wave, j);
        else cb.issue(n0, wave, j);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (FAR_B) cb.issue(f0, wave, j);
        else ca.issue(f0, wave, j);
      }
      uint8_t *f = f0, *n = n0;
      f0 = f1;
      f1 = f2;
      f2 = f;
      n0 = n1;
      n1 = n;
      __builtin_amdgcn_s_waitcnt(FOUR);
      barrier();
    }
    __builtin_amdgcn_s_waitcnt(NONE);
    barrier();
    return;
  }
  auto rows = [&](int tm, const v8i (&bf)[4], const v8i& a) {
#pragma unroll
    for (int tn = 0; tn < 4; ++tn) acc[tm][tn] = mma<0>(bf[tn], a, acc[tm][tn]);
#pragma unroll
    for (int tn = 0; tn < 4; ++tn) acc[tm][tn] = mma<1>(bf[tn], a, acc[tm][tn]);
    asm volatile("" : "+v"(acc[tm][0]), "+v"(acc[tm][1]), "+v"(acc[tm][2]), "+v"(acc[tm][3])::"memory");
  };
  v8i b0[4], b1[4], af[4];
  FragAt<false, D> fa(wm * 16 * MT, lane);
  FragAt<false, D> fb(wn * 64, lane);
#pragma unroll
  for (int i = 0; i < 4; ++i) b1[i] = af[i] = (v8i){0, 0, 0, 0, 0, 0, 0, 0};
  __builtin_amdgcn_s_waitcnt(FOUR);
  barrier();
  // step kt, from stages tf and tn, the step after next's copies to nf, the next one's to nn; bo: B's fragments
  // of the step before.
  // Copies of steps past k1 are made all the same, so that no step has a branch: past the
  // contraction they fetch nothing (all of them is out of their resources' bounds).
  auto step = [&](uint8_t* tf, uint8_t* tn, uint8_t* nf, uint8_t* nn, int kt, const v8i (&bo)[4], v8i (&bf)[4]) {
    uint8_t *ta = FAR_B ? tn : tf, *tb = FAR_B ? tf : tn;
    ca.set(kt + (FAR_B ? 1 : 2));
    cb.set(kt + (FAR_B ? 2 : 1));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      fb.anew();
      bf[i] = frag(tb, fb, i);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      fa.anew();
      af[i] = frag(ta, fa, i);
#pragma unroll
      for (int j = 2 * i; j < 2 * i + 2; ++j) {
        if constexpr (FAR_B) ca.issue(nn, wave, j);
        else cb.issue(nn, wave, j);
      }
      rows(MT - 2 + i, bo, af[2 + i]);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (FAR_B) cb.issue(nf, wave, j);
      else ca.issue(nf, wave, j);
    }
#pragma unroll
    for (int tm = 0; tm < MT - 2; ++tm) {
      fa.anew();
      af[(tm + 2) & 3] = frag(ta, fa, tm + 2);
      rows(tm, bf, af[tm & 3]);
    }
    __builtin_amdgcn_s_waitcnt(FOUR);
    barrier();
  };
#define NTLB_STEP(I, BO, BF) step(st.far<(I) % 3>(), st.near<(I) % 2>(), st.far<((I) + 2) % 3>(), st.near<((I) + 1) % 2>(), kt + I, BO, BF)
  // A contraction may end behind each of the six steps.  (Up to five steps in a loop of
  // their own, stages found at run time: the compiler then waits for every copy before
  // it reads one, 32768 x 7168 by 32 matrices of 4096 rows 1700 us and so 1657.  Of
  // transposed operands the exits cost more registers than there are.)
  for (int kt = k0;; kt += 6) {
    NTLB_STEP(0, b1, b0);
    if (kt + 1 >= k1) goto even;
    NTLB_STEP(1, b0, b1);
    if (kt + 2 >= k1) break;
    NTLB_STEP(2, b1, b0);
    if (kt + 3 >= k1) goto even;
    NTLB_STEP(3, b0, b1);
    if (kt + 4 >= k1) break;
    NTLB_STEP(4, b1, b0);
    if (kt + 5 >= k1) goto even;
    NTLB_STEP(5, b0, b1);
    if (kt + 6 >= k1) break;
  }
  if (false) {
  even:
#pragma unroll
    for (int i = 0; i < 4; ++i) b1[i] = b0[i];
  }
  rows(MT - 2, b1, af[2]);
  rows(MT - 1, b1, af[3]);
#undef NTLB_STEP
  __builtin_amdgcn_s_waitcnt(NONE);
  barrier();  // nothing is on its way into a stage any more
}

}  // namespace tile
}  // namespace ntlb

// two stages of both operands of a tile
#define NTLB_TILE_STAGES(D)                                            \
  __shared__ __attribute__((aligned(16))) uint8_t la0[D * ROWB]; \
  __shared__ __attribute__((aligned(16))) uint8_t lb0[D * ROWB]; \
  __shared__ __attribute__((aligned(16))) uint8_t la1[D * ROWB]; \
  __shared__ __attribute__((aligned(16))) uint8_t lb1[D * ROWB]
// three of the far operand, two of the near one
#define NTLB_TILE_STAGES_AHEAD(D)                                   \
  __shared__ __attribute__((aligned(16))) uint8_t stage_0[D * ROWB]; \
  __shared__ __attribute__((aligned(16))) uint8_t stage_1[D * ROWB]; \
  __shared__ __attribute__((aligned(16))) uint8_t stage_2[D * ROWB]; \
  __shared__ __attribute__((aligned(16))) uint8_t stage_3[D * ROWB]; \
  __shared__ __attribute__((aligned(16))) uint8_t stage_4[D * ROWB]; \
  const Stages stages{stage_2, stage_3, stage_4, stage_0, stage_1}
