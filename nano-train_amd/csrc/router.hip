// Routing of tokens to experts from the router's logits z [T, E], forward and
// backward:
//   p = softmax(z) or sigmoid(z),  c = p + bias (the choice; c = p without one)
//   groups: a group's score is the sum of its two highest choices; the choices
//           outside the topk_groups best groups drop out
//   ids = the top_k highest choices, highest first, equal ones lowest index first
//   w_i = scale p_i / (sum of the chosen p + 1e-20), or scale p_i
// and from dw the gradient of z (the choice itself has none):
//   d_i = scale dw_i, renormalised: (d_i - sum(d p) / S) / S
//   softmax: dz = p (dp - sum(dp p)); sigmoid: dz = dp p (1 - p)
// Everything is fp32; w is stored as fp32, dz rounded once to z's type.
//
// A few bytes per expert and token: HBM-bound for many tokens if the choice
// costs few instructions.  LPT lanes hold a token's choices, J each (16 lanes
// up to 256 experts, so a wave has four tokens; 64 lanes above).  The choice
// is a tournament of sorted lists: each lane sorts its J keys in registers,
// then log2(LPT) times merges its list with its partner's, keeping the KN >=
// top_k highest: a bitonic merge has no data-dependent step, so nothing waits
// on a reduction per chosen expert.  A key is a positive double whose upper
// bits order as the choice and whose lowest ten bits hold 1023 - e: keys of one
// token are distinct, v_max_f64 / v_min_f64 compare and exchange choice and
// index together, and ties go to the lowest index by themselves.
// Measured: 65536 tokens, 256 fp32 experts in 8 groups, sigmoid and bias: forward
// 31 to 32 us, the vector unit's: 1075 instructions for a wave's four tokens, of
// which 320 sort and merge, 16 x 2 are transcendental, and 288 stand before the
// loop (edges, places in LDS, which lanes hold earlier groups, scalars kept in
// vector registers): at 16 workgroups a compute unit every wave here has one step,
// which shares them with no other.  Its 67 MB alone would take 13.  Backward 15.5 us
// for 134 MB (part of z is still in the last cache).  4096 tokens of 32 experts: 3.5
// and 3.4 us, 32 tokens of 256: 4.8 us, little more than an empty launch.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "ntlb_device.h"
#include "ntlb_host.h"
#include "ntlb_splitk.h"

namespace ntlb {
namespace router {

typedef __bf16 v2bf __attribute__((ext_vector_type(2)));

constexpr int MAX_E = 1024, MAX_K = 16, MAX_G = 16;
constexpr int WAVES = 4;  // waves of a workgroup; none waits on another
constexpr float RENORM_EPS = 1e-20f;

struct Args {
  const void* z;
  int64_t ldz;  // elements
  int64_t T;
  int E, k, sigmoid, renorm;
  int G, Gk, gsize, gmagic;  // e / gsize == (e * gmagic) >> 20
  int per, gshift;           // where groups are runs of lanes: experts of a lane, log2 of a group's lanes
  float scale;
  const float* bias;
  int32_t* ids;  // [T, k]
  float* w;      // [T, k]
  const float* dw;
  void* dz;
  int64_t lddz;
};

// exp(x), within two units of the last place: v_exp_f32 of x log2(e) with the
// product's rounding error put back to first order.  From |x| of about 88.7 on
// there is nothing to put back: 0 or infinity (whose correction would be infinity
// times 0, or less infinity: NaN), and NaN stays.
__device__ __forceinline__ float exp_f32(float x) {
  constexpr float L = 1.44269502e+00f, L_LO = 1.92596303e-08f, LN2 = 6.93147182e-01f;
  const float t = x * L;
  float r = __builtin_fmaf(x, L, -t);
  r = __builtin_fmaf(x, L_LO, r) * LN2;
  const float e = __builtin_amdgcn_exp2f(t);
  return __builtin_fabsf(t) < 128.f ? __builtin_fmaf(e, r, e) : e;
}

// Lane l of a token's LPT lanes holds elements e(l, j): chunks of V consecutive
// ones per lane, so that the lanes' loads lie side by side
template <int LPT, int J>
struct Lay {
  static constexpr int V = J < 4 ? J : 4;
  __device__ static int e(int l, int j) { return (j / V) * (LPT * V) + l * V + j % V; }
};

template <int DT, int LPT, int J>
__device__ __forceinline__ void load_row(const void* z, int64_t at, int l, int E, float fill, float (&f)[J]) {
  constexpr int V = Lay<LPT, J>::V;
#pragma unroll
  for (int c = 0; c < J / V; ++c) {
    const int e = Lay<LPT, J>::e(l, c * V);
    if (e + V <= E) {
      if constexpr (DT == DT_F32) {
        typedef float vec __attribute__((ext_vector_type(V), aligned(4)));
        const vec v = *reinterpret_cast<const vec*>((const float*)z + at + e);
#pragma unroll
        for (int i = 0; i < V; ++i) f[c * V + i] = v[i];
      } else {
        typedef uint16_t vec __attribute__((ext_vector_type(V), aligned(2)));
        const vec v = *reinterpret_cast<const vec*>((const uint16_t*)z + at + e);
#pragma unroll
        for (int i = 0; i < V; ++i)
          f[c * V + i] = DT == DT_BF16 ? bf16_bits_to_f32(v[i]) : __half2float(__ushort_as_half(v[i]));
      }
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) f[c * V + i] = e + i < E ? load_elem(z, DT, at + e + i) : fill;
    }
  }
}

template <int DT, int LPT, int J>
__device__ __forceinline__ void store_row(void* z, int64_t at, int l, int E, const float (&f)[J]) {
  constexpr int V = Lay<LPT, J>::V;
#pragma unroll
  for (int c = 0; c < J / V; ++c) {
    const int e = Lay<LPT, J>::e(l, c * V);
    if (e + V <= E) {
      if constexpr (DT == DT_F32) {
        typedef float vec __attribute__((ext_vector_type(V), aligned(4)));
        vec v;
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = f[c * V + i];
        __builtin_nontemporal_store(v, reinterpret_cast<vec*>((float*)z + at + e));
      } else {
        typedef uint16_t vec __attribute__((ext_vector_type(V), aligned(2)));
        vec v;
#pragma unroll
        for (int i = 0; i < V; ++i)
          v[i] = DT == DT_BF16 ? f32_to_bf16_bits(f[c * V + i]) : __half_as_ushort(f32_to_f16(f[c * V + i]));
        __builtin_nontemporal_store(v, reinterpret_cast<vec*>((uint16_t*)z + at + e));
      }
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (e + i < E) store_elem(z, DT, at + e + i, f[c * V + i]);
    }
  }
}

// the value of the partner lane of step S: lane ^ 1, ^ 2, 7 - lane, 15 - lane
// (in its row of 16), then lane ^ 16, lane ^ 32
template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, CTRL, 0xF, 0xF, true);
}
template <int S>
__device__ __forceinline__ uint32_t partner(uint32_t v) {
  if constexpr (S == 0) return dpp<0xB1>(v);
  if constexpr (S == 1) return dpp<0x4E>(v);
  if constexpr (S == 2) return dpp<0x141>(v);
  if constexpr (S == 3) return dpp<0x140>(v);
  if constexpr (S == 4) return (uint32_t)__shfl_xor((int)v, 16);
  return (uint32_t)__shfl_xor((int)v, 32);
}
template <int S>
__device__ __forceinline__ float partner(float v) {
  return __uint_as_float(partner<S>(__float_as_uint(v)));
}
template <int S>
__device__ __forceinline__ double partner(double v) {
  const uint64_t u = (uint64_t)__double_as_longlong(v);
  const uint32_t lo = partner<S>((uint32_t)u), hi = partner<S>((uint32_t)(u >> 32));
  return __longlong_as_double((long long)(((uint64_t)hi << 32) | lo));
}

template <int LPT>
__device__ __forceinline__ float token_sum(float v) {
  v += partner<0>(v);
  v += partner<1>(v);
  v += partner<2>(v);
  v += partner<3>(v);
  if constexpr (LPT == 64) {
    v += partner<4>(v);
    v += partner<5>(v);
  }
  return v;
}
// NaN in any lane gives NaN
__device__ __forceinline__ float max_nan(float a, float b) { return a != a || a > b ? a : b; }
template <int LPT>
__device__ __forceinline__ float token_max(float v) {
  v = max_nan(v, partner<0>(v));
  v = max_nan(v, partner<1>(v));
  v = max_nan(v, partner<2>(v));
  v = max_nan(v, partner<3>(v));
  if constexpr (LPT == 64) {
    v = max_nan(v, partner<4>(v));
    v = max_nan(v, partner<5>(v));
  }
  return v;
}

// score(z) of one expert, given what is common to the token: sigmoid, or the
// softmax's maximum and 1 / sum.  Softmax of a row of -infinities is 0 everywhere.
struct Common {
  float m, inv;
};
__device__ __forceinline__ float score(float z, int sigmoid, const Common& c) {
  return sigmoid ? __builtin_amdgcn_rcpf(1.0f + exp_f32(-z)) : exp_f32(z - c.m) * c.inv;
}
// scores of the lane's elements; those past E are 0
template <int LPT, int J>
__device__ __forceinline__ Common scores(const float (&z)[J], int sigmoid, float (&p)[J]) {
  Common c{0.f, 0.f};
  if (sigmoid) {
#pragma unroll
    for (int j = 0; j < J; ++j) p[j] = score(z[j], 1, c);
    return c;
  }
  c.m = z[0];
#pragma unroll
  for (int j = 1; j < J; ++j) c.m = max_nan(c.m, z[j]);
  c.m = token_max<LPT>(c.m);
  c.m = c.m == -__builtin_inff() ? 0.f : c.m;
  float s = 0.f;
#pragma unroll
  for (int j = 0; j < J; ++j) {
    p[j] = exp_f32(z[j] - c.m);
    s += p[j];
  }
  s = token_sum<LPT>(s);
  c.inv = s == 0.f ? 0.f : 1.0f / s;
#pragma unroll
  for (int j = 0; j < J; ++j) p[j] *= c.inv;
  return c;
}

// the order of a choice as a 32-bit whole number: -inf lowest (and above 0), NaN
// highest; a choice, p + bias with p >= 0, is never -0
__device__ __forceinline__ uint32_t order_bits(float c) {
  const uint32_t s = __float_as_uint(c);
  const uint32_t u = s ^ ((uint32_t)((int32_t)s >> 31) | 0x80000000u);
  return c != c ? 0xFFFFFFFFu : u;
}
__device__ __forceinline__ float order_value(uint32_t u) {  // of order_bits, NaN for NaN
  return __uint_as_float((u & 0x80000000u) ? u ^ 0x80000000u : ~u);
}
__device__ __forceinline__ double make_key(uint32_t order, int e) {
  const uint32_t hi = order >> 2, lo = (order << 30) | (uint32_t)(1023 - e);
  return __longlong_as_double((long long)(((uint64_t)hi << 32) | lo));
}

// the instructions themselves: keys are no NaNs, and the compiler would first
// make sure of it, value by value
__device__ __forceinline__ double max64(double a, double b) {
  double r;
  asm("v_max_f64 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
  return r;
}
__device__ __forceinline__ double min64(double a, double b) {
  double r;
  asm("v_min_f64 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
  return r;
}
__device__ __forceinline__ void exchange(double& a, double& b) {
  const double hi = max64(a, b), lo = min64(a, b);
  a = hi;
  b = lo;
}
// a bitonic list of N into descending order
template <int N>
__device__ __forceinline__ void bitonic(double* v) {
#pragma unroll
  for (int d = N / 2; d > 0; d /= 2)
#pragma unroll
    for (int i = 0; i < N; ++i)
      if ((i & d) == 0) exchange(v[i], v[i + d]);
}
// v[0, N) into descending order: halves sorted, one reversed, merged
template <int N>
__device__ __forceinline__ void sort_desc(double* v) {
  if constexpr (N > 1) {
    sort_desc<N / 2>(v);
    sort_desc<N / 2>(v + N / 2);
#pragma unroll
    for (int i = 0; i < N / 2; ++i) exchange(v[i], v[N - 1 - i]);
    bitonic<N / 2>(v);
    bitonic<N / 2>(v + N / 2);
  }
}

// one round: the lane's L sorted keys and its partner's into the min(2L, KN)
// highest of both, sorted, the same in both lanes
template <int L, int KN, int S>
__device__ __forceinline__ void merge_round(double* v) {
  if constexpr (2 * L <= KN) {
#pragma unroll
    for (int i = 0; i < L; ++i) v[2 * L - 1 - i] = partner<S>(v[i]);
    bitonic<2 * L>(v);
  } else {
    double o[L];
#pragma unroll
    for (int i = 0; i < L; ++i) o[i] = partner<S>(v[i]);
#pragma unroll
    for (int i = 0; i < L; ++i) v[i] = max64(v[i], o[L - 1 - i]);
    bitonic<L>(v);
  }
}
template <int L, int KN, int S, int STEPS>
__device__ __forceinline__ void merge_lanes(double* v) {
  if constexpr (S < STEPS) {
    merge_round<L, KN, S>(v);
    merge_lanes<(2 * L <= KN ? 2 * L : L), KN, S + 1, STEPS>(v);
  }
}
// the lane's J keys to its min(J, KN) highest, sorted, in v[0 ...]
template <int J, int KN>
__device__ __forceinline__ void lane_list(double* v) {
  if constexpr (J <= KN) {
    sort_desc<J>(v);
  } else {
#pragma unroll
    for (int c = 0; c < J / KN; ++c) sort_desc<KN>(v + c * KN);
#pragma unroll
    for (int c = 1; c < J / KN; ++c) {
#pragma unroll
      for (int i = 0; i < KN; ++i) v[i] = max64(v[i], v[c * KN + KN - 1 - i]);
      bitonic<KN>(v);
    }
  }
}

// place of expert e in a token's LDS row: four words of skew per 16, so that
// lanes that read runs of 16 start in different banks
__device__ __forceinline__ int slot(int e) { return e + ((e >> 4) << 2); }
template <int LPT, int J>
constexpr int row_words() { return LPT * J + LPT * J / 4; }

// a wave's LDS traffic is in order; this keeps the compiler's order too
__device__ __forceinline__ void wave_fence() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

template <int LPT, int J, typename T>
__device__ __forceinline__ void to_lds(T* row, int l, const T (&f)[J]) {
  constexpr int V = Lay<LPT, J>::V;
  typedef T vec __attribute__((ext_vector_type(V)));
#pragma unroll
  for (int c = 0; c < J / V; ++c) {
    vec v;
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = f[c * V + i];
    *reinterpret_cast<vec*>(row + slot(Lay<LPT, J>::e(l, c * V))) = v;
  }
}

// the two highest, a >= b, of a, b and v
__device__ __forceinline__ void top2(uint32_t& a, uint32_t& b, uint32_t v) {
  b = max(min(a, v), b);
  a = max(a, v);
}
// a group's score, as its order
__device__ __forceinline__ uint32_t group_order(uint32_t a, uint32_t b, int gsize) {
  return gsize == 1 ? a : order_bits(order_value(a) + order_value(b));
}
// how many of the other lanes' groups come before this lane's (each once for
// each of its lanes): earlier holds bit R where the lane R round the row of 16
// lies in an earlier group
template <int R>
__device__ __forceinline__ int groups_before(uint32_t order, uint32_t earlier) {
  if constexpr (R > 15) {
    return 0;
  } else {
    // an equal group counts if it is the earlier one
    return (dpp<0x120 + R>(order) > order - ((earlier >> R) & 1u) ? 1 : 0) + groups_before<R + 1>(order, earlier);
  }
}

// GM: how the groups are chosen.  NONE: all are kept; LANES: a group is 16 / G
// lanes of a row of 16, each reading its E / 16 experts in a row (LPT 16, E a
// multiple of 16, G a power of two); WALK: any other, each walked by one lane
constexpr int NONE = 0, LANES = 1, WALK = 2;

template <int DT, int LPT, int J, int KN, int GM>
__global__ void __launch_bounds__(64 * WAVES) forward_kernel(Args g) {
  constexpr int TPW = 64 / LPT, W = row_words<LPT, J>(), STEPS = LPT == 64 ? 6 : 4;
  constexpr int NL = J > KN ? J : KN;
  __shared__ __attribute__((aligned(16))) uint32_t rows[GM == NONE ? 1 : WAVES][TPW][GM == NONE ? 4 : W];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l = lane % LPT, sub = lane / LPT;
  uint32_t* row = rows[GM == NONE ? 0 : wave][sub];
  const int E = g.E;
  uint32_t earlier = 0;  // LANES: bit R, whether lane (l - R) % 16 lies in an earlier group
  if constexpr (GM == LANES) {
#pragma unroll
    for (int r = 1; r < 16; ++r) earlier |= (((l - r) & 15) >> g.gshift < l >> g.gshift ? 1u : 0u) << r;
  }
  const int64_t step = (int64_t)gridDim.x * WAVES * TPW;
  // the loop's bound is the wave's, not the lane's: every lane takes part in
  // the exchanges, those of tokens past T on a copy of the last one
  for (int64_t t0 = ((int64_t)blockIdx.x * WAVES + wave) * TPW; t0 < g.T; t0 += step) {
    const int64_t t = min<int64_t>(t0 + sub, g.T - 1);
    uint32_t o[J];  // the choices' order
    Common common;
    {
      float z[J], p[J];
      load_row<DT, LPT, J>(g.z, t * g.ldz, l, E, -__builtin_inff(), z);
      common = scores<LPT, J>(z, g.sigmoid, p);
      if (g.bias) {
        load_row<DT_F32, LPT, J>(g.bias, 0, l, E, 0.f, z);
#pragma unroll
        for (int j = 0; j < J; ++j) p[j] += z[j];
      }
#pragma unroll
      for (int j = 0; j < J; ++j) o[j] = order_bits(p[j]);
    }
    double key[NL];
    if constexpr (GM == LANES) {
      wave_fence();
      to_lds<LPT, J>(row, l, o);
      wave_fence();
      // from here the lane holds experts l * per ... in a row
      const int e0 = l * g.per;
      uint32_t a = 0, b = 0;
      if (g.per == J) {
#pragma unroll
        for (int j = 0; j < J; ++j) o[j] = row[slot(l * J + j)];
      } else {
#pragma unroll
        for (int j = 0; j < J; ++j) o[j] = j < g.per ? row[slot(e0 + j)] : 0u;
      }
#pragma unroll
      for (int j = 0; j < J; ++j) top2(a, b, o[j]);
      if (g.gshift > 0) {
        const uint32_t oa = partner<0>(a), ob = partner<0>(b);
        top2(a, b, oa);
        b = max(b, ob);
      }
      if (g.gshift > 1) {
        const uint32_t oa = partner<1>(a), ob = partner<1>(b);
        top2(a, b, oa);
        b = max(b, ob);
      }
      if (g.gshift > 2) {
        const uint32_t oa = partner<2>(a), ob = partner<2>(b);
        top2(a, b, oa);
        b = max(b, ob);
      }
      const bool in = groups_before<1>(group_order(a, b, g.gsize), earlier) < g.Gk << g.gshift;
#pragma unroll
      for (int j = 0; j < J; ++j) key[j] = make_key(in ? o[j] : 0u, e0 + j);  // below any expert's where dropped
    } else if constexpr (GM == WALK) {
      wave_fence();
      to_lds<LPT, J>(row, l, o);
      wave_fence();
      uint32_t a = 0, b = 0;
      if (l < g.G)
        for (int i = 0; i < g.gsize; ++i) top2(a, b, row[slot(l * g.gsize + i)]);
      const uint32_t go = l < g.G ? group_order(a, b, g.gsize) : 0u;
      int rank = 0;
      for (int q = 0; q < g.G; ++q) {
        const uint32_t oq = (uint32_t)__shfl((int)go, sub * LPT + q);
        rank += oq > go || (oq == go && q < l);
      }
      const uint64_t vote = __ballot(l < g.G && rank < g.Gk);
      const uint32_t kept = (uint32_t)(vote >> (sub * LPT)) & 0xFFFFu;
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const int e = Lay<LPT, J>::e(l, j);
        const bool in = e < E && ((kept >> (__umul24(e, g.gmagic) >> 20)) & 1u);
        key[j] = make_key(in ? o[j] : 0u, e);
      }
    } else {
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const int e = Lay<LPT, J>::e(l, j);
        key[j] = make_key(e < E ? o[j] : 0u, e);
      }
    }
    lane_list<J, KN>(key);
    merge_lanes<(J < KN ? J : KN), KN, 0, STEPS>(key);
    // lane i takes the i-th of the list
    uint32_t lo = 0;
#pragma unroll
    for (int i = 0; i < KN; ++i) lo = l == i ? (uint32_t)__double_as_longlong(key[i]) : lo;
    const int id = 1023 - (int)(lo & 1023u);
    const bool mine = l < g.k;
    float q = 0.f;
    if (mine) q = score(load_elem(g.z, DT, t * g.ldz + min(id, E - 1)), g.sigmoid, common);
    if (g.renorm) {
      const float s = token_sum<LPT>(q) + RENORM_EPS;
      q = q / s;
    }
    if (mine && t0 + sub < g.T) {
      g.ids[t * g.k + l] = id;
      g.w[t * g.k + l] = g.scale * q;
    }
  }
}

template <int DT, int LPT, int J, bool SIG>
__global__ void __launch_bounds__(64 * WAVES) backward_kernel(Args g) {
  constexpr int TPW = 64 / LPT, W = row_words<LPT, J>(), V = Lay<LPT, J>::V;
  __shared__ __attribute__((aligned(16))) float rows[WAVES][TPW][W];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l = lane % LPT, sub = lane / LPT;
  float* row = rows[wave][sub];
  const int E = g.E;
  const int64_t step = (int64_t)gridDim.x * WAVES * TPW;
  for (int64_t t0 = ((int64_t)blockIdx.x * WAVES + wave) * TPW; t0 < g.T; t0 += step) {
    const int64_t t = min<int64_t>(t0 + sub, g.T - 1);
    const bool mine = l < g.k;
    const int id = mine ? min(max(g.ids[t * g.k + l], 0), E - 1) : 0;
    float d = mine ? g.scale * g.dw[t * g.k + l] : 0.f;
    const float zc = mine ? load_elem(g.z, DT, t * g.ldz + id) : 0.f;
    float p[J], q = 0.f, q1 = 0.f;  // q: the chosen score, q1: 1 - q
    if constexpr (SIG) {
      // only the chosen logits matter
      if (mine) {
        const float ex = exp_f32(-__builtin_fabsf(zc));
        const float r = __builtin_amdgcn_rcpf(1.0f + ex);
        q = zc < 0.f ? ex * r : r;
        q1 = zc < 0.f ? r : ex * r;
      }
#pragma unroll
      for (int j = 0; j < J; ++j) p[j] = 0.f;
    } else {
      float z[J];
      load_row<DT, LPT, J>(g.z, t * g.ldz, l, E, -__builtin_inff(), z);
      const Common c = scores<LPT, J>(z, 0, p);
      if (mine) q = score(zc, 0, c);
    }
    if (g.renorm) {
      // relative to the first chosen one's gradient, so that what all have in common
      // does not cancel: d - sum(d q) / s = c - sum(c q) / s + d0 eps / s for c = d - d0
      const float d0 = g.scale * g.dw[t * g.k], c = mine ? d - d0 : 0.f;
      const float s = token_sum<LPT>(q) + RENORM_EPS;
      const float a = token_sum<LPT>(c * q);
      d = mine ? (c - a / s + d0 * (RENORM_EPS / s)) / s : 0.f;
    }
    float own;  // the gradient at a chosen logit
    if constexpr (SIG) {
      own = d * q * q1;
    } else {
      const float s = token_sum<LPT>(d * q);
      own = q * (d - s);
#pragma unroll
      for (int j = 0; j < J; ++j) p[j] = -p[j] * s;
    }
    wave_fence();
    to_lds<LPT, J>(row, l, p);
    wave_fence();
    if (mine) row[slot(id)] = own;
    wave_fence();
    typedef float vec __attribute__((ext_vector_type(V)));
#pragma unroll
    for (int c = 0; c < J / V; ++c) {
      const vec v = *reinterpret_cast<const vec*>(row + slot(Lay<LPT, J>::e(l, c * V)));
#pragma unroll
      for (int i = 0; i < V; ++i) p[c * V + i] = v[i];
    }
    if (t0 + sub < g.T) store_row<DT, LPT, J>(g.dz, t * g.lddz, l, E, p);
  }
}

static unsigned groups_for(int64_t T, int lpt) {
  const int64_t per = WAVES * (64 / lpt);
  return (unsigned)std::max<int64_t>(1, std::min<int64_t>(cdiv(T, per), split_device_cus() * 16));
}

template <int DT, int LPT, int J, int KN>
static void launch_forward(const Args& g, unsigned n, hipStream_t st) {
  if constexpr (LPT == 16) {
    if (g.G > 1 && g.E % 16 == 0 && 16 % g.G == 0) {
      forward_kernel<DT, LPT, J, KN, LANES><<<n, 64 * WAVES, 0, st>>>(g);
      return;
    }
  }
  if (g.G > 1)
    forward_kernel<DT, LPT, J, KN, WALK><<<n, 64 * WAVES, 0, st>>>(g);
  else
    forward_kernel<DT, LPT, J, KN, NONE><<<n, 64 * WAVES, 0, st>>>(g);
}

template <int DT, int LPT, int J>
static void launch(const Args& a, bool back, hipStream_t st) {
  Args g = a;
  g.per = g.E / 16;
  g.gshift = g.G > 8 ? 0 : g.G > 4 ? 1 : g.G > 2 ? 2 : 3;
  const unsigned n = groups_for(g.T, LPT);
  if (back) {
    if (g.sigmoid)
      backward_kernel<DT, LPT, J, true><<<n, 64 * WAVES, 0, st>>>(g);
    else
      backward_kernel<DT, LPT, J, false><<<n, 64 * WAVES, 0, st>>>(g);
  } else if (g.k <= 4) {
    launch_forward<DT, LPT, J, 4>(g, n, st);
  } else if (g.k <= 8) {
    launch_forward<DT, LPT, J, 8>(g, n, st);
  } else {
    launch_forward<DT, LPT, J, 16>(g, n, st);
  }
}

// 16 lanes of 2 to 16 experts, above 256 experts 64 lanes of 8 or 16
template <int DT>
static void dispatch(const Args& g, bool back, hipStream_t st) {
  if (g.E <= 32)
    launch<DT, 16, 2>(g, back, st);
  else if (g.E <= 64)
    launch<DT, 16, 4>(g, back, st);
  else if (g.E <= 128)
    launch<DT, 16, 8>(g, back, st);
  else if (g.E <= 256)
    launch<DT, 16, 16>(g, back, st);
  else if (g.E <= 512)
    launch<DT, 64, 8>(g, back, st);
  else
    launch<DT, 64, 16>(g, back, st);
}

static int check(const char* fn, const Args& g, int dt) {
  if (!valid_dtype(dt)) return fail(NTLB_EINVAL, "%s: bad dtype %d", fn, dt);
  if (g.T < 0 || g.E < 1 || g.E > MAX_E) return fail(NTLB_EINVAL, "%s: %d experts (1 to %d)", fn, g.E, MAX_E);
  if (g.k < 1 || g.k > MAX_K || g.k > g.E) return fail(NTLB_EINVAL, "%s: top_k %d of %d experts (at most %d)", fn, g.k, g.E, MAX_K);
  if (g.T > 0 && (!g.z || !g.ids)) return fail(NTLB_EINVAL, "%s: NULL pointer", fn);
  if (g.ldz != 0 && g.ldz < g.E) return fail(NTLB_EINVAL, "%s: row pitch %lld below %d", fn, (long long)g.ldz, g.E);
  return NTLB_OK;
}

static int run(const char* fn, const Args& g, int dt, bool back, void* stream) {
  hipStream_t st = as_stream(stream);
  if (dt == NTLB_F32)
    dispatch<DT_F32>(g, back, st);
  else if (dt == NTLB_BF16)
    dispatch<DT_BF16>(g, back, st);
  else
    dispatch<DT_F16>(g, back, st);
  return check_launch(fn);
}

}  // namespace router
}  // namespace ntlb

using namespace ntlb;

extern "C" int ntlb_route_topk(const void* logits, int dtype, int64_t T, int64_t E, int64_t ld, int64_t top_k,
                               int sigmoid, const float* bias, int64_t n_groups, int64_t topk_groups, int renormalize,
                               float scale, int32_t* ids, float* weights, void* stream) {
  const char* fn = "ntlb_route_topk";
  clear_error();
  router::Args g{};
  g.z = logits; g.ldz = ld; g.T = T; g.E = (int)std::min<int64_t>(E, 1 << 30); g.k = (int)std::min<int64_t>(top_k, 1 << 30);
  g.sigmoid = sigmoid != 0; g.renorm = renormalize != 0; g.scale = scale; g.bias = bias; g.ids = ids; g.w = weights;
  if (int rc = router::check(fn, g, dtype)) return rc;
  if (n_groups < 1 || n_groups > router::MAX_G || E % n_groups)
    return fail(NTLB_EINVAL, "%s: %lld groups of %lld experts (equal groups, at most %d)", fn, (long long)n_groups, (long long)E, router::MAX_G);
  if (topk_groups < 1 || topk_groups > n_groups || topk_groups * (E / n_groups) < top_k)
    return fail(NTLB_EINVAL, "%s: %lld of %lld groups cannot give %lld experts", fn, (long long)topk_groups, (long long)n_groups, (long long)top_k);
  if (T == 0) return NTLB_OK;
  if (!weights) return fail(NTLB_EINVAL, "%s: NULL pointer", fn);
  g.G = topk_groups < n_groups ? (int)n_groups : 1;  // all groups kept: no choice of groups
  g.Gk = (int)topk_groups;
  g.gsize = (int)(E / n_groups);
  g.gmagic = (int)cdiv((int64_t)1 << 20, g.gsize);
  return router::run(fn, g, dtype, false, stream);
}

extern "C" int ntlb_route_topk_backward(const void* logits, int dtype, int64_t T, int64_t E, int64_t ld, int64_t top_k,
                                        int sigmoid, int renormalize, float scale, const int32_t* ids, const float* dw,
                                        void* dlogits, int64_t ldd, void* stream) {
  const char* fn = "ntlb_route_topk_backward";
  clear_error();
  router::Args g{};
  g.z = logits; g.ldz = ld; g.T = T; g.E = (int)std::min<int64_t>(E, 1 << 30); g.k = (int)std::min<int64_t>(top_k, 1 << 30);
  g.sigmoid = sigmoid != 0; g.renorm = renormalize != 0; g.scale = scale; g.ids = const_cast<int32_t*>(ids); g.dw = dw;
  g.dz = dlogits; g.lddz = ldd;
  if (int rc = router::check(fn, g, dtype)) return rc;
  if (T == 0) return NTLB_OK;
  if (!dw || !dlogits || ldd < E) return fail(NTLB_EINVAL, "%s: bad dw or dlogits", fn);
  return router::run(fn, g, dtype, true, stream);
}
