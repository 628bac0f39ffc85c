// An activation that keeps its input in 8 bits for the backward pass, and the
// gradient taken from those bits.
//
// The input row (each half of a gated pair) is cut into groups of 128; a group
// keeps int8 codes and one fp32 scale:
//   scale = max(amax / 127, 1e-30),  q = rne(x / scale)      (IEEE divisions)
// a quarter to a half of the bytes of the input.  Forward: y = f(x) from the
// input itself.  Backward: dx = dy f'(q scale).
//   gelu_tanh  f = x s, s = sigmoid(2u), u = sqrt(2/pi) (x + 0.044715 x^3)
//              (0.5 (1 + tanh u) = sigmoid(2u)); f' = s + 2 x s (1 - s) u'
//   silu       f = x s, s = sigmoid(x);          f' = s (1 + x (1 - s))
//   swiglu     f = silu(gate) up for rows [gate | up]
// sigmoid from e = exp(-|z|) alone: s = 1 / (1 + e) or e / (1 + e), and
// s (1 - s) = e / (1 + e)^2, with no cancellation and no overflow.
//
// Both passes read and write every byte once.  At 16 bits they are held by HBM only
// if an element costs fewer than about twenty instructions, hence the arithmetic
// on pairs, and a group in four lanes of 32 elements each (four 16-byte loads in
// flight): the scale's two divisions, the index arithmetic and the shuffles are
// paid once for 32 elements.  With 16 lanes of 8 the forward pass was issue-bound.
// At 5856 x 12288 bf16: GELU forward 78 us (365 MB, 4.7 TB/s), gradient 63 us (364 MB,
// 5.7 TB/s), with issue slots two thirds in use; SwiGLU (rows of 2 x 12288) forward 150 us
// (580 MB, 3.9 TB/s; both halves' chunks take 106 registers a thread, two blocks a
// multiprocessor where GELU has four), gradient 92 us (580 MB, 6.3 TB/s: the rate of a copy).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "pieces.cuh"
#include "quant_common.cuh"
#include "w8a8_internal.h"

namespace w8a8 {
namespace {

constexpr int kThreads = 256;
constexpr int kGroup = 128;
// How a group lies in lanes.
//   kWhole     rows (or halves) of whole groups on vector boundaries, the usual case, in which
//              nothing has to be looked at element by element: lane l of four has the chunks of
//              eight elements l, l + 4, l + 8, l + 12
//   kVectors   the same with a last group that may be shorter
//   kElements  rows that vectors cannot take: lane l of sixteen has the pairs of elements l, l + 16,
//              ..., so that neighbours share the memory sectors that each access touches (GELU,
//              1837 x 2455 bf16, both passes: 72 us with eight neighbouring elements a lane, 19 so);
//              pairs, since two elements share a reciprocal: the bits are those of the others
enum Layout : int { kWhole = 0, kVectors = 1, kElements = 2 };
template <int kLayout>
struct Lay {
  static constexpr int kLanes = kLayout == kElements ? 16 : 4;
  static constexpr int kChunks = kGroup / (8 * kLanes);
  static constexpr int kFirst = kLayout == kElements ? 2 : 8;  // from a lane's first element to the next lane's
  // element i of a lane's chunk
  static __device__ constexpr int at(int i) { return kLayout == kElements ? (i >> 1) * 2 * kLanes + (i & 1) : i; }
};
constexpr int kStep = 32;  // elements from one of a lane's chunks to the next

constexpr float kC0 = 0.7978845608028654f;  // sqrt(2 / pi)
constexpr float kC1 = 0.044715f;
constexpr float kLog2e = 1.4426950408889634f;

enum Act : int { kGelu = 1, kSwiglu = 2, kSilu = 3 };

// ---- fp32: the accurate exponential and an IEEE division
__device__ __forceinline__ void exp_recip(float z, float& e, float& r) {
  e = expf(-fabsf(z));
  r = __fdiv_rn(1.0f, 1.0f + e);
}
// sigmoid's argument and that argument's slope
template <int kAct>
__device__ __forceinline__ void argument(float x, float& z, float& dz) {
  if constexpr (kAct == kGelu) {
    const float x2 = x * x;
    z = 2.0f * kC0 * (x + kC1 * x2 * x);
    dz = 2.0f * kC0 * (1.0f + 3.0f * kC1 * x2);
  } else {
    z = x;
    dz = 1.0f;
  }
}
template <int kAct>
__device__ __forceinline__ float act_one(float x) {
  float z, dz, e, r;
  argument<kAct>(x, z, dz);
  exp_recip(z, e, r);
  return x * (z >= 0.0f ? r : e * r);
}
// The slope of x sigmoid(z(x)), and sigmoid(z) itself.
template <int kAct>
__device__ __forceinline__ float slope_one(float x, float& s) {
  float z, dz, e, r;
  // beyond 16 gelu's second term is below 1e-100 and x^2 may overflow
  const float c = kAct == kGelu ? (x != x ? x : fminf(fmaxf(x, -16.0f), 16.0f)) : x;
  argument<kAct>(c, z, dz);
  exp_recip(z, e, r);
  s = z >= 0.0f ? r : e * r;
  const float t = c * (e * r * r) * dz;
  return s + (fabsf(z) > 200.0f ? 0.0f : t);  // exp(-200) |z|: 0 in fp32; an infinite x times 0
}

// ---- 16-bit types: two elements an instruction (f32x2), approximate
// exponential and reciprocal (2^-22, far below the output's rounding).
__device__ __forceinline__ float ex2(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float rcp(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ uint64_t both(float v) { return pk(v, v); }

// z log2(e)
template <int kAct>
__device__ __forceinline__ uint64_t argument_two(uint64_t x) {
  if constexpr (kAct == kGelu) {
    constexpr float k = 2.0f * kC0 * kLog2e;
    return mul2(x, fma2(mul2(x, x), both(k * kC1), both(k)));
  } else {
    return mul2(x, both(kLog2e));
  }
}
// With e = exp(-|z|): er = e / (1 + e) and r = 1 / (1 + e); the sigmoid is r where z >= 0, else er.
// kApart: one of the two may be NaN and the other not.  The two share a reciprocal, so a
// NaN argument is taken as 0 (fminf drops it) and leaves a finite sigmoid; x itself carries the NaN on.
template <bool kApart>
__device__ __forceinline__ void exp_recip_two(uint64_t z, uint64_t& er, uint64_t& r, uint64_t& s) {
  // the exponential 2^24 too large, so that flushing its subnormals to zero loses
  // nothing that bf16 holds (ftz: one instruction instead of four)
  float e0 = 24.0f - fabsf(lo(z)), e1 = 24.0f - fabsf(hi(z));
  if constexpr (kApart) {
    e0 = fminf(e0, 24.0f);
    e1 = fminf(e1, 24.0f);
  }
  const uint64_t e = mul2(pk(ex2(e0), ex2(e1)), both(5.9604644775390625e-8f));
  const uint64_t d = add2(e, both(1.0f));
  // both reciprocals from that of the product, which lies in [1, 4]: the special
  // function unit (a quarter of the rate) is the busiest
  r = mul2(both(rcp(lo(d) * hi(d))), pk(hi(d), lo(d)));
  er = mul2(e, r);
  s = pk(lo(z) >= 0.0f ? lo(r) : lo(er), hi(z) >= 0.0f ? hi(r) : hi(er));
}
template <int kAct>
__device__ __forceinline__ uint64_t act_two(uint64_t x) {
  uint64_t er, r, s;
  exp_recip_two<true>(argument_two<kAct>(x), er, r, s);
  return mul2(x, s);
}
// The slope of x sigmoid(z(x)), and sigmoid(z) itself.  Both elements are of one group, whose scale
// is NaN for all of it or for none.
template <int kAct>
__device__ __forceinline__ uint64_t slope_two(uint64_t x, uint64_t& s) {
  uint64_t er, r;
  if constexpr (kAct == kGelu) {
    // beyond |x| = 16 the second term is below 1e-100 whatever its factor: x^2 held
    // at 256 keeps the factor finite
    constexpr float k = 2.0f * kC0;
    const uint64_t x2 = mul2(x, x);
    const uint64_t m = pk(fminf(lo(x2), 256.0f), fminf(hi(x2), 256.0f));
    exp_recip_two<false>(mul2(x, fma2(m, both(k * kC1 * kLog2e), both(k * kLog2e))), er, r, s);
    return fma2(mul2(x, mul2(er, r)), fma2(m, both(3.0f * k * kC1), both(k)), s);
  } else {
    exp_recip_two<false>(argument_two<kAct>(x), er, r, s);
    return fma2(x, mul2(er, r), s);
  }
}

// The scale of a group from the bits of its absolute maximum, and its reciprocal.
// A group with an infinity or a NaN keeps NaN as its scale, so that its
// gradient is NaN, and codes of zero.
__device__ __forceinline__ float group_scale(uint32_t amax, float& recip) {
  if (amax >= 0x7F800000u) {
    recip = 0.0f;
    return __uint_as_float(0x7FC00000u);
  }
  const float scale = fmaxf(__fdiv_rn(__uint_as_float(amax), 127.0f), 1.0e-30f);
  recip = __frcp_rn(scale);
  return scale;
}

// Codes of eight elements: rne(x / scale) from the product with the reciprocal,
// which is within 2^-22 of the quotient (below 4e-5 in all): only next to a half does
// the divide decide.  Adding 1.5 * 2^23 rounds to an integer, whose low byte is
// the code.
__device__ __forceinline__ uint2 codes_of(const uint64_t (&v)[4], float scale, float recip) {
  const uint64_t magic = both(12582912.0f);
  uint64_t n[4];
  float off = 0.0f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint64_t y = mul2(v[i], both(recip));
    n[i] = add2(y, magic);
    const uint64_t d = sub2(y, sub2(n[i], magic));
    off = fmaxf(off, fmaxf(fabsf(lo(d)), fabsf(hi(d))));
  }
  if (off > 0.49995f) {
#pragma unroll
    for (int i = 0; i < 4; ++i) n[i] = add2(pk(__fdiv_rn(lo(v[i]), scale), __fdiv_rn(hi(v[i]), scale)), magic);
  }
  uint32_t w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t p = __byte_perm(static_cast<uint32_t>(n[2 * i]), static_cast<uint32_t>(n[2 * i] >> 32), 0x0040);
    const uint32_t q = __byte_perm(static_cast<uint32_t>(n[2 * i + 1]), static_cast<uint32_t>(n[2 * i + 1] >> 32), 0x0040);
    w[i] = __byte_perm(p, q, 0x5410);
  }
  // a spoiled group's codes are 0 (its elements times a reciprocal of 0 may be NaN)
  return scale == scale ? make_uint2(w[0], w[1]) : make_uint2(0, 0);
}

// |x| of eight elements: the largest, as the bits of its fp32 value (NaN is the largest of all).
template <typename T>
__device__ __forceinline__ uint32_t abs_max(const Raw8<T>& r) {
  if constexpr (sizeof(T) == 2) {
    const uint2* u = reinterpret_cast<const uint2*>(r.e);
    const uint32_t k = 0x7FFF7FFFu;
    return __vmaxu2(__vmaxu2(u[0].x & k, u[0].y & k), __vmaxu2(u[1].x & k, u[1].y & k));
  } else {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(r.e[i]) & 0x7FFFFFFFu);
    return m;
  }
}
// The group's, over its lanes.
template <typename T, int kLanes>
__device__ __forceinline__ uint32_t group_max(uint32_t m) {
#pragma unroll
  for (int o = kLanes / 2; o > 0; o >>= 1) {
    const uint32_t other = __shfl_xor_sync(0xffffffffu, m, o);
    m = sizeof(T) == 2 ? __vmaxu2(m, other) : max(m, other);
  }
  if constexpr (sizeof(T) == 2) {
    const uint16_t h = static_cast<uint16_t>(max(m & 0xFFFFu, m >> 16));
    if constexpr (std::is_same<T, __half>::value) {
      m = __float_as_uint(__half2float(__ushort_as_half(h)));
    } else {
      m = static_cast<uint32_t>(h) << 16;
    }
  }
  return m;
}

template <typename T>
__device__ __forceinline__ void widen(uint64_t (&v)[4], const Raw8<T>& r) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      const uint32_t u = reinterpret_cast<const uint32_t*>(r.e)[i];
      v[i] = pk(__uint_as_float(u << 16), __uint_as_float(u & 0xFFFF0000u));
    } else {
      v[i] = pk(to_f(r.e[2 * i]), to_f(r.e[2 * i + 1]));
    }
  }
}
// Eight codes times their scale.  A code's float comes from its byte placed in
// the mantissa of 2^23 (an integer conversion takes a quarter of the rate).
__device__ __forceinline__ void widen_codes(uint64_t (&v)[4], const Raw8<int8_t>& r, float scale) {
  const uint2 u = *reinterpret_cast<const uint2*>(r.e);
  const uint32_t x[2] = {u.x ^ 0x80808080u, u.y ^ 0x80808080u};
  const uint64_t base = both(-8388736.0f);  // -(2^23 + 128)
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t a = __byte_perm(x[i >> 1], 0x4B000000u, (i & 1) ? 0x7542 : 0x7540);
    const uint32_t b = __byte_perm(x[i >> 1], 0x4B000000u, (i & 1) ? 0x7543 : 0x7541);
    v[i] = mul2(add2(pk(__uint_as_float(a), __uint_as_float(b)), base), both(scale));
  }
}

// A lane's chunk; `left`: elements of the row from its first on.
template <int kLayout, typename T>
__device__ __forceinline__ void load_chunk(Raw8<T>& r, const T* p, int left) {
  if constexpr (kLayout == kElements) {
#pragma unroll
    for (int i = 0; i < 8; ++i) r.e[i] = Lay<kLayout>::at(i) < left ? p[Lay<kLayout>::at(i)] : T(0.0f);
  } else {
    load8(r, p, kLayout == kWhole ? (left > 0 ? 8 : 0) : min(8, left), true);
  }
}

template <int kLayout, typename T>
__device__ __forceinline__ void store_two(T* p, const uint64_t (&v)[4], int left) {
  Raw8<T> o;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      reinterpret_cast<uint32_t*>(o.e)[i] = pack_bf16(lo(v[i]), hi(v[i]));
    } else {
      o.e[2 * i] = from_f<T>(lo(v[i]));
      o.e[2 * i + 1] = from_f<T>(hi(v[i]));
    }
  }
  if (kLayout == kWhole || (kLayout == kVectors && left >= 8)) {
#pragma unroll
    for (int q = 0; q < static_cast<int>(sizeof(T) / 2); ++q) {
      const uint2* s = reinterpret_cast<const uint2*>(o.e) + 2 * q;
      reinterpret_cast<uint4*>(p)[q] = make_uint4(s[0].x, s[0].y, s[1].x, s[1].y);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (Lay<kLayout>::at(i) < left) p[Lay<kLayout>::at(i)] = o.e[i];
  }
}

template <int kLayout>
__device__ __forceinline__ void store_codes(int8_t* p, uint2 w, int left) {
  if (kLayout == kWhole || (kLayout == kVectors && left >= 8)) {
    *reinterpret_cast<uint2*>(p) = w;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (Lay<kLayout>::at(i) < left)
        p[Lay<kLayout>::at(i)] = static_cast<int8_t>((i < 4 ? w.x : w.y) >> (8 * (i & 3)));
  }
}

// Quotient of an item number below 2^31 by the number of groups in a row: one wide
// multiplication by m = ceil(2^(31 + l) / d), 2^l >= d, whose excess over the
// true factor is below 2^l and moves no quotient of a number below 2^31.
struct Groups {
  uint32_t count;
  uint64_t m;
  int shift;
  __device__ __forceinline__ uint32_t row_of(uint32_t item) const {
    return static_cast<uint32_t>((static_cast<uint64_t>(item) * m) >> shift);
  }
};
Groups groups_of(int K) {
  Groups g;
  g.count = static_cast<uint32_t>((K + kGroup - 1) / kGroup);
  int l = 0;
  while ((1ull << l) < g.count) ++l;
  g.shift = 31 + l;
  g.m = ((1ull << g.shift) + g.count - 1) / g.count;
  return g;
}

struct Item {
  int64_t row;
  int c;       // the lane's first chunk; chunk j is 32 j further
  int left;    // elements of the row (or half) from c on, 0 for no item
  uint32_t g;
};
template <int kLayout>
__device__ __forceinline__ Item item_at(uint64_t item, uint32_t items, const Groups& groups, int K) {
  Item t;
  const bool live = item < items;
  const uint32_t i = live ? static_cast<uint32_t>(item) : 0;
  const uint32_t row = groups.row_of(i);
  t.row = row;
  t.g = i - row * groups.count;
  t.c = static_cast<int>(t.g) * kGroup + (threadIdx.x % Lay<kLayout>::kLanes) * Lay<kLayout>::kFirst;
  t.left = live ? K - t.c : 0;
  return t;
}

// Forward.  Item = one group of one row (of both halves when gated).  Every lane
// of a warp makes the same number of steps (shuffles).
template <typename T, int kAct, int kLayout>
__global__ void __launch_bounds__(kThreads, kAct == kSwiglu || sizeof(T) == 4 ? 1 : 4) act_checkpoint_kernel(
    const T* __restrict__ x, int64_t ldx, uint32_t items, int K, Groups groups,
    T* __restrict__ y, int8_t* __restrict__ q, float* __restrict__ scale) {
  constexpr int kHalves = kAct == kSwiglu ? 2 : 1;
  constexpr int kLanes = Lay<kLayout>::kLanes, kChunks = Lay<kLayout>::kChunks;
  constexpr uint32_t kPerBlock = kThreads / kLanes;
  const Item it = item_at<kLayout>(static_cast<uint64_t>(blockIdx.x) * kPerBlock + threadIdx.x / kLanes, items, groups, K);
  Raw8<T> raw[kHalves][kChunks];
#pragma unroll
  for (int h = 0; h < kHalves; ++h)
#pragma unroll
    for (int j = 0; j < kChunks; ++j)
      load_chunk<kLayout>(raw[h][j], x + it.row * ldx + h * static_cast<int64_t>(K) + it.c + j * kStep,
                          it.left - j * kStep);
  float s[kHalves], recip[kHalves];
#pragma unroll
  for (int h = 0; h < kHalves; ++h) {
    uint32_t m = abs_max(raw[h][0]);
#pragma unroll
    for (int j = 1; j < kChunks; ++j) {
      const uint32_t o = abs_max(raw[h][j]);
      m = sizeof(T) == 2 ? __vmaxu2(m, o) : max(m, o);
    }
    s[h] = group_scale(group_max<T, kLanes>(m), recip[h]);
    if (it.left > 0 && threadIdx.x % kLanes == 0) scale[(it.row * kHalves + h) * groups.count + it.g] = s[h];
  }
#pragma unroll
  for (int j = 0; j < kChunks; ++j) {
    const int left = it.left - j * kStep;
    if (kLayout == kWhole ? it.left <= 0 : left <= 0) break;
    const int c = it.c + j * kStep;
    uint64_t v[kHalves][4], o[4];
#pragma unroll
    for (int h = 0; h < kHalves; ++h) {
      widen(v[h], raw[h][j]);
      store_codes<kLayout>(q + (it.row * kHalves + h) * K + c, codes_of(v[h], s[h], recip[h]), left);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      constexpr int kOne = kAct == kGelu ? kGelu : kSilu;
      if constexpr (std::is_same<T, float>::value) {
        o[i] = pk(act_one<kOne>(lo(v[0][i])), act_one<kOne>(hi(v[0][i])));
      } else {
        o[i] = act_two<kOne>(v[0][i]);
      }
      if constexpr (kAct == kSwiglu) o[i] = mul2(o[i], v[kHalves - 1][i]);
    }
    store_two<kLayout>(y + it.row * K + c, o, left);
  }
}

// Backward: dx [rows, halves * K] from dy [rows, K] and the checkpoint.
template <typename T, int kAct, int kLayout>
__global__ void __launch_bounds__(kThreads) act_backward_kernel(
    const T* __restrict__ dy, int64_t lddy, uint32_t items, int K, Groups groups,
    const int8_t* __restrict__ q, const float* __restrict__ scale, T* __restrict__ dx) {
  constexpr int kHalves = kAct == kSwiglu ? 2 : 1;
  constexpr int kLanes = Lay<kLayout>::kLanes, kChunks = Lay<kLayout>::kChunks;
  constexpr uint32_t kPerBlock = kThreads / kLanes;
  const Item it = item_at<kLayout>(static_cast<uint64_t>(blockIdx.x) * kPerBlock + threadIdx.x / kLanes, items, groups, K);
  Raw8<T> rd[kChunks];
  Raw8<int8_t> rq[kHalves][kChunks];
  float sc[kHalves];
#pragma unroll
  for (int h = 0; h < kHalves; ++h) sc[h] = __ldg(scale + (it.row * kHalves + h) * groups.count + it.g);
#pragma unroll
  for (int j = 0; j < kChunks; ++j) {
    load_chunk<kLayout>(rd[j], dy + it.row * lddy + it.c + j * kStep, it.left - j * kStep);
#pragma unroll
    for (int h = 0; h < kHalves; ++h)
      load_chunk<kLayout>(rq[h][j], q + (it.row * kHalves + h) * K + it.c + j * kStep, it.left - j * kStep);
  }
#pragma unroll
  for (int j = 0; j < kChunks; ++j) {
    const int left = it.left - j * kStep;
    if (kLayout == kWhole ? it.left <= 0 : left <= 0) break;
    uint64_t d[4], v[kHalves][4], o[kHalves][4];
    widen(d, rd[j]);
#pragma unroll
    for (int h = 0; h < kHalves; ++h) widen_codes(v[h], rq[h][j], sc[h]);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      constexpr int kOne = kAct == kGelu ? kGelu : kSilu;
      uint64_t s, slope;
      if constexpr (std::is_same<T, float>::value) {
        float s0, s1;
        const float a0 = slope_one<kOne>(lo(v[0][i]), s0), a1 = slope_one<kOne>(hi(v[0][i]), s1);
        slope = pk(a0, a1);
        s = pk(s0, s1);
      } else {
        slope = slope_two<kOne>(v[0][i], s);
      }
      if constexpr (kAct == kSwiglu) {
        o[0][i] = mul2(mul2(d[i], v[kHalves - 1][i]), slope);
        o[kHalves - 1][i] = mul2(mul2(d[i], v[0][i]), s);
      } else {
        o[0][i] = mul2(d[i], slope);
      }
    }
#pragma unroll
    for (int h = 0; h < kHalves; ++h)
      store_two<kLayout>(dx + (it.row * kHalves + h) * K + it.c + j * kStep, o[h], left);
  }
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

template <int kLayout>
unsigned blocks_for(int64_t items) {
  const int64_t per = kThreads / Lay<kLayout>::kLanes;
  return static_cast<unsigned>((items + per - 1) / per);  // below 2^31 / 16
}

#define BY_LAYOUT(F, ACT)                \
  if (!vec) F(ACT, kElements);           \
  else if (K % kGroup) F(ACT, kVectors); \
  else F(ACT, kWhole)

int launched(const char* what) {
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) {
    set_error("%s launch failed: %s", what, cudaGetErrorString(e));
    return W8A8_ERR_ACCELERATOR;
  }
  return 0;
}

// Rows a launch takes: item numbers stay below 2^31.
int64_t rows_per_launch(const Groups& g) { return std::max<int64_t>(1, ((1ll << 31) - 1) / g.count); }

template <typename T>
int checkpoint_typed(const void* x, int64_t ldx, int64_t rows, int K, int act, void* y, int8_t* q,
                     float* scale, cudaStream_t stream) {
  const Groups groups = groups_of(K);
  const int64_t halves = act == kSwiglu ? 2 : 1;
  // every group starts on a vector boundary: rows, halves and codes alike
  const int vec = K % 8 == 0 && aligned16(x) && (ldx * static_cast<int64_t>(sizeof(T))) % 16 == 0 &&
                  aligned16(y) && reinterpret_cast<uintptr_t>(q) % 8 == 0;
  const T* xp = static_cast<const T*>(x);
  T* yp = static_cast<T*>(y);
  for (int64_t r = 0; r < rows; r += rows_per_launch(groups)) {
    const uint32_t items = static_cast<uint32_t>(std::min(rows - r, rows_per_launch(groups)) * groups.count);
#define CHECKPOINT(ACT, LAYOUT)                                                                   \
  act_checkpoint_kernel<T, ACT, LAYOUT><<<blocks_for<LAYOUT>(items), kThreads, 0, stream>>>(      \
      xp + r * ldx, ldx, items, K, groups, yp + r * K, q + r * halves * K,                   \
      scale + r * halves * groups.count)
    switch (act) {
      case kGelu: BY_LAYOUT(CHECKPOINT, kGelu); break;
      case kSilu: BY_LAYOUT(CHECKPOINT, kSilu); break;
      default: BY_LAYOUT(CHECKPOINT, kSwiglu); break;
    }
#undef CHECKPOINT
    if (int rc = launched("act_checkpoint")) return rc;
  }
  return 0;
}

template <typename T>
int backward_typed(const void* dy, int64_t lddy, int64_t rows, int K, int act, const int8_t* q,
                   const float* scale, void* dx, cudaStream_t stream) {
  const Groups groups = groups_of(K);
  const int64_t halves = act == kSwiglu ? 2 : 1;
  const int vec = K % 8 == 0 && aligned16(dy) && (lddy * static_cast<int64_t>(sizeof(T))) % 16 == 0 &&
                  aligned16(dx) && reinterpret_cast<uintptr_t>(q) % 8 == 0;
  const T* dp = static_cast<const T*>(dy);
  T* xp = static_cast<T*>(dx);
  for (int64_t r = 0; r < rows; r += rows_per_launch(groups)) {
    const uint32_t items = static_cast<uint32_t>(std::min(rows - r, rows_per_launch(groups)) * groups.count);
#define BACKWARD(ACT, LAYOUT)                                                                   \
  act_backward_kernel<T, ACT, LAYOUT><<<blocks_for<LAYOUT>(items), kThreads, 0, stream>>>(      \
      dp + r * lddy, lddy, items, K, groups, q + r * halves * K,                             \
      scale + r * halves * groups.count, xp + r * halves * K)
    switch (act) {
      case kGelu: BY_LAYOUT(BACKWARD, kGelu); break;
      case kSilu: BY_LAYOUT(BACKWARD, kSilu); break;
      default: BY_LAYOUT(BACKWARD, kSwiglu); break;
    }
#undef BACKWARD
    if (int rc = launched("act_backward")) return rc;
  }
  return 0;
}

}  // namespace

int act_checkpoint_launch(const void* x, int dtype, int64_t ldx, int64_t rows, int64_t cols, int act,
                          void* y, int8_t* q, float* scale, cudaStream_t stream) {
  const int K = static_cast<int>(cols);
  switch (dtype) {
    case W8A8_BF16: return checkpoint_typed<__nv_bfloat16>(x, ldx, rows, K, act, y, q, scale, stream);
    case W8A8_F16: return checkpoint_typed<__half>(x, ldx, rows, K, act, y, q, scale, stream);
    default: return checkpoint_typed<float>(x, ldx, rows, K, act, y, q, scale, stream);
  }
}

int act_backward_launch(const void* dy, int dtype, int64_t lddy, int64_t rows, int64_t cols, int act,
                        const int8_t* q, const float* scale, void* dx, cudaStream_t stream) {
  const int K = static_cast<int>(cols);
  switch (dtype) {
    case W8A8_BF16: return backward_typed<__nv_bfloat16>(dy, lddy, rows, K, act, q, scale, dx, stream);
    case W8A8_F16: return backward_typed<__half>(dy, lddy, rows, K, act, q, scale, dx, stream);
    default: return backward_typed<float>(dy, lddy, rows, K, act, q, scale, dx, stream);
  }
}

}  // namespace w8a8
