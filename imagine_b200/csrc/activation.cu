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
// Both passes read and write every byte once and are bound by HBM: a group is
// 16 lanes of 8 elements (one 16-byte load a lane at 16 bits), so the absolute
// maximum is four shuffles.
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
constexpr int kLanes = 16;  // lanes per group, eight elements each

// e = exp(-|z|) and r = 1 / (1 + e).  The 16-bit types take the approximate
// exponential and reciprocal (2^-21, far below their rounding).
template <typename T>
__device__ __forceinline__ void exp_recip(float z, float& e, float& r) {
  if constexpr (std::is_same<T, float>::value) {
    e = expf(-fabsf(z));
    r = __fdiv_rn(1.0f, 1.0f + e);
  } else {
    e = __expf(-fabsf(z));
    r = __fdividef(1.0f, 1.0f + e);
  }
}

constexpr float kC0 = 0.7978845608028654f;  // sqrt(2 / pi)
constexpr float kC1 = 0.044715f;

template <typename T>
__device__ __forceinline__ float gelu(float x) {
  float e, r;
  const float z = 2.0f * kC0 * (x + kC1 * x * x * x);
  exp_recip<T>(z, e, r);
  return x * (z >= 0.0f ? r : e * r);
}
template <typename T>
__device__ __forceinline__ float gelu_slope(float x) {
  float e, r;
  const float x2 = x * x;
  const float z = 2.0f * kC0 * (x + kC1 * x2 * x);
  exp_recip<T>(z, e, r);
  const float s = z >= 0.0f ? r : e * r;
  // beyond |x| = 16 the second term is below 1e-100; x2 may overflow there
  const float t = fabsf(x) > 16.0f ? 0.0f : x * e * r * r * (2.0f * kC0) * (1.0f + 3.0f * kC1 * x2);
  return x != x ? x : s + t;
}
template <typename T>
__device__ __forceinline__ float silu(float x) {
  float e, r;
  exp_recip<T>(x, e, r);
  return x * (x >= 0.0f ? r : e * r);
}
// sigmoid(x) and the slope of silu
template <typename T>
__device__ __forceinline__ float silu_slope(float x, float& s) {
  float e, r;
  exp_recip<T>(x, e, r);
  s = x >= 0.0f ? r : e * r;
  const float other = x >= 0.0f ? e * r : r;  // 1 - s
  return s + x * s * other;
}

enum Act : int { kGelu = 1, kSwiglu = 2, kSilu = 3 };

// One group (this thread's eight elements v): codes and scale.  A group with
// an infinity or a NaN keeps NaN as its scale, so that its gradient is NaN.
__device__ __forceinline__ uint2 quant_group(const float (&v)[8], float& scale) {
  // as integers, so that NaN is the largest
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7FFFFFFFu);
#pragma unroll
  for (int o = kLanes / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (m >= 0x7F800000u) {
    scale = __uint_as_float(0x7FC00000u);
    return make_uint2(0, 0);
  }
  scale = fmaxf(__fdiv_rn(__uint_as_float(m), 127.0f), 1.0e-30f);
  const float recip = __frcp_rn(scale);
  uint32_t w[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    // rne(x / scale) from the product with the reciprocal, which is within
    // 2^-22 of the quotient (below 4e-5): only next to a half does the divide decide
    const float y = v[i] * recip;
    const float n = rintf(y);
    int q = static_cast<int>(n);
    if (fabsf(y - n) > 0.4999f) q = __float2int_rn(__fdiv_rn(v[i], scale));
    w[i >> 2] |= static_cast<uint32_t>(q & 0xFF) << (8 * (i & 3));
  }
  return make_uint2(w[0], w[1]);
}

template <typename T>
__device__ __forceinline__ void store8_out(T* p, const float (&v)[8], int valid, bool vec) {
  Raw8<T> o;
#pragma unroll
  for (int i = 0; i < 8; ++i) o.e[i] = from_f<T>(v[i]);
  if (vec && valid >= 8) {
#pragma unroll
    for (int q = 0; q < static_cast<int>(sizeof(T) / 2); ++q) {
      const uint2* s = reinterpret_cast<const uint2*>(o.e) + 2 * q;
      reinterpret_cast<uint4*>(p)[q] = make_uint4(s[0].x, s[0].y, s[1].x, s[1].y);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < valid) p[i] = o.e[i];
  }
}

__device__ __forceinline__ void store_codes(int8_t* p, uint2 w, int valid, bool vec) {
  if (vec && valid >= 8) {
    *reinterpret_cast<uint2*>(p) = w;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < valid) p[i] = static_cast<int8_t>((i < 4 ? w.x : w.y) >> (8 * (i & 3)));
  }
}

template <typename T>
__device__ __forceinline__ void load_f8(float (&v)[8], const T* p, int valid, bool vec) {
  Raw8<T> r;
  load8(r, p, valid, vec);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = to_f(r.e[i]);
}

// Forward.  Item = one group of one row (of both halves when gated); 16 lanes each.
template <typename T, int kAct>
__global__ void __launch_bounds__(kThreads) act_checkpoint_kernel(
    const T* __restrict__ x, int64_t ldx, int64_t rows, int K, int groups, int vec, T* __restrict__ y,
    int8_t* __restrict__ q, float* __restrict__ scale) {
  constexpr int kHalves = kAct == kSwiglu ? 2 : 1;
  const int64_t items = rows * groups;
  const int sub = threadIdx.x % kLanes;
  // whole half-warps pair up: both run the same number of steps (shuffles)
  for (int64_t base = static_cast<int64_t>(blockIdx.x) * (kThreads / kLanes); base < items;
       base += static_cast<int64_t>(gridDim.x) * (kThreads / kLanes)) {
    const int64_t item = base + threadIdx.x / kLanes;
    const bool live = item < items;
    const int64_t row = live ? item / groups : 0;
    const int g = live ? static_cast<int>(item - row * groups) : 0;
    const int c = g * kGroup + sub * 8;
    const int valid = live ? min(8, K - c) : 0;
    float v[kHalves][8];
#pragma unroll
    for (int h = 0; h < kHalves; ++h) load_f8(v[h], x + row * ldx + h * static_cast<int64_t>(K) + c, valid, vec != 0);
#pragma unroll
    for (int h = 0; h < kHalves; ++h) {
      float s;
      const uint2 w = quant_group(v[h], s);
      if (valid > 0) store_codes(q + (row * kHalves + h) * K + c, w, valid, vec != 0);
      if (live && sub == 0) scale[(row * kHalves + h) * groups + g] = s;
    }
    float o[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if constexpr (kAct == kGelu) o[i] = gelu<T>(v[0][i]);
      if constexpr (kAct == kSilu) o[i] = silu<T>(v[0][i]);
      if constexpr (kAct == kSwiglu) o[i] = silu<T>(v[0][i]) * v[kHalves - 1][i];
    }
    if (valid > 0) store8_out(y + row * K + c, o, valid, vec != 0);
  }
}

// Backward: dx [rows, halves * K] from dy [rows, K] and the checkpoint.
template <typename T, int kAct>
__global__ void __launch_bounds__(kThreads) act_backward_kernel(
    const T* __restrict__ dy, int64_t lddy, int64_t rows, int K, int groups, int vec,
    const int8_t* __restrict__ q, const float* __restrict__ scale, T* __restrict__ dx) {
  constexpr int kHalves = kAct == kSwiglu ? 2 : 1;
  const int64_t items = rows * groups;
  const int sub = threadIdx.x % kLanes;
  for (int64_t item = static_cast<int64_t>(blockIdx.x) * (kThreads / kLanes) + threadIdx.x / kLanes;
       item < items; item += static_cast<int64_t>(gridDim.x) * (kThreads / kLanes)) {
    const int64_t row = item / groups;
    const int g = static_cast<int>(item - row * groups);
    const int c = g * kGroup + sub * 8;
    const int valid = min(8, K - c);
    if (valid <= 0) continue;
    float d[8], v[kHalves][8], o[kHalves][8];
    load_f8(d, dy + row * lddy + c, valid, vec != 0);
#pragma unroll
    for (int h = 0; h < kHalves; ++h) {
      load_f8(v[h], q + (row * kHalves + h) * K + c, valid, vec != 0);
      const float s = __ldg(scale + (row * kHalves + h) * groups + g);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[h][i] *= s;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if constexpr (kAct == kGelu) o[0][i] = d[i] * gelu_slope<T>(v[0][i]);
      if constexpr (kAct == kSilu) {
        float s;
        o[0][i] = d[i] * silu_slope<T>(v[0][i], s);
      }
      if constexpr (kAct == kSwiglu) {
        float s;
        const float slope = silu_slope<T>(v[0][i], s);
        o[0][i] = d[i] * v[kHalves - 1][i] * slope;
        o[kHalves - 1][i] = d[i] * v[0][i] * s;
      }
    }
#pragma unroll
    for (int h = 0; h < kHalves; ++h)
      store8_out(dx + (row * kHalves + h) * K + c, o[h], valid, vec != 0);
  }
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

unsigned blocks_for(int64_t items) {
  const int64_t need = (items + kThreads / kLanes - 1) / (kThreads / kLanes);
  return static_cast<unsigned>(std::min<int64_t>(need, 32ll * device_sm_count()));
}

int launched(const char* what) {
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) {
    set_error("%s launch failed: %s", what, cudaGetErrorString(e));
    return W8A8_ERR_ACCELERATOR;
  }
  return 0;
}

template <typename T>
int checkpoint_typed(const void* x, int64_t ldx, int64_t rows, int K, int act, void* y, int8_t* q,
                     float* scale, cudaStream_t stream) {
  const int groups = (K + kGroup - 1) / kGroup;
  // every group starts on a vector boundary: rows, halves and codes alike
  const int vec = K % 8 == 0 && aligned16(x) && (ldx * static_cast<int64_t>(sizeof(T))) % 16 == 0 &&
                  aligned16(y) && reinterpret_cast<uintptr_t>(q) % 8 == 0;
  const unsigned grid = blocks_for(rows * groups);
  const T* xp = static_cast<const T*>(x);
  T* yp = static_cast<T*>(y);
  switch (act) {
    case kGelu: act_checkpoint_kernel<T, kGelu><<<grid, kThreads, 0, stream>>>(xp, ldx, rows, K, groups, vec, yp, q, scale); break;
    case kSilu: act_checkpoint_kernel<T, kSilu><<<grid, kThreads, 0, stream>>>(xp, ldx, rows, K, groups, vec, yp, q, scale); break;
    default: act_checkpoint_kernel<T, kSwiglu><<<grid, kThreads, 0, stream>>>(xp, ldx, rows, K, groups, vec, yp, q, scale); break;
  }
  return launched("act_checkpoint");
}

template <typename T>
int backward_typed(const void* dy, int64_t lddy, int64_t rows, int K, int act, const int8_t* q,
                   const float* scale, void* dx, cudaStream_t stream) {
  const int groups = (K + kGroup - 1) / kGroup;
  const int vec = K % 8 == 0 && aligned16(dy) && (lddy * static_cast<int64_t>(sizeof(T))) % 16 == 0 &&
                  aligned16(dx) && reinterpret_cast<uintptr_t>(q) % 8 == 0;
  const unsigned grid = blocks_for(rows * groups);
  const T* dp = static_cast<const T*>(dy);
  T* xp = static_cast<T*>(dx);
  switch (act) {
    case kGelu: act_backward_kernel<T, kGelu><<<grid, kThreads, 0, stream>>>(dp, lddy, rows, K, groups, vec, q, scale, xp); break;
    case kSilu: act_backward_kernel<T, kSilu><<<grid, kThreads, 0, stream>>>(dp, lddy, rows, K, groups, vec, q, scale, xp); break;
    default: act_backward_kernel<T, kSwiglu><<<grid, kThreads, 0, stream>>>(dp, lddy, rows, K, groups, vec, q, scale, xp); break;
  }
  return launched("act_backward");
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
