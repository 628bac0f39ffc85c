// bf16 pieces of wider values, and the tensor-core fragments made of them:
// shared by the kernels that multiply f16, fp32 or int8 values (and fp32 sums)
// as bf16 x bf16 -> fp32.
//
// A value is cut into pieces of eight significant bits that add up to it: an
// f16 value into two, an fp32 value into three, both exactly; an int8 code is
// one.  Of the products of two values' pieces those below the last kept bit
// are dropped (pair()).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>
#include <type_traits>

namespace w8a8 {

// bf16 pieces of a value of type T
template <typename T>
struct Pieces;
template <>
struct Pieces<__nv_bfloat16> { static constexpr int n = 1; };
template <>
struct Pieces<int8_t> { static constexpr int n = 1; };
template <>
struct Pieces<__half> { static constexpr int n = 2; };
template <>
struct Pieces<float> { static constexpr int n = 3; };

// Whether the product of piece i of one factor and piece j of the other counts:
// pieces fall by 2^-8 each, the longer factor has `most` of them.
__host__ __device__ constexpr bool pair(int i, int j, int most) { return i + j < most; }

__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(int8_t v) { return static_cast<float>(v); }

template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ __nv_bfloat16 from_f(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ float from_f(float v) { return v; }

// Eight elements of a row in registers.
template <typename T>
struct alignas(8) Raw8 {
  T e[8];
};

template <typename T>
__device__ __forceinline__ void load8(Raw8<T>& r, const T* p, int valid, bool vec) {
  if (vec && valid >= 8) {
    if constexpr (sizeof(T) == 1) {
      *reinterpret_cast<uint2*>(r.e) = __ldg(reinterpret_cast<const uint2*>(p));
    } else {
#pragma unroll
      for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) {
        const uint4 v = __ldg(reinterpret_cast<const uint4*>(p) + i);
        uint2* d = reinterpret_cast<uint2*>(r.e) + 2 * i;
        d[0] = make_uint2(v.x, v.y);
        d[1] = make_uint2(v.z, v.w);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) r.e[i] = i < valid ? p[i] : T(0.0f);
  }
}

__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// The next bf16 piece of v (v rounded to eight significant bits), v becoming the
// rest, which is exact.  A finite value that would round to infinity is cut off
// instead; infinity and NaN go whole into the first piece.
__device__ __forceinline__ float next_piece(float& v) {
  float hi = __bfloat162float(__float2bfloat16_rn(v));
  if (!(fabsf(hi) <= 3.402823466e38f)) {
    if (!(fabsf(v) <= 3.402823466e38f)) {
      const float all = v;
      v = 0.0f;
      return all;
    }
    hi = __uint_as_float(__float_as_uint(v) & 0xFFFF0000u);
  }
  v = v - hi;
  return hi;
}

// Eight values into `n` planes of shared memory, `plane` elements apart.
template <int n>
__device__ __forceinline__ void store_pieces(__nv_bfloat16* dst, int plane, float (&v)[8]) {
#pragma unroll
  for (int p = 0; p < n; ++p) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (p + 1 < n) {
        const float a = next_piece(v[2 * i]);
        const float b = next_piece(v[2 * i + 1]);
        w[i] = pack_bf16(a, b);
      } else {
        w[i] = pack_bf16(v[2 * i], v[2 * i + 1]);
      }
    }
    *reinterpret_cast<uint4*>(dst + p * plane) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

template <typename T>
__device__ __forceinline__ void store8(__nv_bfloat16* dst, int plane, const Raw8<T>& r) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    const uint2* s = reinterpret_cast<const uint2*>(r.e);
    *reinterpret_cast<uint4*>(dst) = make_uint4(s[0].x, s[0].y, s[1].x, s[1].y);
  } else {
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = to_f(r.e[i]);
    store_pieces<Pieces<T>::n>(dst, plane, v);
  }
}

// ---- tensor-core fragments
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], const __nv_bfloat16* p) {
  const uint32_t a = static_cast<uint32_t>(__cvta_generic_to_shared(p));
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(a));
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], const __nv_bfloat16* p) {
  const uint32_t a = static_cast<uint32_t>(__cvta_generic_to_shared(p));
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(a));
}
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// The same for one pair of pieces of fp32 data.  The tensor core cuts low bits off as
// it adds, always towards zero: over a long contraction a bias of 1e-5.  The
// first pieces' product is therefore summed alone and added with rounding; the
// others, 2^-8 of it, run on in `low`.
__device__ __forceinline__ void mma_apart(float (&d)[4], float (&low)[4], const uint32_t (&a)[4],
                                          uint32_t b0, uint32_t b1, bool first) {
  if (first) {
    float one[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    mma(one, a, b0, b1);
#pragma unroll
    for (int j = 0; j < 4; ++j) d[j] += one[j];
  } else {
    mma(low, a, b0, b1);
  }
}
// Addresses of the four 8 x 8 blocks of a 16 x 16 block at (row, col) of a
// row-major tile with row stride ld: lane l points at row l % 16, column half
// l / 16 (blocks in the order rows 0-7, rows 8-15, then the right half).
__device__ __forceinline__ const __nv_bfloat16* at16(const __nv_bfloat16* t, int row, int col, int ld,
                                                     int lane) {
  return t + (row + (lane & 15)) * ld + col + (lane >> 4) * 8;
}
// The same with the halves first: blocks (rows 0-7, left), (rows 0-7, right), (rows 8-15, left), ...
__device__ __forceinline__ const __nv_bfloat16* at16h(const __nv_bfloat16* t, int row, int col, int ld,
                                                      int lane) {
  return t + (row + (lane & 7) + (lane >> 4) * 8) * ld + col + ((lane >> 3) & 1) * 8;
}

}  // namespace w8a8
