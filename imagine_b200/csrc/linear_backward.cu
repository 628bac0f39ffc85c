// Gradient of the W8A8 linear's input: dx[m, k] = sum_n dy[m, n] ws[n] w[n, k].
//
// The codes w are exact in bf16, so the product runs as bf16 x bf16 -> fp32
// with the weight scales folded into dy: dy ws, an fp32 product, is cut into
// one bf16 piece for a bf16 dy (one rounding of 2^-9, as a dequantised bf16
// weight would have), two for f16 and three for fp32 (pieces.cuh), which keeps
// each type's own precision.
//
// Tile: 64 rows x 128 columns, 64 of the contraction a step, 8 warps (four of
// 16 rows, two of 64 columns).  With few tiles the contraction is cut over
// blocks and the fp32 partial sums are added in a fixed order.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "pieces.cuh"
#include "w8a8_internal.h"

namespace w8a8 {
namespace {

constexpr int kThreads = 256;
constexpr int kBM = 64, kBC = 128, kBN = 64;
constexpr int kLdA = kBN + 8, kLdB = kBC + 8;

template <typename T>
__global__ void __launch_bounds__(kThreads) input_grad_kernel(
    const T* __restrict__ dy, int64_t lddy, const float* __restrict__ ws, int ws_one,
    const int8_t* __restrict__ w, int64_t ldw, int64_t M, int N, int K, int col_tiles, int n_split,
    int vec_dy, int vec_w, int vec_o, T* __restrict__ dx, int64_t lddx, float* __restrict__ part) {
  constexpr int kP = Pieces<T>::n;
  constexpr int kPlane = kBM * kLdA;
  constexpr bool kApart = std::is_same<T, float>::value;
  extern __shared__ __align__(16) uint8_t smem[];
  __nv_bfloat16* sa = reinterpret_cast<__nv_bfloat16*>(smem);
  __nv_bfloat16* sb = sa + kP * kPlane;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int wm = warp & 3, wn = warp >> 2;
  const int64_t row0 = static_cast<int64_t>(blockIdx.x / col_tiles) * kBM;
  const int col0 = static_cast<int>(blockIdx.x % col_tiles) * kBC;
  const int n_lo = blockIdx.y * n_split, n_hi = min(N, n_lo + n_split);

  float acc[8][4];
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = 0.0f;
  float low[kApart ? 8 : 1][4] = {};

  Raw8<T> ra[2];
  float rs[2][8];
  Raw8<int8_t> rb[4];
  auto fetch = [&](int n0) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int gi = tid + i * kThreads;
      const int r = gi >> 3, c = (gi & 7) * 8;
      const int valid = row0 + r < M ? min(8, n_hi - n0 - c) : 0;
      load8(ra[i], dy + (row0 + r) * lddy + n0 + c, valid, vec_dy != 0);
#pragma unroll
      for (int j = 0; j < 8; ++j) rs[i][j] = j < valid ? __ldg(ws + (ws_one ? 0 : n0 + c + j)) : 0.0f;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int gi = tid + i * kThreads;
      const int r = gi >> 4, c = (gi & 15) * 8;
      const int valid = n0 + r < n_hi ? min(8, K - col0 - c) : 0;
      load8(rb[i], w + (n0 + r) * ldw + col0 + c, valid, vec_w != 0);
    }
  };
  fetch(n_lo);
  for (int n0 = n_lo; n0 < n_hi; n0 += kBN) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int gi = tid + i * kThreads;
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = to_f(ra[i].e[j]) * rs[i][j];
      store_pieces<kP>(sa + (gi >> 3) * kLdA + (gi & 7) * 8, kPlane, v);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int gi = tid + i * kThreads;
      store8(sb + (gi >> 4) * kLdB + (gi & 15) * 8, 0, rb[i]);
    }
    __syncthreads();
    if (n0 + kBN < n_hi) fetch(n0 + kBN);
#pragma unroll
    for (int kk = 0; kk < kBN; kk += 16) {
      uint32_t a[kP][4];
#pragma unroll
      for (int p = 0; p < kP; ++p) ldsm4(a[p], at16(sa + p * kPlane, wm * 16, kk, kLdA, lane));
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        uint32_t b[4];
        ldsm4_t(b, at16(sb, kk, wn * 64 + n * 16, kLdB, lane));
#pragma unroll
        for (int p = 0; p < kP; ++p) {
          if constexpr (kApart) {
            mma_apart(acc[2 * n], low[2 * n], a[p], b[0], b[1], p == 0);
            mma_apart(acc[2 * n + 1], low[2 * n + 1], a[p], b[2], b[3], p == 0);
          } else {
            mma(acc[2 * n], a[p], b[0], b[1]);
            mma(acc[2 * n + 1], a[p], b[2], b[3]);
          }
        }
      }
    }
  }
  if constexpr (kApart) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] += low[i][j];
  }
#pragma unroll
  for (int n = 0; n < 8; ++n)
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int64_t row = row0 + wm * 16 + (lane >> 2) + half * 8;
      const int c = col0 + wn * 64 + n * 8 + (lane & 3) * 2;
      if (row >= M) continue;
      const float v0 = acc[n][2 * half], v1 = acc[n][2 * half + 1];
      if (part) {
        float* p = part + (blockIdx.y * M + row) * K + c;
        if (c < K) p[0] = v0;
        if (c + 1 < K) p[1] = v1;
      } else {
        T* p = dx + row * lddx + c;
        if (vec_o && c + 1 < K) {
          T two[2] = {from_f<T>(v0), from_f<T>(v1)};
          if constexpr (sizeof(T) == 2) {
            *reinterpret_cast<uint32_t*>(p) = *reinterpret_cast<const uint32_t*>(two);
          } else {
            *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(two);
          }
        } else {
          if (c < K) p[0] = from_f<T>(v0);
          if (c + 1 < K) p[1] = from_f<T>(v1);
        }
      }
    }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) sum_parts_kernel(const float* __restrict__ part,
                                                             int parts, int64_t M, int K,
                                                             T* __restrict__ dx, int64_t lddx) {
  const int64_t total = M * K;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; i < total;
       i += static_cast<int64_t>(gridDim.x) * kThreads) {
    float v = 0.0f;
    for (int p = 0; p < parts; ++p) v += __ldg(part + p * total + i);
    const int64_t row = i / K;
    dx[row * lddx + (i - row * K)] = from_f<T>(v);
  }
}

// Blocks for two a multiprocessor, at least four steps each, at most 16 pieces.
struct NSplit {
  int count, per;
};
NSplit n_split_of(int64_t M, int64_t N, int64_t K) {
  const int64_t tiles = ((M + kBM - 1) / kBM) * ((K + kBC - 1) / kBC);
  const int64_t steps = std::max<int64_t>(1, (N + kBN - 1) / kBN);
  int64_t want = (2ll * device_sm_count() + tiles - 1) / std::max<int64_t>(1, tiles);
  want = std::max<int64_t>(1, std::min<int64_t>({want, 16, steps / 4}));
  const int64_t per = (steps + want - 1) / want;
  return {static_cast<int>((steps + per - 1) / per), static_cast<int>(per * kBN)};
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
int typed(const InputGradArgs& g, cudaStream_t stream) {
  const int N = static_cast<int>(g.N), K = static_cast<int>(g.K);
  const NSplit sp = n_split_of(g.M, g.N, g.K);
  auto al = [](const void* p, int64_t bytes, int unit) {
    return reinterpret_cast<uintptr_t>(p) % unit == 0 && bytes % unit == 0;
  };
  const int64_t size = sizeof(T);
  const int vdy = al(g.dy, g.lddy * size, 16), vw = al(g.w, g.ldw, 8);
  const int vo = al(g.dx, g.lddx * size, 2 * sizeof(T));
  const int cols = (K + kBC - 1) / kBC;
  const int64_t tiles = (g.M + kBM - 1) / kBM;
  float* part = sp.count > 1 ? static_cast<float*>(g.workspace) : nullptr;
  constexpr int bytes = 2 * (Pieces<T>::n * kBM * kLdA + kBN * kLdB);
  static_assert(bytes <= 48 * 1024, "no opt-in shared memory needed");
  const dim3 grid(static_cast<unsigned>(tiles * cols), sp.count);
  input_grad_kernel<T><<<grid, kThreads, bytes, stream>>>(
      static_cast<const T*>(g.dy), g.lddy, g.ws, g.ws_numel == 1, g.w, g.ldw, g.M, N, K, cols, sp.per,
      vdy, vw, vo, static_cast<T*>(g.dx), g.lddx, part);
  if (int rc = launched("input gradient")) return rc;
  if (part) {
    const int64_t blocks =
        std::min<int64_t>((g.M * K + kThreads - 1) / kThreads, 16ll * device_sm_count());
    sum_parts_kernel<T><<<static_cast<unsigned>(blocks), kThreads, 0, stream>>>(
        part, sp.count, g.M, K, static_cast<T*>(g.dx), g.lddx);
    return launched("input gradient sum");
  }
  return 0;
}

}  // namespace

int64_t input_grad_workspace_bytes(int64_t M, int64_t N, int64_t K, int dtype) {
  (void)dtype;
  const NSplit sp = n_split_of(M, N, K);
  return sp.count > 1 ? sp.count * M * K * 4 : 0;
}

int input_grad_launch(const InputGradArgs& g, cudaStream_t stream) {
  switch (g.dtype) {
    case W8A8_BF16: return typed<__nv_bfloat16>(g, stream);
    case W8A8_F16: return typed<__half>(g, stream);
    default: return typed<float>(g, stream);
  }
}

}  // namespace w8a8
