// Gradient of the W8A8 linear's input: dx[m, k] = sum_n dy[m, n] ws[n] w[n, k].
//
// The products run as bf16 x bf16 -> fp32; the codes w are exact in bf16.  Where the weight
// scales go:
//   f16, fp32   into dy: the fp32 product dy ws is cut into two or three bf16 pieces
//               (pieces.cuh), which keeps the type's own precision
//   bf16        one scale for all: onto the fp32 sum, and nothing is rounded on the way.
//               A scale a row: into the weight, bf16(w ws), a dequantised bf16 weight,
//               off by 2^-8 of itself at most.  Two pieces of dy ws would keep it exact and cost
//               as many products again (5856 x 12288 -> 4096 takes 400 us of them).  All
//               kernels below round the same value, so that a row's gradient does not
//               depend on which of them its batch goes to, but for the order of the fp32 sum.
//
// Three kernels:
//   input_grad_few_kernel  up to 16 rows: w from HBM straight into mma.sync fragments
//   input_grad_tc_kernel   16-bit types: tcgen05, pairs of CTAs on 256 x 256 tiles
//   input_grad_kernel      mma.sync tiles of 64 rows x 128 columns, for the rest: fp32
//                          (whose sums the tensor cores' long runs would bias),
//                          rows that the others cannot load
// With few tiles the contraction is cut over blocks and the fp32 partial sums
// are added in a fixed order.
#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cstdint>
#include <mutex>
#include <type_traits>

#include "lora_rows.cuh"
#include "pieces.cuh"
#include "quant_common.cuh"
#include "sm100_ptx.cuh"
#include "w8a8_internal.h"

namespace w8a8 {

// Why a bounded wait of input_grad_tc_kernel gave up (DeviceError).
__device__ int g_input_grad_error;

int read_and_clear_input_grad_error(cudaStream_t stream, int* value) {
  int v = 0;
  cudaError_t e = cudaMemcpyFromSymbolAsync(&v, g_input_grad_error, sizeof(int), 0,
                                            cudaMemcpyDeviceToHost, stream);
  if (e == cudaSuccess) e = cudaStreamSynchronize(stream);
  if (e != cudaSuccess) return static_cast<int>(e);
  if (v != 0) {
    const int zero = 0;
    e = cudaMemcpyToSymbolAsync(g_input_grad_error, &zero, sizeof(int), 0, cudaMemcpyHostToDevice,
                                stream);
    if (e == cudaSuccess) e = cudaStreamSynchronize(stream);
    if (e != cudaSuccess) return static_cast<int>(e);
  }
  *value = v;
  return 0;
}

namespace {

constexpr int kThreads = 256;
constexpr int kBC = 128, kBN = 64;
constexpr int kLdA = kBN + 8, kLdB = kBC + 8;

// Two blocks a multiprocessor.  With 173 registers an fp32 call had one, and the
// blocks of a cut contraction ran in two waves (712 x 5584 -> 1152: 294 us, now 201).
// Whether the weight's scale is folded into the weight (or, a single one, put on the sum).
template <typename T>
constexpr bool kScaleWeight = std::is_same<T, __nv_bfloat16>::value;

template <typename T>
__global__ void __launch_bounds__(kThreads, 2) input_grad_kernel(
    const T* __restrict__ dy, int64_t lddy, const float* __restrict__ ws, int ws_one,
    const int8_t* __restrict__ w, int64_t ldw, int64_t M, int N, int K, int col_tiles, int n_split,
    int vec_dy, int vec_w, int vec_o, T* __restrict__ dx, int64_t lddx, float* __restrict__ part) {
  constexpr int kP = Pieces<T>::n;
  griddep_launch_dependents();
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

  __shared__ __align__(16) float s_ws[kBN];  // the step's weight scales
  Raw8<T> ra[2];
  float next_ws = 0.0f;
  Raw8<int8_t> rb[4];
  auto fetch = [&](int n0) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int gi = tid + i * kThreads;
      const int r = gi >> 3, c = (gi & 7) * 8;
      const int valid = row0 + r < M ? min(8, n_hi - n0 - c) : 0;
      load8(ra[i], dy + (row0 + r) * lddy + n0 + c, valid, vec_dy != 0);
    }
    if (tid < kBN) {
      next_ws = kScaleWeight<T> && ws_one ? 1.0f : n0 + tid < n_hi ? __ldg(ws + (ws_one ? 0 : n0 + tid)) : 0.0f;
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
    if (tid < kBN) s_ws[tid] = next_ws;  // the step before read its own before its second barrier
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int gi = tid + i * kThreads;
      __nv_bfloat16* to = sa + (gi >> 3) * kLdA + (gi & 7) * 8;
      if constexpr (kScaleWeight<T>) {
        store8(to, kPlane, ra[i]);
      } else {
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = to_f(ra[i].e[j]) * s_ws[(gi & 7) * 8 + j];  // zeros past n_hi
        store_pieces<kP>(to, kPlane, v);
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int gi = tid + i * kThreads;
      __nv_bfloat16* to = sb + (gi >> 4) * kLdB + (gi & 15) * 8;
      if constexpr (kScaleWeight<T>) {
        const float scale = s_ws[gi >> 4];
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = to_f(rb[i].e[j]) * scale;
        store_pieces<1>(to, 0, v);
      } else {
        store8(to, 0, rb[i]);
      }
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
  const float post = kScaleWeight<T> && ws_one ? __ldg(ws) : 1.0f;
#pragma unroll
  for (int n = 0; n < 8; ++n)
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int64_t row = row0 + wm * 16 + (lane >> 2) + half * 8;
      const int c = col0 + wn * 64 + n * 8 + (lane & 3) * 2;
      if (row >= M) continue;
      const float v0 = acc[n][2 * half] * post, v1 = acc[n][2 * half + 1] * post;
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

// dx from the fp32 partial sums of its cuts, in a fixed order; four elements a
// thread where the rows allow it.
template <typename T>
__global__ void __launch_bounds__(kThreads) sum_parts_kernel(const float* __restrict__ part,
                                                             int parts, int64_t M, int K, int vec,
                                                             T* __restrict__ dx, int64_t lddx) {
  griddep_wait();
  const int64_t total = M * K;
  const int64_t start = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kThreads;
  if (vec) {
    for (int64_t i = start * 4; i < total; i += step * 4) {
      float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      for (int p = 0; p < parts; ++p) {
        const float4 o = __ldcg(reinterpret_cast<const float4*>(part + p * total + i));
        v.x += o.x;
        v.y += o.y;
        v.z += o.z;
        v.w += o.w;
      }
      const int64_t row = i / K;
      T* dst = dx + row * lddx + (i - row * K);
      const T o[4] = {from_f<T>(v.x), from_f<T>(v.y), from_f<T>(v.z), from_f<T>(v.w)};
      if constexpr (sizeof(T) == 2) {
        *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(o);
      } else {
        *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(o);
      }
    }
    return;
  }
  for (int64_t i = start; i < total; i += step) {
    float v = 0.0f;
    for (int p = 0; p < parts; ++p) v += __ldcg(part + p * total + i);
    const int64_t row = i / K;
    dx[row * lddx + (i - row * K)] = from_f<T>(v);
  }
}

template <typename T>
int sum_parts(const float* part, int parts, const InputGradArgs& g, cudaStream_t stream) {
  const int K = static_cast<int>(g.K);
  const int vec = K % 4 == 0 && reinterpret_cast<uintptr_t>(g.dx) % (4 * sizeof(T)) == 0 && g.lddx % 4 == 0;
  const int64_t items = g.M * K / (vec ? 4 : 1);
  const int64_t blocks = std::min<int64_t>((items + kThreads - 1) / kThreads, 16ll * device_sm_count());
  const cudaError_t e = launch_chained(true, sum_parts_kernel<T>, dim3(static_cast<unsigned>(blocks)), kThreads, 0,
                                       stream, part, parts, g.M, K, vec, static_cast<T*>(g.dx), g.lddx);
  if (e != cudaSuccess) {
    set_error("input gradient sum launch failed: %s", cudaGetErrorString(e));
    return W8A8_ERR_ACCELERATOR;
  }
  return 0;
}

// At most two blocks a multiprocessor (all resident), at least four steps each, at
// most 16 pieces.
struct NSplit {
  int count, per;
};
NSplit n_split_of(int64_t M, int64_t N, int64_t K) {
  const int64_t tiles = ((M + kBM - 1) / kBM) * ((K + kBC - 1) / kBC);
  const int64_t steps = std::max<int64_t>(1, (N + kBN - 1) / kBN);
  int64_t want = 2ll * device_sm_count() / std::max<int64_t>(1, tiles);
  want = std::max<int64_t>(1, std::min<int64_t>({want, 16, steps / 4}));
  const int64_t per = (steps + want - 1) / want;
  return {static_cast<int>((steps + per - 1) / per), static_cast<int>(per * kBN)};
}

// ================================================================ tcgen05
// D[256 x 256] of a CTA pair: rows of dy (or of its pieces) times 256 columns
// of w, 64 of the contraction a stage, six stages.  The weights come as bf16,
// transposed to [K][n] once per call by widen_weights_kernel (30 us for 12288 x
// 4096, against 395 us of products at 5856 rows, 1.49 PFLOP/s with the tensor pipe
// active 91 % of the time; under the power cap of a long run 450).  Per CTA:
//   warp 4     TMA: its 128 rows of dy and its 128 columns of w (both K-major,
//              128-byte swizzle)
//   warp 5     MMA issue (the pair's leader), two TMEM accumulators of 256 columns
//   warps 0-3  epilogue: TMEM -> registers -> dx (or a split's fp32 partial sums)
// Twelve warps that converted the int8 weights inside this kernel, registers to
// swizzled shared memory, held it to 643 us where the MMAs alone take 381: every
// row tile converts the weights again, 500 instructions a warp and stage.
constexpr int kTmaWarp = 4, kMmaWarp = 5;
constexpr int kTcThreads = 192;
constexpr int kTcRows = 128, kTcCols = 256, kTcK = 64, kTcStages = 6;
constexpr int kTcTile = kTcRows * kTcK * 2;  // bytes of A, and of B, of a stage and CTA
constexpr int kTcSmem = 1024 + kTcStages * 2 * kTcTile + 256;

__device__ __forceinline__ void mma_bf16_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                              uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}

struct TcArgs {
  int64_t M;
  int K;
  int n_blocks;   // blocks of 64 of N; the contraction runs over pieces * n_blocks
  int kb_total;
  int col_tiles, row_tiles, splits;
  void* dx;
  int64_t lddx;
  int vec_o;
  float* part;    // splits > 1
  const float* one_scale;  // the single scale of a bf16 call's weight, for the sums; or NULL
};

// Unit u: split, then tiles in groups of eight row tiles (the CTAs that run
// together share rows of dy and columns of w in L2).
__device__ __forceinline__ void tc_unit(const TcArgs& g, int unit, int& mb, int& cb, int& kb_lo,
                                        int& kb_hi, int& split) {
  const int tiles = g.col_tiles * g.row_tiles;
  split = unit / tiles;
  const int tile = unit - split * tiles;
  constexpr int kGroup = 8;
  const int per = kGroup * g.col_tiles;
  const int grp = tile / per;
  const int rows = min(kGroup, g.row_tiles - grp * kGroup);
  const int r = tile - grp * per;
  mb = grp * kGroup + r % rows;
  cb = r / rows;
  kb_lo = static_cast<int>(static_cast<int64_t>(split) * g.kb_total / g.splits);
  kb_hi = static_cast<int>(static_cast<int64_t>(split + 1) * g.kb_total / g.splits);
}

template <typename T>
__global__ void __launch_bounds__(kTcThreads, 1)
    input_grad_tc_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b,
                         const TcArgs g) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint8_t* s_a = smem;
  uint8_t* s_b = smem + kTcStages * kTcTile;
  uint64_t* full = reinterpret_cast<uint64_t*>(s_b + kTcStages * kTcTile);
  uint64_t* empty = full + kTcStages;
  uint64_t* tfull = empty + kTcStages;
  uint64_t* tempty = tfull + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty + 2);
  int* abort_flag = reinterpret_cast<int*>(tmem_slot + 1);
  volatile int* abortv = abort_flag;
  int* err = &g_input_grad_error;

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  const int units = g.col_tiles * g.row_tiles * g.splits;
  const int first = static_cast<int>(blockIdx.x) / 2, step = static_cast<int>(gridDim.x) / 2;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kTcStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&tfull[b], 1);
      mbar_init(&tempty[b], 8);  // four epilogue warps of each CTA
    }
    *abort_flag = 0;
    fence_mbarrier_init();
  }
  if (warp == kTmaWarp && lane == 0) {
    tma_prefetch_desc(&tm_a);
    tma_prefetch_desc(&tm_b);
  }
  if (warp == kMmaWarp) {
    tmem_alloc<512, 2>(tmem_slot);
    tmem_relinquish<2>();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  griddep_launch_dependents();
  griddep_wait();  // the widened weights

  if (warp == kTmaWarp) {
    if (lane == 0) {
      uint32_t it = 0;
      bool ok = true;
      for (int unit = first; ok && unit < units; unit += step) {
        int mb, cb, lo, hi, split;
        tc_unit(g, unit, mb, cb, lo, hi, split);
        const int row = (mb * 2 + static_cast<int>(rank)) * kTcRows;
        const int col = (cb * 2 + static_cast<int>(rank)) * kTcRows;
        for (int kb = lo; kb < hi; ++kb, ++it) {
          const int s = static_cast<int>(it % kTcStages);
          if (!mbar_wait(&empty[s], ((it / kTcStages) & 1u) ^ 1u, abortv, err, kDevTimeoutEmpty)) {
            ok = false;
            break;
          }
          // both CTAs' bytes are counted on the leader's barrier
          if (leader) mbar_arrive_expect_tx(&full[s], 4 * kTcTile);
          const uint32_t bar = mapa_shared(smem_u32(&full[s]), 0);
          tma_load_2d_pair(s_a + s * kTcTile, &tm_a, bar, kb * kTcK, row);
          tma_load_2d_pair(s_b + s * kTcTile, &tm_b, bar, (kb % g.n_blocks) * kTcK, col);
        }
      }
      if (!ok) {  // let loads already in flight land (bounded)
        const uint64_t t0 = globaltimer_ns();
        while (globaltimer_ns() - t0 < 1000000) {
        }
      }
    }
  } else if (warp == kMmaWarp) {
    if (lane == 0 && leader) {
      constexpr uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10)  // f32 = bf16 x bf16
                                 | (static_cast<uint32_t>(kTcCols >> 3) << 17) |
                                 (static_cast<uint32_t>(2 * kTcRows >> 4) << 24);
      uint32_t it = 0, tl = 0;
      bool ok = true;
      for (int unit = first; ok && unit < units; unit += step, ++tl) {
        int mb, cb, lo, hi, split;
        tc_unit(g, unit, mb, cb, lo, hi, split);
        const uint32_t acc = tl & 1u;
        if (!mbar_wait(&tempty[acc], ((tl >> 1) & 1u) ^ 1u, abortv, err, kDevTimeoutTmemEmpty)) break;
        tc_fence_after();
        for (int kb = lo; kb < hi; ++kb, ++it) {
          const int s = static_cast<int>(it % kTcStages);
          if (!mbar_wait(&full[s], (it / kTcStages) & 1u, abortv, err, kDevTimeoutFull)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t a0 = smem_u32(s_a + s * kTcTile), b0 = smem_u32(s_b + s * kTcTile);
#pragma unroll
          for (int k = 0; k < kTcK / 16; ++k) {
            mma_bf16_pair(tmem + acc * kTcCols, smem_desc_k_sw128(a0 + k * 32),
                          smem_desc_k_sw128(b0 + k * 32), idesc, (kb != lo || k != 0) ? 1u : 0u);
          }
          umma_commit_pair(mapa_shared(smem_u32(&empty[s]), 0));
          umma_commit_pair(mapa_shared(smem_u32(&empty[s]), 1));
        }
        if (ok) {
          umma_commit_pair(mapa_shared(smem_u32(&tfull[acc]), 0));
          umma_commit_pair(mapa_shared(smem_u32(&tfull[acc]), 1));
        }
      }
    }
  } else {
    // ------------------------------------------------------------ epilogue
    const float post = g.one_scale ? __ldg(g.one_scale) : 1.0f;
    uint32_t tl = 0;
    for (int unit = first; unit < units; unit += step, ++tl) {
      int mb, cb, lo, hi, split;
      tc_unit(g, unit, mb, cb, lo, hi, split);
      const uint32_t acc = tl & 1u;
      const bool done = mbar_wait(&tfull[acc], (tl >> 1) & 1u, abortv, err, kDevTimeoutTmemFull);
      if (!__all_sync(0xffffffffu, done)) break;
      tc_fence_after();
      const int64_t row = static_cast<int64_t>(mb * 2 + static_cast<int>(rank)) * kTcRows + warp * 32 + lane;
      for (int c = 0; c < kTcCols / 32; ++c) {
        const int col = cb * kTcCols + c * 32;
        if (col >= g.K) break;
        uint32_t v[32];
        __syncwarp();
        tmem_ld_32x32b_x32(tmem + (static_cast<uint32_t>(warp * 32) << 16) + acc * kTcCols + c * 32, v);
        tmem_ld_wait();
        if (g.one_scale) {
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = __float_as_uint(__uint_as_float(v[j]) * post);
        }
        if (row >= g.M) {
        } else if (g.part) {
          float* p = g.part + (static_cast<int64_t>(split) * g.M + row) * g.K + col;
#pragma unroll
          for (int j = 0; j < 32; j += 4) {
            if (g.K % 4 == 0 && col + j < g.K) {
              *reinterpret_cast<uint4*>(p + j) = make_uint4(v[j], v[j + 1], v[j + 2], v[j + 3]);
            } else {
#pragma unroll
              for (int q = 0; q < 4; ++q)
                if (col + j + q < g.K) p[j + q] = __uint_as_float(v[j + q]);
            }
          }
        } else {
          T* p = static_cast<T*>(g.dx) + row * g.lddx + col;
#pragma unroll
          for (int j = 0; j < 32; j += 8) {
            T o[8];
#pragma unroll
            for (int q = 0; q < 8; ++q) o[q] = from_f<T>(__uint_as_float(v[j + q]));
            if (g.vec_o && col + j + 8 <= g.K) {
              const uint32_t* u = reinterpret_cast<const uint32_t*>(o);
              *reinterpret_cast<uint4*>(p + j) = make_uint4(u[0], u[1], u[2], u[3]);
            } else {
#pragma unroll
              for (int q = 0; q < 8; ++q)
                if (col + j + q < g.K) p[j + q] = o[q];
            }
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(mapa_shared(smem_u32(&tempty[acc]), 0));
    }
  }
  __syncthreads();
  cluster_sync();  // the peer is done with its TMEM and these barriers
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc<512, 2>(tmem);
  }
}

// bf16(w ws) (ws NULL: w itself, which bf16 holds) transposed to out[K][n_pad],
// zero past N.  A block takes 128 rows by 64 columns; a thread 8 rows by 4
// columns: eight words, from which byte permutations make the floats (a byte in
// the mantissa of 2^23), four 16-byte pieces of output rows, exchanged through
// shared memory so that the stores run along n.
__global__ void __launch_bounds__(kThreads) widen_weights_kernel(
    const int8_t* __restrict__ w, int64_t ldw, const float* __restrict__ ws, int N, int K, int n_pad,
    int k_tiles, int vec, __nv_bfloat16* __restrict__ out) {
  griddep_launch_dependents();
  __shared__ __align__(16) uint4 tile[64][16];
  const int n0 = static_cast<int>(blockIdx.x / k_tiles) * 128, k0 = static_cast<int>(blockIdx.x % k_tiles) * 64;
  const int kc = threadIdx.x & 15, ng = threadIdx.x >> 4;
  const int col = k0 + 4 * kc;
  uint32_t x[8];
  uint64_t sc[4];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int n = n0 + ng * 8 + j;
    uint32_t v = 0;
    if (n < N) {
      const int8_t* p = w + n * ldw + col;
      if (vec && col + 4 <= K) {
        v = __ldg(reinterpret_cast<const uint32_t*>(p));
      } else {
#pragma unroll
        for (int b = 0; b < 4; ++b)
          if (col + b < K) v |= static_cast<uint32_t>(static_cast<uint8_t>(p[b])) << (8 * b);
      }
    }
    x[j] = v ^ 0x80808080u;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int n = n0 + ng * 8 + 2 * j;
    sc[j] = pk(ws && n < N ? __ldg(ws + n) : 1.0f, ws && n + 1 < N ? __ldg(ws + n + 1) : 1.0f);
  }
#pragma unroll
  for (int b = 0; b < 4; ++b) {
    uint32_t o[4];
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      const uint64_t f = pk(__uint_as_float(__byte_perm(x[2 * p], 0x4B000000u, 0x7540 + b)),
                            __uint_as_float(__byte_perm(x[2 * p + 1], 0x4B000000u, 0x7540 + b)));
      const uint64_t v = mul2(add2(f, pk(-8388736.0f, -8388736.0f)), sc[p]);  // -(2^23 + 128)
      o[p] = pack_bf16(lo(v), hi(v));
    }
    const int k = 4 * kc + b;
    tile[k][ng ^ kc] = make_uint4(o[0], o[1], o[2], o[3]);  // 16 threads, 16 different pieces of a row
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int at = static_cast<int>(threadIdx.x) + i * kThreads;
    const int k = at >> 4, c = at & 15;
    const int n = n0 + c * 8;
    if (k0 + k < K && n < n_pad)
      *reinterpret_cast<uint4*>(out + static_cast<int64_t>(k0 + k) * n_pad + n) = tile[k][c ^ (k >> 2)];
  }
  griddep_wait();  // what follows this kernel may then use what the one before it wrote
}

// bf16 pieces of dy ws as planes [row][piece][n_pad], zero past N: the operand
// of input_grad_tc_kernel for f16.
template <typename T>
__global__ void __launch_bounds__(kThreads) pieces_kernel(const T* __restrict__ dy, int64_t lddy,
                                                          const float* __restrict__ ws, int ws_one,
                                                          int64_t M, int N, int n_pad, int vec,
                                                          __nv_bfloat16* __restrict__ out) {
  griddep_launch_dependents();
  constexpr int kP = Pieces<T>::n;
  const int64_t total = M * (n_pad / 8);
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; i < total;
       i += static_cast<int64_t>(gridDim.x) * kThreads) {
    const int64_t row = i / (n_pad / 8);
    const int c = static_cast<int>(i - row * (n_pad / 8)) * 8;
    const int valid = min(8, N - c);
    Raw8<T> r;
    load8(r, dy + row * lddy + c, valid, vec != 0);
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      v[j] = to_f(r.e[j]);
      if (j < valid) v[j] *= __ldg(ws + (ws_one ? 0 : c + j));
    }
    store_pieces<kP>(out + row * kP * n_pad + c, n_pad, v);
  }
}

PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess) {
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
    }
  });
  return fn;
}

// bf16 rows [rows][ld], `inner` of them used, in boxes of 128 rows x 64.
bool map_rows(CUtensorMap* map, const void* base, int64_t inner, int64_t rows, int64_t ld) {
  auto fn = tensor_map_encoder();
  cuuint64_t dims[2] = {static_cast<cuuint64_t>(inner), static_cast<cuuint64_t>(rows)};
  cuuint64_t strides[1] = {static_cast<cuuint64_t>(ld) * 2};
  cuuint32_t box[2] = {kTcK, kTcRows}, ones[2] = {1, 1};
  return fn && fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(base), dims, strides, box, ones,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Whether input_grad_tc_kernel takes a call: 16-bit types (fp32 needs its sums
// apart), more rows than one mma.sync tile and, for bf16, rows of dy that TMA
// can read.
bool tc_shape(int64_t M, int64_t N, int64_t K, int dtype) {
  return dtype != W8A8_F32 && M > kBM && N > 0 && K > 0;
}
bool rows_of_16_bytes(const InputGradArgs& g) {
  return reinterpret_cast<uintptr_t>(g.dy) % 16 == 0 && (g.lddy * 2) % 16 == 0;
}
bool tc_operands(const InputGradArgs& g) {
  return g.dtype != W8A8_BF16 || rows_of_16_bytes(g);
}
int64_t round_up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

struct TcPlan {
  int n_blocks, kb_total, row_tiles, col_tiles, splits;
  int64_t pieces_bytes, weight_bytes, part_bytes;
};
// The contraction is cut until every pair of multiprocessors has a unit, with
// at least sixteen stages a unit (the pipeline's fill and the sum of the parts).
TcPlan tc_plan(int64_t M, int64_t N, int64_t K, int dtype) {
  TcPlan p;
  const int pieces = dtype == W8A8_F16 ? 2 : 1;
  p.n_blocks = static_cast<int>((N + kTcK - 1) / kTcK);
  p.kb_total = pieces * p.n_blocks;
  p.row_tiles = static_cast<int>((M + 2 * kTcRows - 1) / (2 * kTcRows));
  p.col_tiles = static_cast<int>((K + kTcCols - 1) / kTcCols);
  const int64_t tiles = static_cast<int64_t>(p.row_tiles) * p.col_tiles;
  const int64_t pairs = device_sm_count() / 2;
  p.splits = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(pairs / tiles, p.kb_total / 16)));
  p.pieces_bytes = pieces > 1 ? round_up(M * pieces * p.n_blocks * kTcK * 2, 256) : 0;
  p.weight_bytes = round_up(K * p.n_blocks * kTcK * 2, 256);
  p.part_bytes = p.splits > 1 ? p.splits * M * K * 4 : 0;
  return p;
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
int tc_typed(const InputGradArgs& g, cudaStream_t stream) {
  const TcPlan p = tc_plan(g.M, g.N, g.K, g.dtype);
  const int N = static_cast<int>(g.N), K = static_cast<int>(g.K);
  const int n_pad = p.n_blocks * kTcK;
  constexpr int kP = Pieces<T>::n;
  constexpr bool direct = kP == 1;  // bf16: TMA takes dy as it lies
  uint8_t* work = static_cast<uint8_t*>(g.workspace);
  // the scales go into the pieces of dy where there are pieces, else into w, a single one onto the sums
  const bool one = direct && g.ws_numel == 1;
  if constexpr (!direct) {
    const int vec = rows_of_16_bytes(g);
    const int64_t total = g.M * (n_pad / 8);
    const int64_t blocks = std::min<int64_t>((total + kThreads - 1) / kThreads, 16ll * device_sm_count());
    pieces_kernel<T><<<static_cast<unsigned>(blocks), kThreads, 0, stream>>>(
        static_cast<const T*>(g.dy), g.lddy, g.ws, g.ws_numel == 1, g.M, N, n_pad, vec,
        reinterpret_cast<__nv_bfloat16*>(work));
    if (int rc = launched("input gradient pieces")) return rc;
  }
  uint8_t* wide = work + p.pieces_bytes;
  const int k_tiles = (K + 63) / 64;
  const cudaError_t we = launch_chained(
      !direct, widen_weights_kernel, dim3(static_cast<unsigned>(static_cast<int64_t>((N + 127) / 128) * k_tiles)),
      kThreads, 0, stream, g.w, g.ldw, direct && !one ? g.ws : nullptr, N, K, n_pad, k_tiles,
      static_cast<int>(reinterpret_cast<uintptr_t>(g.w) % 4 == 0 && g.ldw % 4 == 0),
      reinterpret_cast<__nv_bfloat16*>(wide));
  if (we != cudaSuccess) {
    set_error("input gradient weights launch failed: %s", cudaGetErrorString(we));
    return W8A8_ERR_ACCELERATOR;
  }
  CUtensorMap map_a, map_b;
  const int64_t inner = direct ? g.N : static_cast<int64_t>(kP) * n_pad;
  if (!map_rows(&map_a, direct ? g.dy : work, inner, g.M, direct ? g.lddy : inner) ||
      !map_rows(&map_b, wide, n_pad, g.K, n_pad)) {
    set_error("cuTensorMapEncodeTiled rejected the operands (M=%lld N=%lld K=%lld)",
              static_cast<long long>(g.M), static_cast<long long>(g.N), static_cast<long long>(g.K));
    return W8A8_ERR_RUNTIME;
  }
  TcArgs a{};
  a.M = g.M;
  a.K = K;
  a.n_blocks = p.n_blocks;
  a.kb_total = p.kb_total;
  a.row_tiles = p.row_tiles;
  a.col_tiles = p.col_tiles;
  a.splits = p.splits;
  a.dx = g.dx;
  a.lddx = g.lddx;
  a.vec_o = reinterpret_cast<uintptr_t>(g.dx) % 16 == 0 && (g.lddx * 2) % 16 == 0;
  a.part = p.splits > 1 ? reinterpret_cast<float*>(wide + p.weight_bytes) : nullptr;
  a.one_scale = one ? g.ws : nullptr;
  auto kern = input_grad_tc_kernel<T>;
  static bool set[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 64 || !set[dev]) {
    const cudaError_t e =
        cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kTcSmem);
    if (e != cudaSuccess) {
      set_error("cudaFuncSetAttribute failed: %s", cudaGetErrorString(e));
      return W8A8_ERR_ACCELERATOR;
    }
    if (dev < 64) set[dev] = true;
  }
  const int64_t units = static_cast<int64_t>(p.row_tiles) * p.col_tiles * p.splits;
  cudaLaunchConfig_t lc{};
  lc.gridDim = dim3(static_cast<unsigned>(2 * std::min<int64_t>(units, device_sm_count() / 2)));
  lc.blockDim = dim3(kTcThreads);
  lc.dynamicSmemBytes = kTcSmem;
  lc.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  lc.attrs = attr;
  lc.numAttrs = 2;
  const cudaError_t e = cudaLaunchKernelEx(&lc, kern, map_a, map_b, a);
  if (e != cudaSuccess) {
    set_error("input gradient launch failed: %s", cudaGetErrorString(e));
    return W8A8_ERR_ACCELERATOR;
  }
  if (a.part) {
    return sum_parts<T>(a.part, p.splits, g, stream);
  }
  return 0;
}

// ================================================================ few rows
// Up to 16 rows: what has to be read is w, once.  A block takes 64 columns and a
// range of the contraction, 128 of it a step, a warp sixteen: w goes from HBM
// straight into the warp's matrix fragments, two steps ahead (a lane reads eight
// columns of four rows; which of the tile's columns a fragment column stands for is
// free to choose), and only dy or the pieces of dy ws pass through shared memory.  The
// eight warps' sums are joined in order at the end.
// A captured call of 16 rows, sum included, memory cold: 4096 -> 4096 in 22.5 us (f16 26.6, fp32
// 30.7) where input_grad_kernel, which stages w in shared memory, takes 24.5 (32.8, 47.1); 12288 ->
// 4096 in 45 (57, 68) against 49 (70, 112).  At 32 rows this form took 27, that one 21.
constexpr int kFewRows = 16, kFewCols = 64, kFewN = 128, kLdFew = kFewN + 8;

template <typename T>
__global__ void __launch_bounds__(kThreads) input_grad_few_kernel(
    const T* __restrict__ dy, int64_t lddy, const float* __restrict__ ws, int ws_one,
    const int8_t* __restrict__ w, int64_t ldw, int M, int N, int K, int n_split, int vec_dy,
    T* __restrict__ dx, int64_t lddx, float* __restrict__ part) {
  constexpr int kP = Pieces<T>::n, kRows = kFewRows;
  griddep_launch_dependents();
  constexpr int kPlane = kRows * kLdFew;
  constexpr bool kApart = std::is_same<T, float>::value;
  constexpr int kBuf = 2 * kP * kPlane * 2, kJoin = kRows * (kFewCols + 1) * 4;
  __shared__ __align__(16) uint8_t smem[kBuf > kJoin ? kBuf : kJoin];
  __nv_bfloat16* sa = reinterpret_cast<__nv_bfloat16*>(smem);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int q = lane & 3, gcol = lane >> 2;
  const int col = blockIdx.x * kFewCols + 8 * gcol;
  const bool in_k = col < K;  // K % 8 == 0
  const int n_lo = blockIdx.y * n_split, n_hi = min(N, n_lo + n_split);

  float acc[8][4] = {};
  float low[kApart ? 8 : 1][4] = {};
  // a step's four rows of w: their codes, and their scales where those go into the weight
  struct Codes {
    uint2 q[4];
    float scale[kScaleWeight<T> ? 4 : 1];
  };
  Codes wq[2];
  auto fetch_w = [&](int n0, Codes& r) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int n = n0 + warp * 16 + 2 * q + (i & 1) + (i >> 1) * 8;
      r.q[i] = in_k && n < n_hi ? __ldg(reinterpret_cast<const uint2*>(w + n * ldw + col)) : make_uint2(0, 0);
      if constexpr (kScaleWeight<T>) r.scale[i] = ws_one || n >= n_hi ? 1.0f : __ldg(ws + n);
    }
  };
  // dy (times ws) of one step: kRows x 128 elements, eight at a time
  static_assert(kRows * (kFewN / 8) == kThreads, "eight elements a thread");
  auto lay = [&](int n0, int buf) {
    {
      const int r = tid / (kFewN / 8), c = (tid % (kFewN / 8)) * 8;
      const int valid = r < M ? min(8, n_hi - n0 - c) : 0;
      Raw8<T> raw;
      load8(raw, dy + static_cast<int64_t>(r) * lddy + n0 + c, valid, vec_dy != 0);
      if constexpr (kScaleWeight<T>) {
        store8(sa + buf * kP * kPlane + r * kLdFew + c, kPlane, raw);
      } else {
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j)
          v[j] = j < valid ? to_f(raw.e[j]) * __ldg(ws + (ws_one ? 0 : n0 + c + j)) : 0.0f;
        store_pieces<kP>(sa + buf * kP * kPlane + r * kLdFew + c, kPlane, v);
      }
    }
  };
  fetch_w(n_lo, wq[0]);
  fetch_w(n_lo + kFewN, wq[1]);
  lay(n_lo, 0);
  __syncthreads();
  auto step = [&](int n0, int buf, Codes& r) {
    uint32_t x[4][2];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[i][0] = r.q[i].x ^ 0x80808080u;
      x[i][1] = r.q[i].y ^ 0x80808080u;
    }
    uint64_t scale[2];
    if constexpr (kScaleWeight<T>) {
      scale[0] = pk(r.scale[0], r.scale[1]);
      scale[1] = pk(r.scale[2], r.scale[3]);
    }
    fetch_w(n0 + 2 * kFewN, r);
    if (n0 + kFewN < n_hi) lay(n0 + kFewN, buf ^ 1);
    uint32_t a[kP][4];
#pragma unroll
    for (int p = 0; p < kP; ++p) ldsm4(a[p], at16(sa + (buf * kP + p) * kPlane, 0, warp * 16, kLdFew, lane));
    const uint64_t magic = pk(-8388736.0f, -8388736.0f);  // -(2^23 + 128)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      uint32_t b[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint64_t f =
            add2(pk(__uint_as_float(__byte_perm(x[2 * h][j >> 2], 0x4B000000u, 0x7540 + (j & 3))),
                    __uint_as_float(__byte_perm(x[2 * h + 1][j >> 2], 0x4B000000u, 0x7540 + (j & 3)))),
                 magic);
        if constexpr (kScaleWeight<T>) f = mul2(f, scale[h]);
        b[h] = pack_bf16(lo(f), hi(f));
      }
#pragma unroll
      for (int p = 0; p < kP; ++p) {
        if constexpr (kApart) {
          mma_apart(acc[j], low[j], a[p], b[0], b[1], p == 0);
        } else {
          mma(acc[j], a[p], b[0], b[1]);
        }
      }
    }
    __syncthreads();
  };
  int buf = 0;
  for (int n0 = n_lo; n0 < n_hi; n0 += 2 * kFewN) {
    step(n0, buf, wq[0]);
    buf ^= 1;
    if (n0 + kFewN < n_hi) {
      step(n0 + kFewN, buf, wq[1]);
      buf ^= 1;
    }
  }
  if constexpr (kApart) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[j][e] += low[j][e];
  }
  // the warps' sums, in order
  float* sum = reinterpret_cast<float*>(smem);
  for (int v = 0; v < kThreads / 32; ++v) {
    if (warp == v) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          // fragment column 2 q + (e & 1) of tile j stands for column 8 (2 q + (e & 1)) + j
          const int r = gcol + (e >> 1) * 8, c = 8 * (2 * q + (e & 1)) + j;
          float* cell = sum + r * (kFewCols + 1) + c;
          *cell = v ? *cell + acc[j][e] : acc[j][e];
        }
    }
    __syncthreads();
  }
  const float post = kScaleWeight<T> && ws_one ? __ldg(ws) : 1.0f;
  for (int i = tid; i < kRows * kFewCols; i += kThreads) {
    const int r = i / kFewCols, c = blockIdx.x * kFewCols + i % kFewCols;
    if (r >= M || c >= K) continue;
    const float v = sum[r * (kFewCols + 1) + i % kFewCols] * post;
    if (part) {
      part[(static_cast<int64_t>(blockIdx.y) * M + r) * K + c] = v;
    } else {
      dx[static_cast<int64_t>(r) * lddx + c] = from_f<T>(v);
    }
  }
}

// Whether input_grad_few_kernel takes a call, by shape (its operands' alignment apart).
bool few_shape(int64_t M, int64_t N, int64_t K) { return M <= kFewRows && N > 0 && K > 0 && K % 8 == 0; }
// Two blocks a multiprocessor, at least two steps each, at most 16 pieces.
struct FewSplit {
  int count, per;
};
FewSplit few_split(int64_t N, int64_t K) {
  const int64_t cols = (K + kFewCols - 1) / kFewCols, steps = (N + kFewN - 1) / kFewN;
  const int64_t want =
      std::max<int64_t>(1, std::min<int64_t>({2ll * device_sm_count() / cols, 16, steps / 2}));
  const int64_t per = (steps + want - 1) / want;
  return {static_cast<int>((steps + per - 1) / per), static_cast<int>(per * kFewN)};
}

template <typename T>
int few_typed(const InputGradArgs& g, cudaStream_t stream) {
  const FewSplit sp = few_split(g.N, g.K);
  const int M = static_cast<int>(g.M), N = static_cast<int>(g.N), K = static_cast<int>(g.K);
  const int vec = reinterpret_cast<uintptr_t>(g.dy) % 16 == 0 && (g.lddy * static_cast<int64_t>(sizeof(T))) % 16 == 0;
  float* part = sp.count > 1 ? static_cast<float*>(g.workspace) : nullptr;
  const T* dy = static_cast<const T*>(g.dy);
  T* dx = static_cast<T*>(g.dx);
  input_grad_few_kernel<T><<<dim3((K + kFewCols - 1) / kFewCols, sp.count), kThreads, 0, stream>>>(
      dy, g.lddy, g.ws, g.ws_numel == 1, g.w, g.ldw, M, N, K, sp.per, vec, dx, g.lddx, part);
  if (int rc = launched("input gradient")) return rc;
  if (part) {
    return sum_parts<T>(part, sp.count, g, stream);
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
  static_assert(bytes + kBN * 4 <= 48 * 1024, "no opt-in shared memory needed");
  const dim3 grid(static_cast<unsigned>(tiles * cols), sp.count);
  input_grad_kernel<T><<<grid, kThreads, bytes, stream>>>(
      static_cast<const T*>(g.dy), g.lddy, g.ws, g.ws_numel == 1, g.w, g.ldw, g.M, N, K, cols, sp.per,
      vdy, vw, vo, static_cast<T*>(g.dx), g.lddx, part);
  if (int rc = launched("input gradient")) return rc;
  if (part) {
    return sum_parts<T>(part, sp.count, g, stream);
  }
  return 0;
}

}  // namespace

int64_t input_grad_workspace_bytes(int64_t M, int64_t N, int64_t K, int dtype) {
  const NSplit sp = n_split_of(M, N, K);
  int64_t bytes = sp.count > 1 ? sp.count * M * K * 4 : 0;
  if (few_shape(M, N, K)) {
    const int few = few_split(N, K).count;
    bytes = std::max(bytes, few > 1 ? few * M * K * 4 : 0);
  }
  if (tc_shape(M, N, K, dtype)) {
    const TcPlan p = tc_plan(M, N, K, dtype);
    bytes = std::max(bytes, p.pieces_bytes + p.weight_bytes + p.part_bytes);
  }
  return bytes;
}

int input_grad_launch(const InputGradArgs& g, cudaStream_t stream) {
  const bool tc = tc_shape(g.M, g.N, g.K, g.dtype) && tc_operands(g);
  if (few_shape(g.M, g.N, g.K) && reinterpret_cast<uintptr_t>(g.w) % 8 == 0 && g.ldw % 8 == 0) {
    switch (g.dtype) {
      case W8A8_BF16: return few_typed<__nv_bfloat16>(g, stream);
      case W8A8_F16: return few_typed<__half>(g, stream);
      default: return few_typed<float>(g, stream);
    }
  }
  switch (g.dtype) {
    case W8A8_BF16: return tc ? tc_typed<__nv_bfloat16>(g, stream) : typed<__nv_bfloat16>(g, stream);
    case W8A8_F16: return tc ? tc_typed<__half>(g, stream) : typed<__half>(g, stream);
    default: return typed<float>(g, stream);
  }
}

}  // namespace w8a8
