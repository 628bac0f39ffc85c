// The adapter contractions of long bf16 batches on tcgen05.
//
//   shrink_tc   part[split][row][r] = sum over the split's k of x[row, k] W_s[k, r]
//               a tile of 128 rows is the M side, the rank the N side
//   expand_tc   out[row][n] = y[row][n] + c[s] * sum over r of h[row, r] W_s[r, n]
//   tokens_tc   part[split][s][r][c] (or [c][r]) = sum over the split's rows m of
//               adapter s of q[m, r] x[m, c]: 128 columns are the M side, read
//               from the same row-major tiles by their transposed (MN-major)
//               descriptors; the rank-side values come as bf16 pieces, [r][m]
//
// Every operand arrives by TMA in 128-byte swizzled rows; a rank below 64 is
// padded by the copies' zero fill.  The tensor core's rate leaves both bound by
// reading x (mma.sync, at 510 TFLOP/s, would hold a rank of 64 with two pieces to a
// third of it).  int8 codes (an 8-bit checkpoint as x) land as bytes and are
// widened to bf16 by four warps on the way.
//
// What keeps rows of other adapters apart (NaN and infinity stay in their rows): shrink_tc and
// expand_tc multiply every row of a tile by every adapter of the tile, but output rows are
// independent and only the row's own adapter's result is stored; tokens_tc sums over rows, so
// there the rows of other adapters are zeroed in both operands first.
//
// Waits are bounded (sm100_ptx.cuh): a wait that gives up records its code, every
// role of the block falls through, and TMEM is released.
#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_bf16.h>

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

__device__ int g_lora_error;

int read_and_clear_lora_error(cudaStream_t stream, int* value) {
  int v = 0;
  cudaError_t e =
      cudaMemcpyFromSymbolAsync(&v, g_lora_error, sizeof(int), 0, cudaMemcpyDeviceToHost, stream);
  if (e == cudaSuccess) e = cudaStreamSynchronize(stream);
  if (e != cudaSuccess) return static_cast<int>(e);
  if (v != 0) {
    const int zero = 0;
    e = cudaMemcpyToSymbolAsync(g_lora_error, &zero, sizeof(int), 0, cudaMemcpyHostToDevice, stream);
    if (e == cudaSuccess) e = cudaStreamSynchronize(stream);
    if (e != cudaSuccess) return static_cast<int>(e);
  }
  *value = v;
  return 0;
}

namespace {

// warps 0-7: widen codes, mask (0-3 also the epilogue); 8: TMA; 9: MMA
constexpr int kThreads = 320;
constexpr int kTmaWarp = 8, kMmaWarp = 9;

__device__ __forceinline__ void tma_load_3d(void* dst, const void* map, uint64_t* bar, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(smem_u32(dst)),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void mma_bf16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Descriptor of an operand whose M (or N) elements run along the 128-byte rows:
// row = one k, 64 elements; eight rows a swizzle atom (1024 bytes, the stride
// offset); the next 64 elements `chunk` bytes further (the leading offset).
__device__ __forceinline__ uint64_t smem_desc_mn_sw128(uint32_t addr, uint32_t chunk) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((addr >> 4) & 0x3FFFu);
  d |= static_cast<uint64_t>((chunk >> 4) & 0x3FFFu) << 16;
  d |= static_cast<uint64_t>(1024u >> 4) << 32;
  d |= static_cast<uint64_t>(1u) << 46;
  d |= static_cast<uint64_t>(2u) << 61;
  return d;
}
// f32 = bf16 x bf16, M 128; a_mn / b_mn: that operand's M / N runs along the rows.
__host__ __device__ constexpr uint32_t idesc_bf16(int n, int a_mn, int b_mn) {
  return (1u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(a_mn) << 15) |
         (static_cast<uint32_t>(b_mn) << 16) | (static_cast<uint32_t>(n >> 3) << 17) | ((128u >> 4) << 24);
}
constexpr uint32_t tmem_cols(int n) { return n <= 32 ? 32u : n <= 64 ? 64u : n <= 128 ? 128u : 256u; }

// Sixteen codes to sixteen bf16 (two 16-byte vectors).
__device__ __forceinline__ void widen16(const uint4& q, uint4& lo8, uint4& hi8) {
  const uint32_t w[4] = {q.x ^ 0x80808080u, q.y ^ 0x80808080u, q.z ^ 0x80808080u, q.w ^ 0x80808080u};
  uint32_t o[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t a = __byte_perm(w[i >> 1], 0x4B000000u, (i & 1) ? 0x7542 : 0x7540);
    const uint32_t b = __byte_perm(w[i >> 1], 0x4B000000u, (i & 1) ? 0x7543 : 0x7541);
    const uint64_t f = add2(pk(__uint_as_float(a), __uint_as_float(b)), pk(-8388736.0f, -8388736.0f));
    o[i] = pack_bf16(lo(f), hi(f));
  }
  lo8 = make_uint4(o[0], o[1], o[2], o[3]);
  hi8 = make_uint4(o[4], o[5], o[6], o[7]);
}

// The distinct adapters of 128 rows in order of appearance, by one warp (a row is
// first if none before it has its adapter).
__device__ __forceinline__ void list_adapters(const int* id, int* list, int& count) {
  const int lane = threadIdx.x & 31;
  int n = 0;
  for (int base = 0; base < 128; base += 32) {
    const int mine = id[base + lane];
    bool first = mine >= 0;
    for (int j = 0; j < base; ++j) first = first && id[j] != mine;
    const unsigned same = __match_any_sync(0xffffffffu, mine);
    first = first && __ffs(same) - 1 == lane;
    const unsigned m = __ballot_sync(0xffffffffu, first);
    if (first) list[n + __popc(m & ((1u << lane) - 1u))] = mine;
    n += __popc(m);
  }
  if (lane == 0) count = n;
}

// After a wait that gave up: copies already in flight land first (bounded).
__device__ __forceinline__ void let_copies_land() {
  const uint64_t t0 = globaltimer_ns();
  while (globaltimer_ns() - t0 < 1000000) {
  }
}

// The splits' sums of the rank side, in order, all of a split's loads in flight at once:
// thread `at` of kThreadsN has the vectors at + i kThreadsN, kV of them a row, of the rows
// from row0 + r0 on.  What lies past R is zero; rows without an adapter give whatever is
// there (the caller leaves them out), rows past M the last row.
template <int kV, int kThreadsN, int kEach>
__device__ __forceinline__ void rank_sums(const float* __restrict__ part, int splits, const Rows& rows, int64_t row0,
                                          int r0, int at, int R, float4 (&sum)[kEach]) {
  const int64_t plane = rows.M * R;
  const int last = static_cast<int>(min(static_cast<int64_t>(127), rows.M - 1 - row0));
  const float* p = part + row0 * R;
  const int c = at % kV * 4;  // kThreadsN % kV == 0: the same for all
  int rel[kEach];
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    rel[i] = min(r0 + (at + i * kThreadsN) / kV, last) * R + (c < R ? c : 0);  // R % 8 == 0
    sum[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  }
  constexpr int kAhead = kEach > 8 ? 1 : kEach > 4 ? 2 : 4;
#pragma unroll kAhead
  for (int sp = 0; sp < splits; ++sp, p += plane) {
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const float4 q = __ldcg(reinterpret_cast<const float4*>(p + rel[i]));
      sum[i].x += q.x;
      sum[i].y += q.y;
      sum[i].z += q.z;
      sum[i].w += q.w;
    }
  }
  if (c >= R) {
#pragma unroll
    for (int i = 0; i < kEach; ++i) sum[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  }
}

struct Bars {
  uint64_t full[8], ready[8], empty[8], acc[8], w_full[4], w_empty[4], done, drained;
  uint32_t tmem;
  int abort_flag;
};
constexpr int kBarBytes = 384;
static_assert(sizeof(Bars) <= kBarBytes, "barriers");

// ======================================================================== shrink
// A tile whose rows have several adapters is multiplied by each of them while it is
// there, into accumulators of their own, as many at a time as TMEM has columns for.
// The contraction is cut so that two blocks a multiprocessor are all there are.  Bound
// by reading x: 11712 x 4096 at rank 64 in 30 us (98 MB, 3.3 TB/s), 5856 x 4096 at
// rank 16 in 12 to 15, 11712 x 12288 in 70 (288 MB, 4.1 TB/s).
constexpr int kSRows = 128, kSK = 64;
constexpr int kXTile = kSRows * kSK * 2;  // 16 KB
template <bool kCodes, int kRank>
struct ShrinkTc {
  static constexpr int kW = kRank == 128 ? 16384 : 8192;
  static constexpr int kRaw = kCodes ? kSRows * kSK : 0;
  static constexpr int kWStages = kRank == 128 ? 2 : kCodes ? 2 : 4;
  static constexpr int kXStages = kCodes ? 3 : 4;
  static constexpr int kBytes = 1024 + kXStages * (kXTile + kRaw) + kWStages * kW + kBarBytes + 1280;
  static constexpr uint32_t kCols = 256;                  // accumulator columns a block takes
  static constexpr int kAtOnce = static_cast<int>(kCols) / kRank;
  static_assert(2 * kBytes + 2048 <= 228 * 1024, "two blocks a multiprocessor");
};

// tm_x: rows of x, boxes 64 x 128 (bf16, swizzled; codes: as they are).  tm_w:
// the adapters, boxes 64 k x kRank of [S][R][K] (kWRows), or 64 r x 64 n of [S][N][R].
template <bool kCodes, int kRank, bool kWRows>
__global__ void __launch_bounds__(kThreads) shrink_tc_kernel(
    const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w, Rows rows,
    const float* __restrict__ row_mul, int K, int R, int kb_split, float* __restrict__ part,
    int* __restrict__ counts) {
  using C = ShrinkTc<kCodes, kRank>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint8_t* s_x = smem;
  uint8_t* s_w = s_x + C::kXStages * kXTile;
  uint8_t* s_raw = s_w + C::kWStages * C::kW;
  Bars* bars = reinterpret_cast<Bars*>(s_raw + C::kXStages * C::kRaw);
  uint64_t *w_full = bars->w_full, *w_empty = bars->w_empty;
  int* id = reinterpret_cast<int*>(reinterpret_cast<uint8_t*>(bars) + kBarBytes);
  int* list = id + kSRows;
  __shared__ int count;
  volatile int* abortv = &bars->abort_flag;
  int* err = &g_lora_error;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * kSRows;
  const int kb_all = (K + kSK - 1) / kSK;
  const int kb_lo = blockIdx.y * kb_split, kb_hi = min(kb_all, kb_lo + kb_split);

  if (tid == 0) {
    for (int s = 0; s < C::kXStages; ++s) {
      mbar_init(&bars->full[s], 1);
      mbar_init(&bars->ready[s], 8);
      mbar_init(&bars->empty[s], 1);
    }
    for (int s = 0; s < C::kWStages; ++s) {
      mbar_init(&w_full[s], 1);
      mbar_init(&w_empty[s], 1);
    }
    mbar_init(&bars->done, 1);
    mbar_init(&bars->drained, 4);
    bars->abort_flag = 0;
    fence_mbarrier_init();
    count = 0;
  }
  int v = -1;
  if (tid < kSRows) {
    v = adapter_of(rows, row0 + tid);
    id[tid] = v;
  }
  if (warp == kTmaWarp && lane == 0) {
    tma_prefetch_desc(&tm_x);
    tma_prefetch_desc(&tm_w);
  }
  if (warp == kMmaWarp) {
    tmem_alloc<C::kCols>(&bars->tmem);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  griddep_launch_dependents();  // not before this block has its TMEM: an early block of the next kernel takes some too
  const bool one = __syncthreads_and(tid >= kSRows || row0 + tid >= rows.M || v == id[0]);
  if (one) {
    if (tid == 0) {
      list[0] = id[0];
      count = id[0] >= 0 ? 1 : 0;
    }
  } else if (warp == 0) {
    list_adapters(id, list, count);
  }
  __syncthreads();
  const int total = count;
  const uint32_t tmem = bars->tmem;
  // this block's adapters of the tile: those from blockIdx.z on, gridDim.z apart, kAtOnce a pass
  const int mine_n = total > static_cast<int>(blockIdx.z) ? (total - blockIdx.z + gridDim.z - 1) / gridDim.z : 0;
  auto adapter = [&](int i) { return list[blockIdx.z + i * gridDim.z]; };

  if (warp == kTmaWarp) {
    if (lane == 0) {
      uint32_t it = 0, wt = 0;
      bool ok = true;
      for (int i0 = 0; ok && i0 < mine_n; i0 += C::kAtOnce) {
        const int n = min(C::kAtOnce, mine_n - i0);
        for (int kb = kb_lo; ok && kb < kb_hi; ++kb, ++it) {
          const int s = static_cast<int>(it % C::kXStages);
          if (!mbar_wait(&bars->empty[s], ((it / C::kXStages) & 1u) ^ 1u, abortv, err, kDevTimeoutEmpty)) {
            ok = false;
            break;
          }
          mbar_arrive_expect_tx(&bars->full[s], kCodes ? C::kRaw : kXTile);
          tma_load_2d(kCodes ? s_raw + s * C::kRaw : s_x + s * kXTile, &tm_x, &bars->full[s], kb * kSK,
                      static_cast<int>(row0));
          for (int i = 0; i < n; ++i, ++wt) {
            const int ws = static_cast<int>(wt % C::kWStages);
            if (!mbar_wait(&w_empty[ws], ((wt / C::kWStages) & 1u) ^ 1u, abortv, err, kDevTimeoutEmpty)) {
              ok = false;
              break;
            }
            constexpr uint32_t w_bytes = kWRows ? kRank * 128 : (kRank == 128 ? 2 : 1) * 64 * 128;
            mbar_arrive_expect_tx(&w_full[ws], w_bytes);
            uint8_t* w = s_w + ws * C::kW;
            const int ad = adapter(i0 + i);
            if constexpr (kWRows) {
              tma_load_3d(w, &tm_w, &w_full[ws], kb * kSK, 0, ad);
            } else {
              tma_load_3d(w, &tm_w, &w_full[ws], 0, kb * kSK, ad);
              if constexpr (kRank == 128) tma_load_3d(w + 8192, &tm_w, &w_full[ws], 64, kb * kSK, ad);
            }
          }
        }
      }
      if (!ok) let_copies_land();
    }
  } else if (warp == kMmaWarp) {
    if (lane == 0) {
      constexpr uint32_t idesc = idesc_bf16(kRank, 0, kWRows ? 0 : 1);
      uint32_t it = 0, wt = 0, pass = 0;
      bool ok = true;
      for (int i0 = 0; ok && i0 < mine_n; i0 += C::kAtOnce, ++pass) {
        const int n = min(C::kAtOnce, mine_n - i0);
        if (!mbar_wait(&bars->drained, (pass & 1u) ^ 1u, abortv, err, kDevTimeoutTmemEmpty)) break;
        tc_fence_after();
        for (int kb = kb_lo; ok && kb < kb_hi; ++kb, ++it) {
          const int s = static_cast<int>(it % C::kXStages);
          const uint32_t ph = (it / C::kXStages) & 1u;
          if (!mbar_wait(&bars->full[s], ph, abortv, err, kDevTimeoutFull) ||
              (kCodes && !mbar_wait(&bars->ready[s], ph, abortv, err, kDevTimeoutFull))) {
            ok = false;
            break;
          }
          const uint32_t a0 = smem_u32(s_x + s * kXTile);
          for (int i = 0; i < n; ++i, ++wt) {
            const int ws = static_cast<int>(wt % C::kWStages);
            if (!mbar_wait(&w_full[ws], (wt / C::kWStages) & 1u, abortv, err, kDevTimeoutFull)) {
              ok = false;
              break;
            }
            tc_fence_after();
            const uint32_t b0 = smem_u32(s_w + ws * C::kW);
#pragma unroll
            for (int k = 0; k < kSK / 16; ++k) {
              mma_bf16(tmem + i * kRank, smem_desc_k_sw128(a0 + k * 32),
                       kWRows ? smem_desc_k_sw128(b0 + k * 32) : smem_desc_mn_sw128(b0 + k * 2048, 8192), idesc,
                       (kb != kb_lo || k != 0) ? 1u : 0u);
            }
            umma_commit(&w_empty[ws]);
          }
          if (ok) umma_commit(&bars->empty[s]);
        }
        if (ok) umma_commit(&bars->done);
      }
    }
  } else {
    // x and W_s are the caller's; what is written may still be in use by the kernel before
    if (warp < 4) griddep_wait();
    if (counts && tid == 0 && blockIdx.y == 0 && blockIdx.z == 0) counts[blockIdx.x] = total;  // for expand_tc_kernel
    uint32_t it = 0, pass = 0;
    bool ok = true;
    for (int i0 = 0; ok && i0 < mine_n; i0 += C::kAtOnce, ++pass) {
      const int n = min(C::kAtOnce, mine_n - i0);
      if constexpr (kCodes) {
        // 128 rows x 64 codes: four neighbours share a row of 64 bytes
        for (int kb = kb_lo; kb < kb_hi; ++kb, ++it) {
          const int s = static_cast<int>(it % C::kXStages);
          const bool there =
              mbar_wait(&bars->full[s], (it / C::kXStages) & 1u, abortv, err, kDevTimeoutFull);
          if (!__all_sync(0xffffffffu, there)) {
            ok = false;
            break;
          }
          const uint8_t* raw = s_raw + s * C::kRaw;
          uint8_t* x = s_x + s * kXTile;
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int r = (tid >> 2) + 64 * i, c = tid & 3;
            uint4 lo8, hi8;
            widen16(*reinterpret_cast<const uint4*>(raw + r * 64 + c * 16), lo8, hi8);
            *reinterpret_cast<uint4*>(x + r * 128 + (((2 * c) ^ (r & 7)) << 4)) = lo8;
            *reinterpret_cast<uint4*>(x + r * 128 + (((2 * c + 1) ^ (r & 7)) << 4)) = hi8;
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&bars->ready[s]);
        }
        if (!ok) break;
      }
      if (warp >= 4) continue;
      const bool there = mbar_wait(&bars->done, pass & 1u, abortv, err, kDevTimeoutTmemFull);
      if (!__all_sync(0xffffffffu, there)) break;
      tc_fence_after();
      const int r = warp * 32 + lane;
      const int64_t row = row0 + r;
      const float mul = id[r] >= 0 && row_mul ? __ldg(row_mul + row) : 1.0f;
      float* dst = part + (static_cast<int64_t>(blockIdx.y) * rows.M + row) * R;
      for (int i = 0; i < n; ++i) {
        const bool mine = id[r] == adapter(i0 + i);
        constexpr int kLoad = kRank < 32 ? kRank : 32;  // no further than the block's columns
#pragma unroll
        for (int c = 0; c < kRank; c += kLoad) {
          uint32_t d[kLoad];
          __syncwarp();
          const uint32_t at = tmem + (static_cast<uint32_t>(warp * 32) << 16) + i * kRank + c;
          if constexpr (kLoad == 32) {
            tmem_ld_32x32b_x32(at, d);
          } else {
            tmem_ld_32x32b_x16(at, d);
          }
          tmem_ld_wait();
          if (mine) {
#pragma unroll
            for (int j = 0; j < kLoad; j += 4) {  // R % 8 == 0
              if (c + j < R) {
                *reinterpret_cast<float4*>(dst + c + j) =
                    make_float4(__uint_as_float(d[j]) * mul, __uint_as_float(d[j + 1]) * mul,
                                __uint_as_float(d[j + 2]) * mul, __uint_as_float(d[j + 3]) * mul);
              }
            }
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->drained);
    }
  }
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc<C::kCols>(tmem);
  }
}

// ======================================================================== pieces
// The rank side as tokens_tc reads it: out[piece][r][m] = bf16 pieces of
// mul[s] * row_mul[m] * (the splits' sum), zero in rows without an adapter, past M and
// past R (11712 rows at rank 64, both sides: 10 us); and info[s][tile]: 0 no row of adapter s in the tile of 64, 2 only such rows,
// 1 others too.  blockIdx.y: which of the two rank sides.
constexpr int kTile = 64;
struct RankSide {
  const float* part;
  int splits;
  const float* row_mul;
  __nv_bfloat16* out;
};
template <int kRank>
__global__ void __launch_bounds__(256) rank_pieces_kernel(RankSide a, RankSide b,
                                                          const float* __restrict__ scaling, Rows rows,
                                                          int R, int64_t m_pad, uint8_t* __restrict__ info) {
  __shared__ float v[kTile][kRank + 1];
  __shared__ TileIds ids;
  griddep_launch_dependents();
  const RankSide g = blockIdx.y ? b : a;
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * kTile;
  tile_ids(rows, row0, ids);
  griddep_wait();
  constexpr int kVecs = kRank / 4;
  constexpr int kEach = kTile * kVecs / 256;  // 1 .. 8 vectors a thread
  float4 sum[kEach];
  rank_sums<kVecs, 256, kEach>(g.part, g.splits, rows, row0, 0, threadIdx.x, R, sum);
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int at = threadIdx.x + i * 256;
    const int r = at / kVecs, c = (at % kVecs) * 4;
    const int own = ids.id[r];
    float mul = 1.0f;
    if (own >= 0 && scaling) mul = __ldg(scaling + own);
    if (own >= 0 && g.row_mul) mul *= __ldg(g.row_mul + row0 + r);
    v[r][c] = own >= 0 ? sum[i].x * mul : 0.0f;
    v[r][c + 1] = own >= 0 ? sum[i].y * mul : 0.0f;
    v[r][c + 2] = own >= 0 ? sum[i].z * mul : 0.0f;
    v[r][c + 3] = own >= 0 ? sum[i].w * mul : 0.0f;
  }
  __syncthreads();
#pragma unroll
  for (int i = threadIdx.x; i < kRank * (kTile / 8); i += 256) {
    const int c = i / (kTile / 8), r = (i % (kTile / 8)) * 8;
    uint4 first, second;
    uint32_t *f = reinterpret_cast<uint32_t*>(&first), *s = reinterpret_cast<uint32_t*>(&second);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float x = v[r + 2 * j][c], y = v[r + 2 * j + 1][c];
      const float x0 = next_piece(x), y0 = next_piece(y);
      f[j] = pack_bf16(x0, y0);
      s[j] = pack_bf16(x, y);
    }
    *reinterpret_cast<uint4*>(g.out + c * m_pad + row0 + r) = first;
    *reinterpret_cast<uint4*>(g.out + (kRank + c) * m_pad + row0 + r) = second;
  }
  if (blockIdx.y == 0) {
    for (int s = threadIdx.x; s < rows.S; s += 256) {
      int f = 0;
      for (int i = 0; i < ids.count; ++i) f = ids.list[i] == s ? 1 : f;
      if (f && ids.count == 1 && !ids.none) f = 2;
      info[static_cast<int64_t>(s) * gridDim.x + blockIdx.x] = static_cast<uint8_t>(f);
    }
  }
}

// ======================================================================== tokens
constexpr int kTCols = 256;
constexpr int kTilesMost = 2048;   // tiles of 64 rows a block goes through
constexpr int kAdaptersMost = 64;  // adapters of a call
template <bool kCodes, int kRank>
struct TokensTc {
  static constexpr int kX = kTile * kTCols * 2;            // four boxes of 64 columns, 32 KB
  static constexpr int kH = 2 * kRank * kTile * 2;
  static constexpr int kRaw = kCodes ? kTile * kTCols : 0;
  static constexpr int kStage = kX + kH + kRaw;
  static constexpr int kStagesRaw = (227 * 1024 - 1024 - kBarBytes - kTilesMost) / kStage;
  static constexpr int kStages = kStagesRaw > 6 ? 6 : kStagesRaw;
  static constexpr int kBytes = 1024 + kStages * kStage + kBarBytes + kTilesMost;
  static_assert(kStages >= 2 && kH % 1024 == 0, "tiles");
};

// A block takes 256 columns and a range of rows, so that x is read once for the whole
// rank; adapters one after the other, tiles without the adapter skipped.  Bound by
// reading x: 11712 x 12288 bf16 at rank 64 in 72 us (288 MB, 4.0 TB/s), 11712 x 4096
// codes, widened on the way, in 32 (48 MB).
// tm_x: boxes of 64 columns x 64 rows (codes: 256 x 64 bytes).  tm_h: the pieces,
// [2 kRank][m_pad], boxes 64 x 2 kRank.
template <bool kCodes, int kRank, bool kByCol>
__global__ void __launch_bounds__(kThreads, 1) tokens_tc_kernel(
    const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_h, Rows rows, int C, int R,
    int tiles, int tiles_split, const uint8_t* __restrict__ info, float* __restrict__ part,
    int* __restrict__ found) {
  using T = TokensTc<kCodes, kRank>;
  griddep_launch_dependents();
  // two accumulators of 2 kRank columns (the sums with the first pieces, then the second)
  constexpr uint32_t kTokenCols = 4 * kRank;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint8_t* s_x = smem;
  uint8_t* s_h = s_x + T::kStages * T::kX;
  uint8_t* s_raw = s_h + T::kStages * T::kH;
  Bars* bars = reinterpret_cast<Bars*>(s_raw + T::kStages * T::kRaw);
  uint8_t* live = reinterpret_cast<uint8_t*>(bars) + kBarBytes;
  __shared__ uint8_t present[kAdaptersMost];
  volatile int* abortv = &bars->abort_flag;
  int* err = &g_lora_error;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const int col0 = blockIdx.x * kTCols;
  const int t_lo = blockIdx.y * tiles_split, n_tiles = min(tiles - t_lo, tiles_split);

  if (tid == 0) {
    for (int i = 0; i < T::kStages; ++i) {
      mbar_init(&bars->full[i], 1);
      mbar_init(&bars->ready[i], 8);
      mbar_init(&bars->empty[i], 1);
    }
    mbar_init(&bars->done, 1);
    bars->abort_flag = 0;
    fence_mbarrier_init();
  }
  griddep_wait();  // info and the pieces
  // which adapters these rows have
  for (int s = warp; s < rows.S; s += kThreads / 32) {
    int any = 0;
    for (int i = lane; i < n_tiles; i += 32) any |= __ldcg(info + static_cast<int64_t>(s) * tiles + t_lo + i);
    any = __any_sync(0xffffffffu, any);
    if (lane == 0) {
      present[s] = static_cast<uint8_t>(any);
      if (blockIdx.x == 0) found[static_cast<int64_t>(blockIdx.y) * rows.S + s] = any;
    }
  }
  if (warp == kTmaWarp && lane == 0) {
    tma_prefetch_desc(&tm_x);
    tma_prefetch_desc(&tm_h);
  }
  if (warp == kMmaWarp) {
    tmem_alloc<kTokenCols>(&bars->tmem);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars->tmem;

  // one adapter after the other: its tiles, then its sums are written
  uint32_t it = 0, segment = 0;
  for (int s = 0; s < rows.S; ++s) {
    if (!present[s]) continue;
    for (int i = tid; i < n_tiles; i += kThreads) live[i] = __ldcg(info + static_cast<int64_t>(s) * tiles + t_lo + i);
    __syncthreads();
    tc_fence_after();
    if (warp == kTmaWarp) {
      if (lane == 0) {
        bool ok = true;
        for (int t = 0; ok && t < n_tiles; ++t) {
          if (!live[t]) continue;
          const int st = static_cast<int>(it % T::kStages);
          if (!mbar_wait(&bars->empty[st], ((it / T::kStages) & 1u) ^ 1u, abortv, err, kDevTimeoutEmpty)) {
            ok = false;
            break;
          }
          const int m = (t_lo + t) * kTile;
          mbar_arrive_expect_tx(&bars->full[st], (kCodes ? T::kRaw : T::kX) + T::kH);
          if constexpr (kCodes) {
            tma_load_2d(s_raw + st * T::kRaw, &tm_x, &bars->full[st], col0, m);
          } else {
#pragma unroll
            for (int c = 0; c < 4; ++c)
              tma_load_2d(s_x + st * T::kX + c * 8192, &tm_x, &bars->full[st], col0 + c * 64, m);
          }
          tma_load_2d(s_h + st * T::kH, &tm_h, &bars->full[st], m, 0);
          ++it;
        }
        if (!ok) let_copies_land();
      }
    } else if (warp == kMmaWarp) {
      if (lane == 0) {
        constexpr uint32_t idesc = idesc_bf16(2 * kRank, 1, 0);
        bool ok = true, first = true;
        for (int t = 0; t < n_tiles; ++t) {
          if (!live[t]) continue;
          const int st = static_cast<int>(it % T::kStages);
          const uint32_t ph = (it / T::kStages) & 1u;
          if (!mbar_wait(&bars->full[st], ph, abortv, err, kDevTimeoutFull) ||
              !mbar_wait(&bars->ready[st], ph, abortv, err, kDevTimeoutFull)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t a0 = smem_u32(s_x + st * T::kX), b0 = smem_u32(s_h + st * T::kH);
#pragma unroll
          for (int blk = 0; blk < 2; ++blk) {
#pragma unroll
            for (int k = 0; k < kTile / 16; ++k) {
              // both pieces side by side: the columns are read once for them
              mma_bf16(tmem + blk * 2 * kRank, smem_desc_mn_sw128(a0 + blk * 16384 + k * 2048, 8192),
                       smem_desc_k_sw128(b0 + k * 32), idesc, (!first || k != 0) ? 1u : 0u);
            }
          }
          umma_commit(&bars->empty[st]);
          first = false;
          ++it;
        }
        if (ok) umma_commit(&bars->done);
      }
    } else {
      bool ok = true;
      for (int t = 0; t < n_tiles; ++t) {
        const int f = live[t];
        if (!f) continue;
        const int st = static_cast<int>(it % T::kStages);
        const bool there = mbar_wait(&bars->full[st], (it / T::kStages) & 1u, abortv, err, kDevTimeoutFull);
        if (!__all_sync(0xffffffffu, there)) {
          ok = false;
          break;
        }
        const int64_t m0 = static_cast<int64_t>(t_lo + t) * kTile;
        uint8_t* x = s_x + st * T::kX;
        if constexpr (kCodes) {
          // 64 rows x 256 codes: 16 neighbours a row
          const uint8_t* raw = s_raw + st * T::kRaw;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int r = (tid >> 4) + 16 * i, c = tid & 15;  // 16 codes of the box c / 4
            uint4 lo8, hi8;
            widen16(*reinterpret_cast<const uint4*>(raw + r * kTCols + c * 16), lo8, hi8);
            uint8_t* row = x + (c >> 2) * 8192 + r * 128;
            const int at = 2 * (c & 3);
            *reinterpret_cast<uint4*>(row + ((at ^ (r & 7)) << 4)) = lo8;
            *reinterpret_cast<uint4*>(row + (((at + 1) ^ (r & 7)) << 4)) = hi8;
          }
        }
        if (f == 1) {
          // rows of other adapters (whatever they hold) leave the products: their
          // values and their rank side are zeroed
          const int r = tid & 63, quarter = tid >> 6;
          if (adapter_of(rows, m0 + r) != s) {
            if (!kCodes) {
              for (int q = 0; q < 8; ++q)
                *reinterpret_cast<uint4*>(x + quarter * 8192 + r * 128 + q * 16) = make_uint4(0, 0, 0, 0);
            }
            uint8_t* h = s_h + st * T::kH;
            for (int k = quarter * (kRank / 2); k < (quarter + 1) * (kRank / 2); ++k)
              *reinterpret_cast<uint16_t*>(h + k * 128 + (((r >> 3) ^ (k & 7)) << 4) + (r & 7) * 2) = 0;
          }
        }
        if (kCodes || f == 1) fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->ready[st]);
        ++it;
      }
      if (ok && warp < 4) {
        const bool there = mbar_wait(&bars->done, segment & 1u, abortv, err, kDevTimeoutTmemFull);
        if (__all_sync(0xffffffffu, there)) {
          tc_fence_after();
          float* dst = part + (static_cast<int64_t>(blockIdx.y) * rows.S + s) * R * C;
#pragma unroll
          for (int blk = 0; blk < 2; ++blk) {
            const int c = col0 + blk * 128 + warp * 32 + lane;
#pragma unroll
            for (int k = 0; k < kRank; k += 32) {
              uint32_t v[32], w[32];
              __syncwarp();
              const uint32_t at = tmem + (static_cast<uint32_t>(warp * 32) << 16) + blk * 2 * kRank + k;
              tmem_ld_32x32b_x32(at, v);
              if constexpr (kRank >= 32) tmem_ld_32x32b_x32(at + kRank, w);
              tmem_ld_wait();
#pragma unroll
              for (int j = 0; j < 32; ++j) {
                const uint32_t second = kRank >= 32 ? w[j] : v[(j + 16) & 31];
                v[j] = __float_as_uint(__uint_as_float(v[j]) + __uint_as_float(second));
              }
              if (c < C) {
                if constexpr (kByCol) {
                  float* p = dst + static_cast<int64_t>(c) * R + k;
#pragma unroll
                  for (int j = 0; j < 32; j += 4)  // R % 8 == 0
                    if (k + j < R && j < kRank)
                      *reinterpret_cast<uint4*>(p + j) = make_uint4(v[j], v[j + 1], v[j + 2], v[j + 3]);
                } else {
#pragma unroll
                  for (int j = 0; j < 32; ++j)
                    if (k + j < R && j < kRank) dst[static_cast<int64_t>(k + j) * C + c] = __uint_as_float(v[j]);
                }
              }
            }
          }
          tc_fence_before();
        }
      }
    }
    ++segment;
    __syncthreads();  // the accumulators and the list are read
    if (*abortv) break;
  }
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc<kTokenCols>(tmem);
  }
}

// ======================================================================== expand
// out[row, n] = bf16(y[row, n] + c[s] * sum_r h[row, r] W_s[r, n]); y NULL: zero.
// One block a multiprocessor takes an equal share of all 128 x 64 tiles, row tile by
// row tile, a tile counted as often as it takes (its adapters are counted by the
// shrink kernel): a segment is its run of columns in one row tile, whose h it keeps as
// pieces in shared memory.  y arrives by TMA up to eight tiles ahead, W_s four; two
// groups of four warps take the tiles in turn, add the product to y in place in shared
// memory, and a TMA store takes the tile away.  Each group has two accumulators and two
// pairs of barriers of its own: a wait tells apart only odd and even phases, so a warp has to
// see every phase of a barrier it waits on, and a tile's products may be any number.  Bound by reading y and writing out: 11712 x 12288 at rank 64 in 112 us,
// 561 MB of HBM traffic at 5.0 TB/s (a copy reaches 6.5).
// Three stages and one group of warps, twice a multiprocessor, waited for the loads:
// 178 us on 11712 x 12288 at rank 64.
// Every row of a tile keeps the h of its own adapter; a tile whose rows have
// different ones is multiplied by each adapter's W_s and a row takes its own's.
constexpr int kERows = 128, kECols = 64;
constexpr int kEThreads = 320, kETmaWarp = 8, kEMmaWarp = 9;
template <int kRank>
struct ExpandTc {
  static constexpr int kBlks = kRank > 64 ? 2 : 1;             // blocks of 64 of the rank
  static constexpr int kHBlk = kERows * 128;                   // 16 KB
  static constexpr int kH = 2 * kBlks * kHBlk;
  static constexpr int kW = kBlks * kECols * 128;              // 8 KB a block, either way round
  static constexpr int kY = kERows * kECols * 2;
  static constexpr int kYStages = kBlks == 2 ? 6 : 8;
  static constexpr int kWStages = kBlks == 2 ? 3 : 4;
  static constexpr int kBytes = 1024 + kH + kYStages * kY + kWStages * kW + kBarBytes + 1024;
  static_assert(kBytes <= 232448, "shared memory");
};

// What a tile of rows with so many adapters costs: a second product takes the thread
// that issues them 1100 cycles, where HBM needs 1260 for the tile.  Where every tile
// has a block (`each`), one: a block with tiles of two row tiles takes twice as long.
__device__ __forceinline__ int tile_cost(int adapters, bool each) {
  return each ? 1 : adapters <= 1 ? 4 : 3 * adapters + 1;
}

template <int kRank, bool kWCols>
__global__ void __launch_bounds__(kEThreads, 1) expand_tc_kernel(
    const __grid_constant__ CUtensorMap tm_y, const __grid_constant__ CUtensorMap tm_w,
    const __grid_constant__ CUtensorMap tm_out, const __nv_bfloat16* y, __nv_bfloat16* out,
    const int* __restrict__ counts, const float* __restrict__ part, int splits, const float* __restrict__ scaling, Rows rows, int N,
    int R) {
  using C = ExpandTc<kRank>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint8_t* s_h = smem;
  uint8_t* s_y = s_h + C::kH;
  uint8_t* s_w = s_y + C::kYStages * C::kY;
  Bars* bars = reinterpret_cast<Bars*>(s_w + C::kWStages * C::kW);
  uint64_t *y_full = bars->full, *y_empty = bars->empty;
  uint64_t *w_full = bars->w_full, *w_empty = bars->w_empty;
  uint64_t* tfull = bars->acc;         // four accumulators, 2 g and 2 g + 1 group g's
  uint64_t* tempty = bars->acc + 4;
  uint64_t* h_there = &bars->done;
  int* id = reinterpret_cast<int*>(reinterpret_cast<uint8_t*>(bars) + kBarBytes);
  int* list = id + kERows;
  __shared__ int count;
  __shared__ int64_t scan[kEThreads / 32], share[2], start_tile, start_at;
  volatile int* abortv = &bars->abort_flag;
  int* err = &g_lora_error;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const int col_tiles = (N + kECols - 1) / kECols;
  const int64_t row_tiles = (rows.M + kERows - 1) / kERows;
  if (tid == 0) {
    for (int s = 0; s < C::kYStages; ++s) {
      mbar_init(&y_full[s], 1);
      mbar_init(&y_empty[s], 4);  // the four warps that take the tile
    }
    for (int s = 0; s < C::kWStages; ++s) {
      mbar_init(&w_full[s], 1);
      mbar_init(&w_empty[s], 1);
    }
    for (int b = 0; b < 4; ++b) {
      mbar_init(&tfull[b], 1);
      mbar_init(&tempty[b], 4);  // the warps of its group
    }
    mbar_init(h_there, 8);
    bars->abort_flag = 0;
    fence_mbarrier_init();
  }
  if (warp == kETmaWarp && lane == 0) {
    tma_prefetch_desc(&tm_y);
    tma_prefetch_desc(&tm_w);
    tma_prefetch_desc(&tm_out);
  }
  if (warp == kEMmaWarp) {
    tmem_alloc<4 * kECols>(&bars->tmem);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  griddep_launch_dependents();  // after the allocation, as in shrink_tc_kernel
  const uint32_t tmem = bars->tmem;
  uint32_t yt = 0;       // tiles this block has gone through; odd ones are group 1's
  uint32_t wt = 0;       // products (a tile times an adapter)
  uint32_t made[2] = {0, 0};  // of them, of each group's tiles (epilogue: its own group's alone)
  uint32_t h_count = 0;  // times h has been laid down
  int to_free = -1;      // the stage whose store may still be reading

  griddep_wait();  // the rank side, and the adapters' counts
  // this block's share [lo, hi) of the whole cost, and the row tile it starts in: a
  // thread adds up a run of row tiles, a scan over the block gives the run's start
  const bool each = gridDim.x == row_tiles * col_tiles;
  {
    const int64_t run = (row_tiles + kEThreads - 1) / kEThreads;
    const int64_t first = min(row_tiles, tid * run), last = min(row_tiles, first + run);
    int64_t mine = 0;
    for (int64_t i = first; i < last; ++i) mine += tile_cost(__ldcg(counts + i), each);
    int64_t upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t other = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += other;
    }
    if (lane == 31) scan[warp] = upto;
    __syncthreads();
    int64_t before = upto - mine, total = 0;
#pragma unroll
    for (int w = 0; w < kEThreads / 32; ++w) {
      if (w < warp) before += scan[w];
      total += scan[w];
    }
    total *= col_tiles;
    const int64_t lo = total * blockIdx.x / gridDim.x, hi = total * (blockIdx.x + 1) / gridDim.x;
    int64_t at = before * col_tiles;
    for (int64_t i = first; i < last; ++i) {
      const int64_t end = at + static_cast<int64_t>(tile_cost(__ldcg(counts + i), each)) * col_tiles;
      if (lo >= at && lo < end) {
        start_tile = i;
        start_at = at;
      }
      at = end;
    }
    if (tid == 0) {
      share[0] = lo;
      share[1] = hi;
    }
  }
  __syncthreads();
  const int64_t lo = share[0], hi = share[1];
  int64_t at = start_at;
  for (int64_t rt = start_tile; rt < row_tiles && at < hi; ++rt) {
    // the row tile's tiles that start in the share
    const int64_t cost = tile_cost(__ldcg(counts + rt), each);
    const int t_lo = static_cast<int>(lo <= at ? 0 : min(static_cast<int64_t>(col_tiles), (lo - at + cost - 1) / cost));
    const int t_hi = static_cast<int>(min(static_cast<int64_t>(col_tiles), (hi - at + cost - 1) / cost));
    at += cost * col_tiles;
    if (t_lo >= t_hi) continue;
    const int64_t row0 = rt * kERows;
    // the adapters of the rows; usually one
    int v = -1;
    if (tid < kERows) {
      v = adapter_of(rows, row0 + tid);
      id[tid] = v;
    }
    __syncthreads();
    const bool one = __syncthreads_and(tid >= kERows || row0 + tid >= rows.M || v == id[0]);
    if (one) {
      if (tid == 0) {
        list[0] = id[0];
        count = id[0] >= 0 ? 1 : 0;
      }
    } else if (warp == 0) {
      list_adapters(id, list, count);
    }
    __syncthreads();
    const int n = count;
    if (n == 0 && y == out) continue;  // nothing to add (the ids are not read again)

    if (warp == kETmaWarp) {
      if (lane == 0) {
        bool ok = true;
        for (int t = t_lo; ok && t < t_hi; ++t, ++yt) {
          const int s = static_cast<int>(yt % C::kYStages);
          if (!mbar_wait(&y_empty[s], ((yt / C::kYStages) & 1u) ^ 1u, abortv, err, kDevTimeoutEmpty)) {
            ok = false;
            break;
          }
          if (y) {
            mbar_arrive_expect_tx(&y_full[s], C::kY);
            tma_load_2d(s_y + s * C::kY, &tm_y, &y_full[s], t * kECols, static_cast<int>(row0));
          } else {
            mbar_arrive(&y_full[s]);
          }
          for (int li = 0; li < n; ++li, ++wt) {
            const int ws = static_cast<int>(wt % C::kWStages);
            if (!mbar_wait(&w_empty[ws], ((wt / C::kWStages) & 1u) ^ 1u, abortv, err, kDevTimeoutEmpty)) {
              ok = false;
              break;
            }
            constexpr uint32_t w_bytes = kWCols ? C::kW : kRank * 128;
            mbar_arrive_expect_tx(&w_full[ws], w_bytes);
            uint8_t* w = s_w + ws * C::kW;
            if constexpr (kWCols) {
#pragma unroll
              for (int b = 0; b < C::kBlks; ++b)
                tma_load_3d(w + b * 8192, &tm_w, &w_full[ws], b * 64, t * kECols, list[li]);
            } else {
              tma_load_3d(w, &tm_w, &w_full[ws], t * kECols, 0, list[li]);
            }
          }
        }
        if (!ok) let_copies_land();
      }
    } else if (warp == kEMmaWarp) {
      if (lane == 0) {
        constexpr uint32_t idesc = idesc_bf16(kECols, 0, kWCols ? 0 : 1);
        bool ok = mbar_wait(h_there, h_count & 1u, abortv, err, kDevTimeoutFull);
        ++h_count;
        const uint32_t tiles = static_cast<uint32_t>(t_hi - t_lo);
        const uint32_t products = tiles * static_cast<uint32_t>(n);
        uint32_t left = static_cast<uint32_t>(n);  // of the tile
        uint32_t group = yt & 1u;
        yt += tiles;
        for (uint32_t i = 0; ok && i < products; ++i, ++wt) {
          if (left == 0) {
            left = static_cast<uint32_t>(n);
            group ^= 1u;
          }
          --left;
          const int ws = static_cast<int>(wt % C::kWStages);
          const uint32_t j = group ? made[1]++ : made[0]++;
          const uint32_t acc = 2 * group + (j & 1u);
          if (!mbar_wait(&tempty[acc], ((j >> 1) & 1u) ^ 1u, abortv, err, kDevTimeoutTmemEmpty) ||
              !mbar_wait(&w_full[ws], (wt / C::kWStages) & 1u, abortv, err, kDevTimeoutFull)) {
            break;
          }
          tc_fence_after();
          const uint32_t h0 = smem_u32(s_h), w0 = smem_u32(s_w + ws * C::kW);
#pragma unroll
          for (int k = 0; k < kRank / 16; ++k) {
            const int blk = k / 4, off = (k % 4) * 32;
            const uint64_t bd =
                kWCols ? smem_desc_k_sw128(w0 + blk * 8192 + off) : smem_desc_mn_sw128(w0 + k * 2048, 8192);
#pragma unroll
            for (int p = 0; p < 2; ++p) {
              mma_bf16(tmem + acc * kECols, smem_desc_k_sw128(h0 + (p * C::kBlks + blk) * C::kHBlk + off), bd,
                       idesc, (k != 0 || p != 0) ? 1u : 0u);
            }
          }
          umma_commit(&w_empty[ws]);
          umma_commit(&tfull[acc]);
        }
      }
    } else {
      const int quad = warp & 3, group = warp >> 2;
      const int r = quad * 32 + lane;
      const int64_t row = row0 + r;
      const int own = id[r];
      // the rows' h as pieces (zero without an adapter), sixteen rows a warp, a lane a
      // vector of four of a row: with a lane a row, 14 splits of 2005 x 64 took the kernel
      // 36 us, now 15.  The products with the last one are done (see the barrier below)
      constexpr int kV = kRank / 4, kEach = kV / 2;
      float4 sum[kEach];
      rank_sums<kV, 32, kEach>(part, splits, rows, row0, warp * 16, lane, R, sum);
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        const int hr = warp * 16 + (lane + i * 32) / kV, c = (lane + i * 32) % kV * 4;
        float x[4] = {sum[i].x, sum[i].y, sum[i].z, sum[i].w};
        if (id[hr] < 0) x[0] = x[1] = x[2] = x[3] = 0.0f;
        const float x0 = next_piece(x[0]), x1 = next_piece(x[1]), x2 = next_piece(x[2]), x3 = next_piece(x[3]);
        uint8_t* h = s_h + (c >> 6) * C::kHBlk + hr * 128 + ((((c >> 3) & 7) ^ (hr & 7)) << 4) + (c & 4) * 2;
        *reinterpret_cast<uint2*>(h) = make_uint2(pack_bf16(x0, x1), pack_bf16(x2, x3));
        *reinterpret_cast<uint2*>(h + C::kBlks * C::kHBlk) = make_uint2(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]));
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(h_there);
      const float mul = own >= 0 && scaling ? __ldg(scaling + own) : 1.0f;
      bool ok = true;
      for (int t = t_lo; ok && t < t_hi; ++t, ++yt) {
        if (static_cast<int>(yt & 1u) != group) continue;
        const int s = static_cast<int>(yt % C::kYStages);
        bool there = mbar_wait(&y_full[s], (yt / C::kYStages) & 1u, abortv, err, kDevTimeoutFull);
        if (!__all_sync(0xffffffffu, there)) {
          ok = false;
          break;
        }
        uint8_t* yr = s_y + s * C::kY + r * 128;
        if (!y && own < 0) {
#pragma unroll
          for (int c = 0; c < 8; ++c) *reinterpret_cast<uint4*>(yr + (c << 4)) = make_uint4(0, 0, 0, 0);
        }
        for (int li = 0; li < n; ++li) {
          const uint32_t j = made[0]++;
          const uint32_t acc = 2 * static_cast<uint32_t>(group) + (j & 1u);
          there = mbar_wait(&tfull[acc], (j >> 1) & 1u, abortv, err, kDevTimeoutTmemFull);
          if (!__all_sync(0xffffffffu, there)) {
            ok = false;
            break;
          }
          if (!__any_sync(0xffffffffu, own == list[li])) {  // none of these 32 rows
            if (lane == 0) mbar_arrive(&tempty[acc]);
            continue;
          }
          tc_fence_after();
          uint32_t d[2][32];
          const uint32_t at = tmem + (static_cast<uint32_t>(quad * 32) << 16) + acc * kECols;
          tmem_ld_32x32b_x32(at, d[0]);
          tmem_ld_32x32b_x32(at + 32, d[1]);
          tmem_ld_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&tempty[acc]);
          if (own == list[li]) {
#pragma unroll
            for (int c = 0; c < 8; ++c) {
              uint4* cell = reinterpret_cast<uint4*>(yr + ((c ^ (r & 7)) << 4));
              const uint4 b = y ? *cell : make_uint4(0, 0, 0, 0);
              const uint32_t w4[4] = {b.x, b.y, b.z, b.w};
              uint32_t o[4];
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                const float x0 = __uint_as_float(d[c >> 2][(c & 3) * 8 + 2 * q]);
                const float x1 = __uint_as_float(d[c >> 2][(c & 3) * 8 + 2 * q + 1]);
                o[q] = pack_bf16(fmaf(mul, x0, __uint_as_float(w4[q] << 16)),
                                 fmaf(mul, x1, __uint_as_float(w4[q] & 0xFFFF0000u)));
              }
              *cell = make_uint4(o[0], o[1], o[2], o[3]);
            }
          }
          __syncwarp();
        }
        if (!ok) break;
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          if (row0 + quad * 32 < rows.M)
            tma_store_2d(&tm_out, s_y + s * C::kY + quad * 4096, t * kECols, static_cast<int>(row0) + quad * 32);
          tma_store_commit();
          if (to_free >= 0) {
            tma_store_wait_read<1>();  // this group's tile before has left shared memory
            mbar_arrive(&y_empty[to_free]);
          }
          to_free = s;
        }
      }
      // both groups have seen the products of all their tiles: h may be replaced
      named_bar_sync(1, 256);
      if (lane == 0 && to_free >= 0) {
        tma_store_wait_read<0>();
        mbar_arrive(&y_empty[to_free]);
        to_free = -1;
      }
    }
    __syncthreads();  // the segment's ids are read
    if (*abortv) break;
  }
  if (warp < kETmaWarp && lane == 0) tma_store_wait_all<0>();
  __syncthreads();
  if (warp == kEMmaWarp) {
    tc_fence_after();
    tmem_dealloc<4 * kECols>(tmem);
  }
}

// ---------------------------------------------------------------- host
PFN_cuTensorMapEncodeTiled_v12000 encoder() {
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

// A map of `rank` dimensions (innermost first), element strides of the outer ones.
bool map_of(CUtensorMap* map, bool bytes, int rank, const void* base, const int64_t* dims,
            const int64_t* strides, const uint32_t* box, bool swizzled) {
  auto fn = encoder();
  cuuint64_t d[3], st[2];
  cuuint32_t bx[3], ones[3] = {1, 1, 1};
  for (int i = 0; i < rank; ++i) {
    d[i] = static_cast<cuuint64_t>(dims[i]);
    bx[i] = box[i];
    if (i) st[i - 1] = static_cast<cuuint64_t>(strides[i - 1]) * (bytes ? 1 : 2);
  }
  return fn && fn(map, bytes ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, rank,
                  const_cast<void*>(base), d, st, bx, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  swizzled ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int refused(const char* what) {
  set_error("cuTensorMapEncodeTiled rejected the operands of %s", what);
  return W8A8_ERR_RUNTIME;
}

template <typename K>
int opt_in(K kernel, int bytes) {
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != cudaSuccess) {
    set_error("lora: shared memory of %d bytes refused: %s", bytes, cudaGetErrorString(e));
    return W8A8_ERR_ACCELERATOR;
  }
  return 0;
}

int launched(const char* what) {
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) {
    set_error("%s launch failed: %s", what, cudaGetErrorString(e));
    return W8A8_ERR_ACCELERATOR;
  }
  return 0;
}

int chained(const char* what, cudaError_t e) {
  if (e != cudaSuccess) {
    set_error("%s launch failed: %s", what, cudaGetErrorString(e));
    return W8A8_ERR_ACCELERATOR;
  }
  return 0;
}

template <bool kCodes, int kRank, bool kWRows>
int shrink_rank(const ShrinkTcArgs& g, const Rows& rows, cudaStream_t stream) {
  CUtensorMap tx, tw;
  const int64_t xd[2] = {g.K, g.M}, xs[1] = {g.ldx};
  const uint32_t xb[2] = {kSK, kSRows};
  const int64_t wd[3] = {kWRows ? g.K : g.R, kWRows ? g.R : g.K, g.S};
  const int64_t wst[2] = {kWRows ? g.K : g.R, g.S > 1 ? g.slot : g.R * g.K};
  const uint32_t wb[3] = {64, kWRows ? static_cast<uint32_t>(kRank) : 64u, 1};
  if (!map_of(&tx, kCodes, 2, g.x, xd, xs, xb, !kCodes) || !map_of(&tw, false, 3, g.w, wd, wst, wb, true)) {
    return refused("the adapters' contraction");
  }
  auto k = shrink_tc_kernel<kCodes, kRank, kWRows>;
  constexpr int bytes = ShrinkTc<kCodes, kRank>::kBytes;
  if (int rc = opt_in(k, bytes)) return rc;
  const dim3 grid(static_cast<unsigned>((g.M + kSRows - 1) / kSRows), g.splits, g.parts);
  if (g.first) {
    k<<<grid, kThreads, bytes, stream>>>(tx, tw, rows, g.x_scale, static_cast<int>(g.K), static_cast<int>(g.R),
                                       g.kb_split, g.part, g.counts);
    return launched("lora shrink");
  }
  return chained("lora shrink",
                 launch_chained(true, k, grid, kThreads, bytes, stream, tx, tw, rows, g.x_scale,
                                static_cast<int>(g.K), static_cast<int>(g.R), g.kb_split, g.part, g.counts));
}

template <bool kCodes, bool kWRows>
int shrink_codes(const ShrinkTcArgs& g, const Rows& rows, cudaStream_t stream) {
  if (g.R <= 16) return shrink_rank<kCodes, 16, kWRows>(g, rows, stream);
  if (g.R <= 32) return shrink_rank<kCodes, 32, kWRows>(g, rows, stream);
  if (g.R <= 64) return shrink_rank<kCodes, 64, kWRows>(g, rows, stream);
  return shrink_rank<kCodes, 128, kWRows>(g, rows, stream);
}

template <bool kCodes, int kRank, bool kByCol>
int tokens_rank(const TokensTcArgs& g, const Rows& rows, cudaStream_t stream) {
  CUtensorMap tx, th;
  const int64_t tiles = (g.M + kTile - 1) / kTile;
  const int64_t xd[2] = {g.C, g.M}, xs[1] = {g.ldx};
  const uint32_t xb[2] = {kCodes ? 256u : 64u, kTile};
  const int64_t hd[2] = {tiles * kTile, 2 * kRank}, hs[1] = {tiles * kTile};
  const uint32_t hb[2] = {kTile, 2 * kRank};
  if (!map_of(&tx, kCodes, 2, g.x, xd, xs, xb, !kCodes) || !map_of(&th, false, 2, g.pieces, hd, hs, hb, true)) {
    return refused("the adapters' gradient");
  }
  auto k = tokens_tc_kernel<kCodes, kRank, kByCol>;
  constexpr int bytes = TokensTc<kCodes, kRank>::kBytes;
  if (int rc = opt_in(k, bytes)) return rc;
  const dim3 grid(static_cast<unsigned>((g.C + kTCols - 1) / kTCols), g.splits);
  return chained("lora tokens",
                 launch_chained(true, k, grid, kThreads, bytes, stream, tx, th, rows, static_cast<int>(g.C),
                                static_cast<int>(g.R), static_cast<int>(tiles), g.tiles_split, g.info, g.part, g.found));
}

template <bool kCodes, bool kByCol>
int tokens_codes(const TokensTcArgs& g, const Rows& rows, cudaStream_t stream) {
  if (g.R <= 16) return tokens_rank<kCodes, 16, kByCol>(g, rows, stream);
  if (g.R <= 32) return tokens_rank<kCodes, 32, kByCol>(g, rows, stream);
  if (g.R <= 64) return tokens_rank<kCodes, 64, kByCol>(g, rows, stream);
  return tokens_rank<kCodes, 128, kByCol>(g, rows, stream);
}

template <int kRank, bool kWCols>
int expand_rank(const ExpandTcArgs& g, const Rows& rows, cudaStream_t stream) {
  CUtensorMap ty, tw, to;
  const int64_t od[2] = {g.N, g.M}, os[1] = {g.ldo}, ys[1] = {g.ldy};
  const uint32_t yb[2] = {kECols, kERows}, ob[2] = {kECols, 32};
  const int64_t wd[3] = {kWCols ? g.R : g.N, kWCols ? g.N : g.R, g.S};
  const int64_t wst[2] = {kWCols ? g.R : g.N, g.S > 1 ? g.slot : g.R * g.N};
  const uint32_t wb[3] = {64, kWCols ? 64u : static_cast<uint32_t>(kRank), 1};
  if (!map_of(&to, false, 2, g.out, od, os, ob, true) ||
      !map_of(&ty, false, 2, g.y ? g.y : g.out, od, g.y ? ys : os, yb, true) ||
      !map_of(&tw, false, 3, g.w, wd, wst, wb, true)) {
    return refused("the adapters' product");
  }
  auto k = expand_tc_kernel<kRank, kWCols>;
  constexpr int bytes = ExpandTc<kRank>::kBytes;
  if (int rc = opt_in(k, bytes)) return rc;
  const int64_t tiles = (g.M + kERows - 1) / kERows * ((g.N + kECols - 1) / kECols);
  const dim3 grid(static_cast<unsigned>(std::min<int64_t>(tiles, device_sm_count())));
  return chained("lora expand",
                 launch_chained(true, k, grid, kEThreads, bytes, stream, ty, tw, to,
                                static_cast<const __nv_bfloat16*>(g.y), static_cast<__nv_bfloat16*>(g.out), g.counts,
                                g.part, g.splits, g.scaling, rows, static_cast<int>(g.N), static_cast<int>(g.R)));
}

template <bool kWCols>
int expand_cols(const ExpandTcArgs& g, const Rows& rows, cudaStream_t stream) {
  if (g.R <= 16) return expand_rank<16, kWCols>(g, rows, stream);
  if (g.R <= 32) return expand_rank<32, kWCols>(g, rows, stream);
  if (g.R <= 64) return expand_rank<64, kWCols>(g, rows, stream);
  return expand_rank<128, kWCols>(g, rows, stream);
}

template <int kRank>
int pieces_rank(const RankPiecesArgs& g, const Rows& rows, cudaStream_t stream) {
  const int64_t tiles = (rows.M + kTile - 1) / kTile;
  const RankSide a{g.part_a, g.splits_a, g.row_mul_a, static_cast<__nv_bfloat16*>(g.out_a)};
  const RankSide b{g.part_b, g.splits_b, nullptr, static_cast<__nv_bfloat16*>(g.out_b)};
  return chained("lora rank pieces",
                 launch_chained(true, rank_pieces_kernel<kRank>, dim3(static_cast<unsigned>(tiles), 2), 256, 0,
                                stream, a, b, g.scaling, rows, g.R, tiles * kTile, g.info));
}

}  // namespace

int lora_shrink_tc(const ShrinkTcArgs& g, const LoraRows& r, cudaStream_t stream) {
  const Rows rows = rows_of(r);
  if (g.codes) return shrink_codes<true, true>(g, rows, stream);  // codes are x, which meets A
  return g.w_rows ? shrink_codes<false, true>(g, rows, stream) : shrink_codes<false, false>(g, rows, stream);
}

int lora_tokens_tc(const TokensTcArgs& g, const LoraRows& r, cudaStream_t stream) {
  const Rows rows = rows_of(r);
  if (g.codes) return tokens_codes<true, false>(g, rows, stream);
  return g.by_col ? tokens_codes<false, true>(g, rows, stream) : tokens_codes<false, false>(g, rows, stream);
}

int lora_expand_tc(const ExpandTcArgs& g, const LoraRows& r, cudaStream_t stream) {
  const Rows rows = rows_of(r);
  return g.w_cols ? expand_cols<true>(g, rows, stream) : expand_cols<false>(g, rows, stream);
}

int lora_rank_pieces(const RankPiecesArgs& g, const LoraRows& r, cudaStream_t stream) {
  const Rows rows = rows_of(r);
  if (g.R <= 16) return pieces_rank<16>(g, rows, stream);
  if (g.R <= 32) return pieces_rank<32>(g, rows, stream);
  if (g.R <= 64) return pieces_rank<64>(g, rows, stream);
  return pieces_rank<128>(g, rows, stream);
}

}  // namespace w8a8
