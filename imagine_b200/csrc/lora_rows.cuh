// Rows of a batch and the adapters they use: shared by the adapter kernels.
#pragma once
#include <cuda_runtime.h>

#include <cstdint>

#include "w8a8_internal.h"

namespace w8a8 {

constexpr int kBM = 64;  // rows per tile

// ---- rows and their adapters
struct Rows {
  const void* idx;  // int32 or int64 [ceil(M / per)], or NULL: adapter 0
  int idx64;
  int64_t per;      // consecutive rows that share an index
  int64_t M;
  int S;
};

__device__ __forceinline__ int adapter_of(const Rows& r, int64_t row) {
  if (row >= r.M) return -1;
  if (!r.idx) return 0;
  const int64_t i = r.per == 1 ? row : row / r.per;
  const int64_t v = r.idx64 ? __ldg(static_cast<const long long*>(r.idx) + i)
                            : static_cast<int64_t>(__ldg(static_cast<const int*>(r.idx) + i));
  return v >= 0 && v < r.S ? static_cast<int>(v) : -1;
}

// The adapters of a tile of 64 rows: id[i] each row's, list the distinct ones
// (in order of appearance), *count how many, *none whether a row has none.
struct TileIds {
  int id[kBM];
  int list[kBM];
  int count;
  int none;
};

__device__ __forceinline__ void tile_ids(const Rows& rows, int64_t row0, TileIds& t) {
  if (threadIdx.x < 32) {
    const unsigned all = 0xffffffffu;
    const int lane = threadIdx.x;
    const int a = adapter_of(rows, row0 + lane);
    const int b = adapter_of(rows, row0 + 32 + lane);
    t.id[lane] = a;
    t.id[lane + 32] = b;
    // every lane takes part in every warp operation: their results are tested afterwards
    const unsigned same_a = __match_any_sync(all, a);
    const unsigned same_b = __match_any_sync(all, b);
    const bool first_a = a >= 0 && __ffs(same_a) - 1 == lane;
    bool first_b = b >= 0 && __ffs(same_b) - 1 == lane;
#pragma unroll
    for (int j = 0; j < 32; ++j) {
      const int other = __shfl_sync(all, a, j);
      first_b = first_b && other != b;
    }
    const unsigned ma = __ballot_sync(all, first_a);
    const unsigned mb = __ballot_sync(all, first_b);
    const unsigned below = (1u << lane) - 1u;
    if (first_a) t.list[__popc(ma & below)] = a;
    if (first_b) t.list[__popc(ma) + __popc(mb & below)] = b;
    const bool n = (a < 0 && row0 + lane < rows.M) || (b < 0 && row0 + 32 + lane < rows.M);
    const bool any = __any_sync(all, n);
    if (lane == 0) {
      t.count = __popc(ma) + __popc(mb);
      t.none = any;
    }
  }
  __syncthreads();
}

// Launches a kernel of a chain: it may start while the one before it on the stream
// still runs, waits (griddep_wait) before it reads what that one wrote or writes
// anything, and lets the next one start in turn (griddep_launch_dependents).  What
// the call's user wrote is there from the start: the chain's first kernel is
// launched plainly (`early` false).  Hiding launches and prologues is worth it at every size: calls
// one after another, early against not, gradients of 5856 rows, 4096 -> 4096, rank 16 in 81 us
// against 98, of 11712 rows, 4096 -> 12288, rank 64 in 237 against 260 (forward 142 against
// 145), of 40000 rows, 4096 -> 4096, rank 32 in 380 against 405.
template <typename... P, typename... A>
cudaError_t launch_chained(bool early, void (*kernel)(P...), dim3 grid, int threads, int bytes, cudaStream_t stream,
                           A... args) {
  cudaLaunchConfig_t lc{};
  lc.gridDim = grid;
  lc.blockDim = dim3(threads);
  lc.dynamicSmemBytes = bytes;
  lc.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  lc.attrs = attr;
  lc.numAttrs = early ? 1 : 0;
  return cudaLaunchKernelEx(&lc, kernel, static_cast<P>(args)...);
}

inline Rows rows_of(const LoraRows& r) { return {r.idx, r.idx64, r.per, r.M, static_cast<int>(r.S)}; }

}  // namespace w8a8
