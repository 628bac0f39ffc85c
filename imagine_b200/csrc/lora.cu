// Low-rank adapters beside a W8A8 projection: many adapters in one batch, and
// their gradients.
//
// Row m uses adapter s = adapter[m / per] of S stacked ones, A[s] [R, K] and
// B[s] [N, R], c[s] its scaling; an s outside [0, S) means no adapter.
//   h = x A[s]^T            out = y + c h B[s]^T
//   g = dy B[s]             dx  = (dx +) c g A[s]
//   dA[s] = c sum_m g^T x   dB[s] = c sum_m dy^T h      (m over the rows of s)
// Kernels (of long bf16 batches: lora_sm100.cu):
//   shrink      [rows, K] x [K, R]: contracts a row with an adapter (h and g); both in one launch
//               in the backward pass (shrink_pair_kernel)
//   expand      [rows, R] x [R, N]: adds the low-rank product to a row (out, dx)
//   tokens      [R, rows] x [rows, C]: contracts over the rows of an adapter (dA and dB in one launch)
//   sum_splits  adds up the pieces of dA and dB that blocks of rows made
//   shrink_row, expand_row   the first two for few rows, on CUDA cores
//
// Arithmetic.  The products run on the tensor cores as bf16 x bf16 -> fp32.  A
// value that bf16 does not hold is cut into bf16 pieces that add up to it
// (each piece rounded from what is left): f16 into two, fp32 into three,
// both exactly.  The rank-side values h and g are sums, kept in fp32, and enter
// the next product as two pieces (2^-16 at most, far below the rounding of a 16-bit
// output) or three for fp32 outputs.  Of the products of pieces, those smaller
// than the last kept bit are dropped (pair()).  int8 codes are exact in bf16;
// their row scale multiplies h, or the rank side of dA, in fp32.
//
// Rows of other adapters, and rows without one, do not enter a product (their values are not loaded,
// their rank side is zero), and of a product only the adapter's own rows are stored, so NaN or
// infinity there stays there.  An infinity in a row or adapter in use gives an infinity or a NaN: pieces of one
// factor meet it with either sign.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "lora_rows.cuh"
#include "pieces.cuh"
#include "sm100_ptx.cuh"
#include "w8a8_internal.h"

namespace w8a8 {
namespace {

constexpr int kThreads = 256;
constexpr int kBK = 64;   // contraction per step of shrink
constexpr int kBN = 128;  // output columns per tile of expand and tokens
constexpr int kPad = 8;   // bf16 elements of padding a shared-memory row (conflict-free ldmatrix)

// pieces of a rank-side fp32 value next to data of type T
template <typename T>
struct RankPieces { static constexpr int n = std::is_same<T, float>::value ? 3 : 2; };

// ======================================================================== shrink
// part[split][row][r] = sum over the split's k of x[row, k] W_s[k, r], times the
// row's scale for int8 codes.  kRank = padded rank (16, 32, 64, 128).
// kWRows: W_s is stored [r][k] (A); otherwise [k][r] (B, k its N).
// 8 warps: four of 16 rows, times two that take every other 16 of a step's k.
template <typename TX, typename TW, int kRank, bool kWRows>
struct ShrinkTile {
  static constexpr int kPX = Pieces<TX>::n, kPW = Pieces<TW>::n;
  static constexpr int kMost = kPX > kPW ? kPX : kPW;
  static constexpr int kXPlane = kBM * (kBK + kPad);
  static constexpr int kLdW = kWRows ? kBK + kPad : kRank + kPad;
  static constexpr int kWPlane = (kWRows ? kRank : kBK) * kLdW;
  static constexpr int kBytes0 = 2 * (kPX * kXPlane + kPW * kWPlane);
  static constexpr int kJoin = kBM * kRank * 4;
  static constexpr int kBytes = kBytes0 > kJoin ? kBytes0 : kJoin;
};

template <typename TX, typename TW>
struct ShrinkArgs {
  const TX* x;
  int64_t ldx;
  const float* xs;
  const TW* w;
  int64_t slot;
  int K, k_split, vec_x, vec_w;
  float* part;
};
template <typename TX, typename TW, int kRank, bool kWRows>
__device__ __forceinline__ void shrink_tile(const ShrinkArgs<TX, TW>& g, const Rows& rows, int R, int split) {
  const TX* __restrict__ x = g.x;
  const TW* __restrict__ w = g.w;
  const float* __restrict__ xs = g.xs;
  float* __restrict__ part = g.part;
  const int64_t ldx = g.ldx, slot = g.slot;
  const int K = g.K, k_split = g.k_split, vec_x = g.vec_x, vec_w = g.vec_w;
  using Tile = ShrinkTile<TX, TW, kRank, kWRows>;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ TileIds ids;
  __nv_bfloat16* sx = reinterpret_cast<__nv_bfloat16*>(smem);
  __nv_bfloat16* sw = sx + Tile::kPX * Tile::kXPlane;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int wm = warp & 3, wk = warp >> 2;
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * kBM;
  const int k_lo = split * k_split;
  const int k_hi = min(K, k_lo + k_split);
  tile_ids(rows, row0, ids);

  constexpr bool kApart = std::is_same<TW, float>::value;
  constexpr int kGX = kBM * (kBK / 8) / kThreads;                       // 2
  constexpr int kGWAll = kRank * kBK / 8;                               // 8-element groups of W
  constexpr int kGW = (kGWAll + kThreads - 1) / kThreads;
  for (int li = blockIdx.z; li < ids.count; li += gridDim.z) {
    const int s = ids.list[li];
    const TW* ws = w + s * slot;
    float acc[kRank / 8][4];
#pragma unroll
    for (int i = 0; i < kRank / 8; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = 0.0f;
    float low[kApart ? kRank / 8 : 1][4] = {};

    Raw8<TX> rx[kGX];
    Raw8<TW> rw[kGW];
    auto fetch = [&](int k0) {
#pragma unroll
      for (int i = 0; i < kGX; ++i) {
        const int gi = tid + i * kThreads;
        const int r = gi / (kBK / 8), c = (gi % (kBK / 8)) * 8;
        const int valid = ids.id[r] == s ? min(8, k_hi - k0 - c) : 0;
        load8(rx[i], x + (row0 + r) * ldx + k0 + c, valid, vec_x != 0);
      }
#pragma unroll
      for (int i = 0; i < kGW; ++i) {
        const int gi = tid + i * kThreads;
        if (kGWAll % kThreads != 0 && gi >= kGWAll) break;
        if constexpr (kWRows) {
          const int r = gi / (kBK / 8), c = (gi % (kBK / 8)) * 8;
          const int valid = r < R ? min(8, k_hi - k0 - c) : 0;
          load8(rw[i], ws + static_cast<int64_t>(r) * K + k0 + c, valid, vec_w != 0);
        } else {
          const int r = gi / (kRank / 8), c = (gi % (kRank / 8)) * 8;
          const int valid = k0 + r < k_hi ? min(8, R - c) : 0;
          load8(rw[i], ws + static_cast<int64_t>(k0 + r) * R + c, valid, vec_w != 0);
        }
      }
    };
    fetch(k_lo);
    for (int k0 = k_lo; k0 < k_hi; k0 += kBK) {
      __syncthreads();  // the previous step's tiles are read
#pragma unroll
      for (int i = 0; i < kGX; ++i) {
        const int gi = tid + i * kThreads;
        store8(sx + (gi / (kBK / 8)) * (kBK + kPad) + (gi % (kBK / 8)) * 8, Tile::kXPlane, rx[i]);
      }
#pragma unroll
      for (int i = 0; i < kGW; ++i) {
        const int gi = tid + i * kThreads;
        if (kGWAll % kThreads != 0 && gi >= kGWAll) break;
        constexpr int kPer = kWRows ? kBK / 8 : kRank / 8;
        store8(sw + (gi / kPer) * Tile::kLdW + (gi % kPer) * 8, Tile::kWPlane, rw[i]);
      }
      __syncthreads();
      if (k0 + kBK < k_hi) fetch(k0 + kBK);
#pragma unroll
      for (int h = 0; h < kBK / 32; ++h) {
        const int kk = (2 * h + wk) * 16;
        uint32_t a[Tile::kPX][4];
#pragma unroll
        for (int p = 0; p < Tile::kPX; ++p)
          ldsm4(a[p], at16(sx + p * Tile::kXPlane, wm * 16, kk, kBK + kPad, lane));
#pragma unroll
        for (int n = 0; n < kRank / 16; ++n) {
#pragma unroll
          for (int pw = 0; pw < Tile::kPW; ++pw) {
            uint32_t b[4];
            if constexpr (kWRows) {
              ldsm4(b, at16h(sw + pw * Tile::kWPlane, n * 16, kk, Tile::kLdW, lane));
            } else {
              ldsm4_t(b, at16(sw + pw * Tile::kWPlane, kk, n * 16, Tile::kLdW, lane));
            }
#pragma unroll
            for (int px = 0; px < Tile::kPX; ++px) {
              if (pair(px, pw, Tile::kMost)) {
                if constexpr (kApart) {
                  mma_apart(acc[2 * n], low[2 * n], a[px], b[0], b[1], px + pw == 0);
                  mma_apart(acc[2 * n + 1], low[2 * n + 1], a[px], b[2], b[3], px + pw == 0);
                } else {
                  mma(acc[2 * n], a[px], b[0], b[1]);
                  mma(acc[2 * n + 1], a[px], b[2], b[3]);
                }
              }
            }
          }
        }
      }
    }
    if constexpr (kApart) {
#pragma unroll
      for (int i = 0; i < kRank / 8; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] += low[i][j];
    }
    // join the two halves of the warps through shared memory
    float* join = reinterpret_cast<float*>(smem);
    __syncthreads();
    const int r0 = wm * 16 + (lane >> 2), c0 = (lane & 3) * 2;
    if (wk == 1) {
#pragma unroll
      for (int n = 0; n < kRank / 8; ++n) {
        *reinterpret_cast<float2*>(join + r0 * kRank + n * 8 + c0) = make_float2(acc[n][0], acc[n][1]);
        *reinterpret_cast<float2*>(join + (r0 + 8) * kRank + n * 8 + c0) =
            make_float2(acc[n][2], acc[n][3]);
      }
    }
    __syncthreads();
    if (wk == 0) {
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int r = r0 + half * 8;
        if (ids.id[r] != s) continue;
        const int64_t row = row0 + r;
        const float sc = xs ? __ldg(xs + row) : 1.0f;
        float* dst = part + (static_cast<int64_t>(split) * rows.M + row) * R;
#pragma unroll
        for (int n = 0; n < kRank / 8; ++n) {
          const int c = n * 8 + c0;
          const float2 o = *reinterpret_cast<const float2*>(join + r * kRank + c);
          if (c < R) dst[c] = (acc[n][2 * half] + o.x) * sc;
          if (c + 1 < R) dst[c + 1] = (acc[n][2 * half + 1] + o.y) * sc;
        }
      }
    }
  }
}

template <typename TX, typename TW, int kRank, bool kWRows>
__global__ void __launch_bounds__(kThreads, kRank <= 64 ? 2 : 1) shrink_kernel(ShrinkArgs<TX, TW> g, Rows rows, int R) {
  griddep_launch_dependents();
  shrink_tile<TX, TW, kRank, kWRows>(g, rows, R, blockIdx.y);
}
// dy times B and x times A in one launch: blockIdx.y below `first` is the former.
template <typename TX, typename T, int kRank>
__global__ void __launch_bounds__(kThreads, kRank <= 64 ? 2 : 1) shrink_pair_kernel(
    ShrinkArgs<T, T> dy, ShrinkArgs<TX, T> x, int first, Rows rows, int R) {
  griddep_launch_dependents();
  if (static_cast<int>(blockIdx.y) < first) {
    shrink_tile<T, T, kRank, false>(dy, rows, R, blockIdx.y);
  } else {
    shrink_tile<TX, T, kRank, true>(x, rows, R, blockIdx.y - first);
  }
}

// Rank-side values of `rows_n` rows from row0 (those of adapter s; zero elsewhere):
// the splits' sums in a fixed order, times mul (and the row's scale), as bf16
// pieces into [row][kRank + kPad] planes.
template <int kRank, int kP>
__device__ __forceinline__ void load_rank_side(__nv_bfloat16* dst, const float* __restrict__ part,
                                               int splits, const Rows& rows, int64_t row0,
                                               const int* id, int s, int R, float mul,
                                               const float* __restrict__ row_mul) {
  constexpr int kLd = kRank + kPad;
  const int64_t plane = rows.M * R;
  for (int gi = threadIdx.x; gi < kBM * kRank / 8; gi += kThreads) {
    const int r = gi / (kRank / 8), c = (gi % (kRank / 8)) * 8;
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = 0.0f;
    if (id[r] == s) {
      const float* p = part + (row0 + r) * R + c;
      if (R % 4 == 0) {
        const bool has_lo = c < R, has_hi = c + 4 < R;
        // four splits' loads in flight (the latency of one after the other showed)
#pragma unroll 4
        for (int sp = 0; sp < splits; ++sp, p += plane) {
          const float4 lo = has_lo ? __ldcg(reinterpret_cast<const float4*>(p)) : make_float4(0, 0, 0, 0);
          const float4 hi = has_hi ? __ldcg(reinterpret_cast<const float4*>(p) + 1) : make_float4(0, 0, 0, 0);
          v[0] += lo.x; v[1] += lo.y; v[2] += lo.z; v[3] += lo.w;
          v[4] += hi.x; v[5] += hi.y; v[6] += hi.z; v[7] += hi.w;
        }
      } else {
        for (int sp = 0; sp < splits; ++sp, p += plane) {
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] += c + i < R ? __ldcg(p + i) : 0.0f;
        }
      }
      const float m = row_mul ? mul * __ldg(row_mul + row0 + r) : mul;
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] *= m;
    }
    store_pieces<kP>(dst + r * kLd + c, kBM * kLd, v);
  }
}

// ======================================================================== expand
// out[row, n] = T(y[row, n] + c[s] * sum_r h[row, r] W_s[r, n]); y NULL: zero.
// kWCols: W_s is stored [n][r] (B); otherwise [r][n] (A).
// A block keeps the rank side of 64 rows and goes through its range of columns,
// 128 at a time; the next tile's W_s and y are fetched into registers while this
// one is multiplied.  Bound by reading y and writing out.
template <typename T, int kRank, bool kWCols>
struct ExpandTile {
  static constexpr int kPH = RankPieces<T>::n, kPW = Pieces<T>::n;
  static constexpr int kMost = kPH > kPW ? kPH : kPW;
  static constexpr int kHPlane = kBM * (kRank + kPad);
  static constexpr int kLdW = kWCols ? kRank + kPad : kBN + kPad;
  static constexpr int kWPlane = (kWCols ? kBN : kRank) * kLdW;
  static constexpr int kLdO = kBN + 4;
  static constexpr int kOperands = 2 * (kPH * kHPlane + kPW * kWPlane);
  static constexpr int kBytes = kOperands + kBM * kLdO * 4;
};

template <typename T, int kRank, bool kWCols>
__global__ void __launch_bounds__(kThreads, sizeof(T) == 2 && kRank <= 64 ? 2 : 1) expand_kernel(
    const T* y, int64_t ldy, const float* __restrict__ part, int splits, const T* __restrict__ w,
    int64_t slot, const float* __restrict__ scaling, Rows rows, int N, int R, int col_parts,
    int cols_part, int vec_w, int vec_o, T* out, int64_t ldo) {
  using Tile = ExpandTile<T, kRank, kWCols>;
  constexpr bool kApart = std::is_same<T, float>::value;
  griddep_launch_dependents();
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ TileIds ids;
  __nv_bfloat16* sh = reinterpret_cast<__nv_bfloat16*>(smem);
  __nv_bfloat16* sw = sh + Tile::kPH * Tile::kHPlane;
  float* so = reinterpret_cast<float*>(smem + Tile::kOperands);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int wm = warp & 3, wn = warp >> 2;
  const int64_t row0 = static_cast<int64_t>(blockIdx.x / col_parts) * kBM;
  const int c_lo = static_cast<int>(blockIdx.x % col_parts) * cols_part;
  const int c_hi = min(N, c_lo + cols_part);
  tile_ids(rows, row0, ids);
  griddep_wait();

  // this thread's outputs of a tile: rows tid / 16 + 16 i, eight columns
  constexpr int kRowsT = kBM / 16;
  const int oc = (tid & 15) * 8;
  constexpr int kGWAll = kRank * kBN / 8;
  constexpr int kGW = (kGWAll + kThreads - 1) / kThreads;
  Raw8<T> y_next[kRowsT], w_next[kGW];
  auto fetch_y = [&](int col0) {
    if (!y) return;
#pragma unroll
    for (int i = 0; i < kRowsT; ++i) {
      const int64_t row = row0 + (tid >> 4) + 16 * i;
      load8(y_next[i], y + row * ldy + col0 + oc, row < rows.M ? min(8, c_hi - col0 - oc) : 0, vec_o != 0);
    }
  };
  auto put = [&](int64_t row, int col0, const Raw8<T>& o) {
    T* dst = out + row * ldo + col0 + oc;
    const int valid = c_hi - col0 - oc;
    if (vec_o && valid >= 8) {
#pragma unroll
      for (int q = 0; q < static_cast<int>(sizeof(T) / 2); ++q) {
        const uint2* sp = reinterpret_cast<const uint2*>(o.e) + 2 * q;
        reinterpret_cast<uint4*>(dst)[q] = make_uint4(sp[0].x, sp[0].y, sp[1].x, sp[1].y);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j < valid) dst[j] = o.e[j];
    }
  };
  // rows without an adapter: y as it is (zero without y)
  if (ids.none && blockIdx.z == 0 && y != out) {
    for (int col0 = c_lo; col0 < c_hi; col0 += kBN) {
      fetch_y(col0);
#pragma unroll
      for (int i = 0; i < kRowsT; ++i) {
        const int r = (tid >> 4) + 16 * i;
        if (!y) {
#pragma unroll
          for (int j = 0; j < 8; ++j) y_next[i].e[j] = T(0.0f);
        }
        if (ids.id[r] < 0 && row0 + r < rows.M) put(row0 + r, col0, y_next[i]);
      }
    }
  }
  for (int li = blockIdx.z; li < ids.count; li += gridDim.z) {
    const int s = ids.list[li];
    const T* ws = w + s * slot;
    const float mul = scaling ? __ldg(scaling + s) : 1.0f;
    auto fetch_w = [&](int col0) {
#pragma unroll
      for (int i = 0; i < kGW; ++i) {
        const int gi = tid + i * kThreads;
        if (kGWAll % kThreads != 0 && gi >= kGWAll) break;
        if constexpr (kWCols) {
          const int n = gi / (kRank / 8), c = (gi % (kRank / 8)) * 8;
          load8(w_next[i], ws + static_cast<int64_t>(col0 + n) * R + c, col0 + n < c_hi ? min(8, R - c) : 0,
                vec_w != 0);
        } else {
          const int r = gi / (kBN / 8), c = (gi % (kBN / 8)) * 8;
          load8(w_next[i], ws + static_cast<int64_t>(r) * N + col0 + c, r < R ? min(8, c_hi - col0 - c) : 0,
                vec_w != 0);
        }
      }
    };
    fetch_w(c_lo);
    fetch_y(c_lo);
    __syncthreads();  // the previous adapter's rank side is read
    load_rank_side<kRank, Tile::kPH>(sh, part, splits, rows, row0, ids.id, s, R, 1.0f, nullptr);
    for (int col0 = c_lo; col0 < c_hi; col0 += kBN) {
#pragma unroll
      for (int i = 0; i < kGW; ++i) {
        const int gi = tid + i * kThreads;
        if (kGWAll % kThreads != 0 && gi >= kGWAll) break;
        constexpr int kPer = kWCols ? kRank / 8 : kBN / 8;
        store8(sw + (gi / kPer) * Tile::kLdW + (gi % kPer) * 8, Tile::kWPlane, w_next[i]);
      }
      Raw8<T> y_now[kRowsT];
#pragma unroll
      for (int i = 0; i < kRowsT; ++i) y_now[i] = y_next[i];
      __syncthreads();
      if (col0 + kBN < c_hi) {
        fetch_w(col0 + kBN);
        fetch_y(col0 + kBN);
      }
      float acc[8][4];
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = 0.0f;
      float low[kApart ? 8 : 1][4] = {};
#pragma unroll
      for (int kk = 0; kk < kRank; kk += 16) {
        uint32_t a[Tile::kPH][4];
#pragma unroll
        for (int p = 0; p < Tile::kPH; ++p)
          ldsm4(a[p], at16(sh + p * Tile::kHPlane, wm * 16, kk, kRank + kPad, lane));
#pragma unroll
        for (int n = 0; n < 4; ++n) {
#pragma unroll
          for (int pw = 0; pw < Tile::kPW; ++pw) {
            uint32_t b[4];
            if constexpr (kWCols) {
              ldsm4(b, at16h(sw + pw * Tile::kWPlane, wn * 64 + n * 16, kk, Tile::kLdW, lane));
            } else {
              ldsm4_t(b, at16(sw + pw * Tile::kWPlane, kk, wn * 64 + n * 16, Tile::kLdW, lane));
            }
#pragma unroll
            for (int ph = 0; ph < Tile::kPH; ++ph) {
              if (pair(ph, pw, Tile::kMost)) {
                if constexpr (kApart) {
                  mma_apart(acc[2 * n], low[2 * n], a[ph], b[0], b[1], ph + pw == 0);
                  mma_apart(acc[2 * n + 1], low[2 * n + 1], a[ph], b[2], b[3], ph + pw == 0);
                } else {
                  mma(acc[2 * n], a[ph], b[0], b[1]);
                  mma(acc[2 * n + 1], a[ph], b[2], b[3]);
                }
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
      const int r0 = wm * 16 + (lane >> 2), c0 = wn * 64 + (lane & 3) * 2;
#pragma unroll
      for (int n = 0; n < 8; ++n) {
        *reinterpret_cast<float2*>(so + r0 * Tile::kLdO + c0 + n * 8) = make_float2(acc[n][0], acc[n][1]);
        *reinterpret_cast<float2*>(so + (r0 + 8) * Tile::kLdO + c0 + n * 8) =
            make_float2(acc[n][2], acc[n][3]);
      }
      __syncthreads();  // the products are staged, and W_s is read
#pragma unroll
      for (int i = 0; i < kRowsT; ++i) {
        const int r = (tid >> 4) + 16 * i;
        if (ids.id[r] != s) continue;
        const float* add = so + r * Tile::kLdO + oc;
        Raw8<T> o;
#pragma unroll
        for (int j = 0; j < 8; ++j)
          o.e[j] = from_f<T>(y ? fmaf(mul, add[j], to_f(y_now[i].e[j])) : mul * add[j]);
        put(row0 + r, col0, o);
      }
    }
  }
}

// ======================================================================== few rows
// Decode steps: each row with an adapter of its own, so a tile would hold one row.
// CUDA cores, a block for each (rank, row) and then for each (256 columns, row);
// what has to be read is the adapters' weights, once, and latency counts.  The
// second kernel starts while the first runs (programmatic dependent launch): its
// weights and y are on their way when h arrives.
// 64 rows, 32 adapters of rank 32, 4096 -> 12288: 9 and 13 us.  Which calls: few_rows below.
template <typename T>
__global__ void __launch_bounds__(kThreads) shrink_row_kernel(const T* __restrict__ x, int64_t ldx,
                                                              const T* __restrict__ a, int64_t slot,
                                                              Rows rows, int K, int R, int vec,
                                                              float* __restrict__ h) {
  griddep_launch_dependents();
  __shared__ float sums[kThreads / 32];
  const int r = blockIdx.x;
  const int64_t row = blockIdx.y;
  const int s = adapter_of(rows, row);
  if (s < 0) return;
  const T* xr = x + row * ldx;
  const T* ar = a + s * slot + static_cast<int64_t>(r) * K;
  float v = 0.0f;
#pragma unroll 4
  for (int k = threadIdx.x * 8; k < K; k += kThreads * 8) {
    Raw8<T> p, q;
    load8(p, xr + k, K - k, vec != 0);
    load8(q, ar + k, K - k, vec != 0);
#pragma unroll
    for (int i = 0; i < 8; ++i) v = fmaf(to_f(p.e[i]), to_f(q.e[i]), v);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) sums[threadIdx.x >> 5] = v;
  __syncthreads();
  if (threadIdx.x == 0) {
    float t = 0.0f;
#pragma unroll
    for (int i = 0; i < kThreads / 32; ++i) t += sums[i];
    h[row * R + r] = t;
  }
}

// kVec: rows of B of whole eight-element vectors.
template <typename T, bool kVec>
__global__ void __launch_bounds__(kThreads) expand_row_kernel(const T* y, int64_t ldy, const float* h,
                                                              const T* __restrict__ b, int64_t slot,
                                                              const float* __restrict__ scaling,
                                                              Rows rows, int N, int R, T* out,
                                                              int64_t ldo) {
  __shared__ float sh[128];
  const int n = blockIdx.x * kThreads + threadIdx.x;
  const int64_t row = blockIdx.y;
  const int s = adapter_of(rows, row);
  const float base = n < N ? to_f(y[row * ldy + n]) : 0.0f;
  const T* br = b + (s < 0 ? 0 : s * slot) + static_cast<int64_t>(n) * R;
  constexpr int kAhead = 4;  // vectors of B fetched before h is there
  Raw8<T> w[kAhead];
  if (kVec && s >= 0 && n < N) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
      if (i * 8 < R) load8(w[i], br + i * 8, 8, true);
  }
  const float mul = s >= 0 && scaling ? __ldg(scaling + s) : 1.0f;
  griddep_wait();
  if (s >= 0 && threadIdx.x < R) sh[threadIdx.x] = __ldcg(h + row * R + threadIdx.x);
  __syncthreads();
  if (n >= N) return;
  T* dst = out + row * ldo + n;
  if (s < 0) {
    if (y != out) *dst = y[row * ldy + n];
    return;
  }
  float v = 0.0f;
  if constexpr (kVec) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      if (i * 8 < R) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v = fmaf(sh[i * 8 + j], to_f(w[i].e[j]), v);
      }
    }
    for (int c = kAhead * 8; c < R; c += 8) {
      Raw8<T> q;
      load8(q, br + c, 8, true);
#pragma unroll
      for (int j = 0; j < 8; ++j) v = fmaf(sh[c + j], to_f(q.e[j]), v);
    }
  } else {
    for (int c = 0; c < R; ++c) v = fmaf(sh[c], to_f(br[c]), v);
  }
  *dst = from_f<T>(fmaf(mul, v, base));
}

// ======================================================================== tokens
// part[split][s][r][c] (kByCol: [split][s][c][r]) = sum over the split's rows m
// of adapter s of q[m, r] X[m, c], with q = mul[s] * (row_mul[m]) * the rank side.
// 128 columns a block, all of the rank; warp w takes columns 16 w .. 16 w + 15.
// found[split][s] says whether the block wrote anything.
template <typename TX, typename TO, int kRank, bool kByCol>
struct TokensTile {
  static constexpr int kPX = Pieces<TX>::n, kPH = RankPieces<TO>::n;
  static constexpr int kMost = kPX > kPH ? kPX : kPH;
  static constexpr int kXPlane = kBM * (kBN + kPad);
  static constexpr int kHPlane = kBM * (kRank + kPad);
  static constexpr int kBytes = 2 * (kPX * kXPlane + kPH * kHPlane);
};

template <typename TX>
struct TokensArgs {
  const TX* x;
  int64_t ldx;
  const float* row_mul;
  const float* rank_part;
  int splits;           // of the rank side
  int C;
  int64_t rows_split;
  int count;            // splits of the rows
  int chunks;           // of 128 columns
  int vec_x;
  float* part;
  int* found;
};
template <typename TX, typename TO, int kRank, bool kByCol>
__device__ __forceinline__ void tokens_tile(const TokensArgs<TX>& g, const float* __restrict__ scaling,
                                            const Rows& rows, int R, int chunk, int split) {
  const TX* __restrict__ x = g.x;
  const float* __restrict__ row_mul = g.row_mul;
  const float* __restrict__ rank_part = g.rank_part;
  float* __restrict__ part = g.part;
  int* __restrict__ found = g.found;
  const int64_t ldx = g.ldx, rows_split = g.rows_split;
  const int splits = g.splits, C = g.C, vec_x = g.vec_x;
  using Tile = TokensTile<TX, TO, kRank, kByCol>;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ int id[kBM];
  __nv_bfloat16* sx = reinterpret_cast<__nv_bfloat16*>(smem);
  __nv_bfloat16* sh = sx + Tile::kPX * Tile::kXPlane;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int col0 = chunk * kBN;
  const int s = blockIdx.z;
  const int64_t m_lo = static_cast<int64_t>(split) * rows_split;
  const int64_t m_hi = min(rows.M, m_lo + rows_split);
  const float mul = scaling ? __ldg(scaling + s) : 1.0f;
  float acc[kRank / 16][2][4];
#pragma unroll
  for (int i = 0; i < kRank / 16; ++i)
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][n][j] = 0.0f;
  constexpr bool kApart = std::is_same<TO, float>::value;
  float low[kApart ? kRank / 16 : 1][2][4] = {};
  bool any = false;
  constexpr int kGX = kBM * (kBN / 8) / kThreads;  // 4
  for (int64_t m0 = m_lo; m0 < m_hi; m0 += kBM) {
    int mine = 0;
    if (tid < kBM) {
      const int v = m0 + tid < m_hi ? adapter_of(rows, m0 + tid) : -1;
      id[tid] = v;
      mine = v == s;
    }
    if (!__syncthreads_or(mine)) continue;
    any = true;
    Raw8<TX> rx[kGX];
#pragma unroll
    for (int i = 0; i < kGX; ++i) {
      const int gi = tid + i * kThreads;
      const int r = gi / (kBN / 8), c = (gi % (kBN / 8)) * 8;
      const int valid = id[r] == s ? min(8, C - col0 - c) : 0;
      load8(rx[i], x + (m0 + r) * ldx + col0 + c, valid, vec_x != 0);
    }
    load_rank_side<kRank, Tile::kPH>(sh, rank_part, splits, rows, m0, id, s, R, mul, row_mul);
#pragma unroll
    for (int i = 0; i < kGX; ++i) {
      const int gi = tid + i * kThreads;
      store8(sx + (gi / (kBN / 8)) * (kBN + kPad) + (gi % (kBN / 8)) * 8, Tile::kXPlane, rx[i]);
    }
    __syncthreads();
#pragma unroll
    for (int kk = 0; kk < kBM; kk += 16) {
      uint32_t b[Tile::kPX][4];
#pragma unroll
      for (int p = 0; p < Tile::kPX; ++p)
        ldsm4_t(b[p], at16(sx + p * Tile::kXPlane, kk, warp * 16, kBN + kPad, lane));
#pragma unroll
      for (int i = 0; i < kRank / 16; ++i) {
#pragma unroll
        for (int ph = 0; ph < Tile::kPH; ++ph) {
          uint32_t a[4];
          ldsm4_t(a, at16h(sh + ph * Tile::kHPlane, kk, i * 16, kRank + kPad, lane));
#pragma unroll
          for (int px = 0; px < Tile::kPX; ++px) {
            if (pair(px, ph, Tile::kMost)) {
              if constexpr (kApart) {
                mma_apart(acc[i][0], low[i][0], a, b[px][0], b[px][1], px + ph == 0);
                mma_apart(acc[i][1], low[i][1], a, b[px][2], b[px][3], px + ph == 0);
              } else {
                mma(acc[i][0], a, b[px][0], b[px][1]);
                mma(acc[i][1], a, b[px][2], b[px][3]);
              }
            }
          }
        }
      }
    }
    __syncthreads();  // tiles and ids are read
  }
  if constexpr (kApart) {
#pragma unroll
    for (int i = 0; i < kRank / 16; ++i)
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][n][j] += low[i][n][j];
  }
  const int64_t block = static_cast<int64_t>(split) * rows.S + s;
  if (chunk == 0 && tid == 0) found[block] = any;
  if (!any) return;
  float* dst = part + block * R * C;
#pragma unroll
  for (int i = 0; i < kRank / 16; ++i)
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int r = i * 16 + (lane >> 2) + (j >> 1) * 8;
        const int c = col0 + warp * 16 + n * 8 + (lane & 3) * 2 + (j & 1);
        if (r < R && c < C) {
          dst[kByCol ? static_cast<int64_t>(c) * R + r : static_cast<int64_t>(r) * C + c] = acc[i][n][j];
        }
      }
}

// Both gradients in one launch: blocks below a.chunks * a.count are dA's.
template <typename TX, typename T, int kRank>
__global__ void __launch_bounds__(kThreads, kRank <= 64 ? 2 : 1) tokens_pair_kernel(TokensArgs<TX> a, TokensArgs<T> b,
                                                               const float* __restrict__ scaling, Rows rows, int R) {
  griddep_launch_dependents();
  griddep_wait();
  const int first = a.chunks * a.count;
  const int i = static_cast<int>(blockIdx.x);
  if (i < first) {
    tokens_tile<TX, T, kRank, false>(a, scaling, rows, R, i % a.chunks, i / a.chunks);
  } else {
    tokens_tile<T, T, kRank, true>(b, scaling, rows, R, (i - first) % b.chunks, (i - first) / b.chunks);
  }
}

// The splits' sums, in a fixed order, rounded to T: dA (blockIdx.z 0) or dB of
// adapter blockIdx.y, four elements a thread where the adapter's size allows it.
struct SumArgs {
  const float* part;
  const int* found;
  int splits;
  int64_t per;  // elements of one adapter
  void* out;
};
constexpr int kSplitsMost = 1024;  // of the rows of a batch (tokens_split, tokens_tc_split)
template <typename T>
__global__ void __launch_bounds__(kThreads) sum_splits_kernel(SumArgs ga, SumArgs gb, int S) {
  griddep_wait();
  const SumArgs g = blockIdx.z ? gb : ga;
  const int s = blockIdx.y;
  const int64_t plane = g.per * S;
  const float* p0 = g.part + s * g.per;
  T* out = static_cast<T*>(g.out) + s * g.per;
  // the splits that have rows of the adapter, in order
  __shared__ uint16_t list[kSplitsMost];
  __shared__ int count;
  if (threadIdx.x < 32) {
    int n = 0;
    for (int base = 0; base < g.splits; base += 32) {
      const int sp = base + static_cast<int>(threadIdx.x);
      const bool there = sp < g.splits && __ldcg(g.found + sp * S + s);
      const unsigned m = __ballot_sync(0xffffffffu, there);
      if (there) list[n + __popc(m & ((1u << threadIdx.x) - 1u))] = static_cast<uint16_t>(sp);
      n += __popc(m);
    }
    if (threadIdx.x == 0) count = n;
  }
  __syncthreads();
  const int n = count;
  const int64_t start = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kThreads;
  if (g.per % 4 == 0 && reinterpret_cast<uintptr_t>(g.out) % (4 * sizeof(T)) == 0) {
    for (int64_t i = start * 4; i < g.per; i += step * 4) {
      float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
      for (int j = 0; j < n; ++j) {
        const float4 o = __ldcg(reinterpret_cast<const float4*>(p0 + list[j] * plane + i));
        v.x += o.x;
        v.y += o.y;
        v.z += o.z;
        v.w += o.w;
      }
      const T o[4] = {from_f<T>(v.x), from_f<T>(v.y), from_f<T>(v.z), from_f<T>(v.w)};
      if constexpr (sizeof(T) == 2) {
        *reinterpret_cast<uint2*>(out + i) = *reinterpret_cast<const uint2*>(o);
      } else {
        *reinterpret_cast<uint4*>(out + i) = *reinterpret_cast<const uint4*>(o);
      }
    }
    return;
  }
  for (int64_t i = start; i < g.per; i += step) {
    float v = 0.0f;
    for (int j = 0; j < n; ++j) v += __ldcg(p0 + list[j] * plane + i);
    out[i] = from_f<T>(v);
  }
}

// ---------------------------------------------------------------- host
int pad_rank(int R) { return R <= 16 ? 16 : R <= 32 ? 32 : R <= 64 ? 64 : 128; }

bool aligned(const void* p, int64_t ld, int size) {
  // rows of eight-element groups that vector loads may take (16 bytes; 8 for int8)
  const int64_t unit = size == 1 ? 8 : 16;
  return reinterpret_cast<uintptr_t>(p) % unit == 0 && (ld * size) % unit == 0;
}

template <typename K>
int prepare(K kernel, int bytes) {
  if (bytes > 40 * 1024) {  // 48 KiB without opting in, the static part included
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) {
      set_error("lora: shared memory of %d bytes refused: %s", bytes, cudaGetErrorString(e));
      return W8A8_ERR_ACCELERATOR;
    }
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

// How a shrink is cut: enough blocks for two a multiprocessor, at least two
// steps of the contraction each, and at most 16 pieces (the next kernel adds
// them up for every tile it makes).
struct Split {
  int count;
  int per;
};
Split shrink_split(int64_t M, int K) {
  const int64_t tiles = (M + kBM - 1) / kBM;
  const int steps = std::max(1, (K + kBK - 1) / kBK);
  int64_t want = (2 * device_sm_count() + tiles - 1) / std::max<int64_t>(tiles, 1);
  want = std::max<int64_t>(1, std::min<int64_t>({want, 16, (steps + 1) / 2}));
  const int per = static_cast<int>((steps + want - 1) / want);
  return {(steps + per - 1) / per, per * kBK};
}
// The same for two shrinks in one launch, which share twice the blocks in proportion to
// their steps (fp32, 641 rows, 7680 and 1152 at rank 64: 68 us with as many blocks for
// each, 44 so, with two blocks a multiprocessor).
void shrink_pair_split(int64_t M, int N, int K, Split& n, Split& k) {
  const int64_t tiles = std::max<int64_t>(1, (M + kBM - 1) / kBM);
  const int64_t steps_n = std::max(1, (N + kBK - 1) / kBK), steps_k = std::max(1, (K + kBK - 1) / kBK);
  const int64_t want = std::max<int64_t>(2, 4 * device_sm_count() / tiles);
  const int64_t per = std::max<int64_t>({2, (steps_n + steps_k + want - 1) / want, (std::max(steps_n, steps_k) + 15) / 16});
  n = {static_cast<int>((steps_n + per - 1) / per), static_cast<int>(per * kBK)};
  k = {static_cast<int>((steps_k + per - 1) / per), static_cast<int>(per * kBK)};
}
// Blocks that share out a tile's adapters (a tile of a decode batch has many).
int parts_of(int64_t M, int S, int blocks) {
  if (S <= 1) return 1;
  const int64_t tiles = (M + kBM - 1) / kBM;
  const int64_t most = std::min<int64_t>({S, M, kBM});
  const int64_t want = (2 * device_sm_count()) / std::max<int64_t>(1, tiles * blocks);
  return static_cast<int>(std::max<int64_t>(1, std::min(want, most)));
}
// How the rows of a token contraction are cut: two blocks a multiprocessor for
// one adapter's columns, whole tiles, and at most 64 MiB of partial sums.
struct RowSplit {
  int count;
  int64_t per;
};
RowSplit tokens_split(int64_t M, int C, int S, int R) {
  const int64_t tiles = std::max<int64_t>(1, (M + kBM - 1) / kBM);
  const int64_t chunks = (C + kBN - 1) / kBN;
  int64_t want = (2 * device_sm_count() + chunks - 1) / std::max<int64_t>(chunks, 1);
  const int64_t one = static_cast<int64_t>(S) * R * C * 4;
  want = std::max<int64_t>(1, std::min<int64_t>({want, tiles, (64ll << 20) / std::max<int64_t>(one, 1)}));
  const int64_t per = (tiles + want - 1) / want;
  return {static_cast<int>((tiles + per - 1) / per), per * kBM};
}

int64_t up(int64_t v) { return (v + 255) / 256 * 256; }

// ---- the tcgen05 form (lora_sm100.cu): long bf16 batches of a few adapters whose
// operands TMA can take (16-byte rows).
constexpr int64_t kTcRows = 256;
constexpr int64_t kTcAdapters = 64;
// Whether a call is work enough for it, M (N + K) elements of the batch.  It reads them at a
// higher rate but has more kernels (a gradient seven against four) and longer prologues, and the
// mma.sync form goes through a tile's adapters one after another.  Captured calls, memory
// cold, rank 16 and 64, us (tcgen05 / mma.sync):
//   gradients  one adapter     256 x 768 -> 256 (0.3 Mi) 35 / 18, 45 / 25;  3000 x 512 -> 512 (2.9 Mi) 45 / 33, 57 / 47;
//                              1000 x 2048 -> 2048 (3.9 Mi) 41 / 35, 57 / 59;  700 x 4096 -> 4096 (5.5 Mi) 43 / 47, 66 / 80;
//                              6000 x 4096 -> 4096 (47 Mi) 84 / 160, 104 / 244
//              32, mixed rows  256 x 4096 -> 4096 (2.0 Mi) 291 / 254, 538 / 504;  1500 x 1024 -> 1024 (2.9 Mi) 313 / 393, 584 / 642
//   forward    one adapter     6000 x 256 -> 256 (2.9 Mi) 21 / 14, 25 / 18;  2000 x 2048 -> 2048 (7.8 Mi) 25 / 23, 33 / 33;
//                              2000 x 4096 -> 4096 (16 Mi) 29 / 33, 43 / 47
//              32, mixed rows  256 x 1024 -> 1024 (0.5 Mi) 41 / 31, 45 / 43;  256 x 4096 -> 4096 (2.0 Mi) 47 / 101, 55 / 162
bool tc_work(int64_t M, int64_t N, int64_t K, int64_t S, bool backward) {
  if (M < kTcRows || S > kTcAdapters) return false;
  const int64_t mi = S <= 8 ? (backward ? 5 : 8) : (backward ? 3 : 2);
  return M * (N + K) >= mi << 20;
}
bool tc_shape(const LoraArgs& g, bool backward) {
  return g.dtype == W8A8_BF16 && g.M <= (1ll << 27) && g.K % 8 == 0 && g.N % 8 == 0 && g.R % 8 == 0 && g.K > 0 &&
         g.N > 0 && tc_work(g.M, g.N, g.K, g.S, backward);
}
bool tc_rows(const void* p, int64_t ld, int size) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && (ld * size) % 16 == 0;
}
bool tc_x(const LoraArgs& g) { return tc_rows(g.x, g.ldx, g.x_scale ? 1 : 2); }
bool tc_weights(const void* p, int64_t slot, int64_t width, int64_t S) {
  return tc_rows(p, width, 2) && (S == 1 || (slot * 2) % 16 == 0);
}
// Two blocks a multiprocessor, at least four steps each.
Split shrink_tc_split(int64_t M, int K) {
  const int64_t tiles = std::max<int64_t>(1, (M + 127) / 128);
  const int steps = std::max(1, (K + 63) / 64);
  const int64_t want =
      std::max<int64_t>(1, std::min<int64_t>({2ll * device_sm_count() / tiles, 16, (steps + 3) / 4}));
  const int per = static_cast<int>((steps + want - 1) / want);
  return {(steps + per - 1) / per, per * 64};
}
// One block a multiprocessor for 256 columns each, at most 256 MiB of partial sums;
// a block lists at most 2048 tiles.
RowSplit tokens_tc_split(int64_t M, int C, int S, int R) {
  const int64_t tiles = std::max<int64_t>(1, (M + kBM - 1) / kBM);
  const int64_t chunks = std::max<int64_t>(1, (C + 255) / 256);
  const int64_t one = std::max<int64_t>(1, static_cast<int64_t>(S) * R * C * 4);
  int64_t want = std::max<int64_t>(1, std::min<int64_t>({device_sm_count() / chunks, tiles, (256ll << 20) / one}));
  want = std::max(want, (tiles + 2047) / 2048);
  const int64_t per = (tiles + want - 1) / want;
  return {static_cast<int>((tiles + per - 1) / per), per * kBM};
}
int shrink_tc(const LoraArgs& g, const void* x, int64_t ldx, bool codes, const float* x_scale, const void* w,
              int64_t slot, bool w_rows, int64_t K, const Split& sp, float* part, int* counts, bool first, cudaStream_t stream) {
  const int64_t blocks = (g.M + 127) / 128 * sp.count;
  const int64_t parts = std::max<int64_t>(1, std::min<int64_t>(g.S, 2ll * device_sm_count() / blocks));
  return lora_shrink_tc({x, codes, ldx, x_scale, w, w_rows, slot, g.M, K, g.S, g.R, sp.count, sp.per / 64,
                         static_cast<int>(parts), part, counts, first},
                        {g.adapter, g.adapter64, g.rows_per_index, g.M, g.S}, stream);
}

template <typename TX, typename TW, bool kWRows>
ShrinkArgs<TX, TW> shrink_args(const TX* x, int64_t ldx, const float* xs, const TW* w, int64_t slot, int K, int R,
                               const Split& sp, float* part) {
  const int vx = aligned(x, ldx, sizeof(TX));
  const int vw = aligned(w, kWRows ? K : R, sizeof(TW)) && aligned(w, slot, sizeof(TW));
  return {x, ldx, xs, w, slot, K, sp.per, vx, vw, part};
}

#define BY_RANK(F)                 \
  switch (pad_rank(R)) {           \
    case 16: F(16) break;          \
    case 32: F(32) break;          \
    case 64: F(64) break;          \
    default: F(128) break;         \
  }

template <typename T>
int shrink(const ShrinkArgs<T, T>& g, bool w_rows, int splits, const Rows& rows, int R, cudaStream_t stream) {
  const int64_t tiles = (rows.M + kBM - 1) / kBM;
  const dim3 grid(static_cast<unsigned>(tiles), splits, parts_of(rows.M, rows.S, splits));
#define SHRINK(RANK)                                                       \
  {                                                                        \
    auto k = w_rows ? shrink_kernel<T, T, RANK, true> : shrink_kernel<T, T, RANK, false>; \
    const int bytes = w_rows ? ShrinkTile<T, T, RANK, true>::kBytes : ShrinkTile<T, T, RANK, false>::kBytes; \
    if (int rc = prepare(k, bytes)) return rc;                             \
    k<<<grid, kThreads, bytes, stream>>>(g, rows, R);                      \
  }
  BY_RANK(SHRINK)
#undef SHRINK
  return launched("lora shrink");
}

template <typename TX, typename T>
int shrink_pair(const ShrinkArgs<T, T>& dy, int splits_dy, const ShrinkArgs<TX, T>& x, int splits_x, const Rows& rows,
                int R, cudaStream_t stream) {
  const int64_t tiles = (rows.M + kBM - 1) / kBM;
  const int splits = splits_dy + splits_x;
  const dim3 grid(static_cast<unsigned>(tiles), splits, parts_of(rows.M, rows.S, splits));
#define SHRINK(RANK)                                                       \
  {                                                                        \
    auto k = shrink_pair_kernel<TX, T, RANK>;                              \
    constexpr int bytes = std::max(ShrinkTile<T, T, RANK, false>::kBytes, ShrinkTile<TX, T, RANK, true>::kBytes); \
    if (int rc = prepare(k, bytes)) return rc;                             \
    k<<<grid, kThreads, bytes, stream>>>(dy, x, splits_dy, rows, R);       \
  }
  BY_RANK(SHRINK)
#undef SHRINK
  return launched("lora shrink");
}

template <typename T, bool kWCols>
int expand(const T* y, int64_t ldy, const float* part, int splits, const T* w, int64_t slot,
           const float* scaling, const Rows& rows, int N, int R, T* out, int64_t ldo,
           cudaStream_t stream) {
  const int64_t tiles = (rows.M + kBM - 1) / kBM;
  const int col_tiles = (N + kBN - 1) / kBN;
  const int vw = aligned(w, kWCols ? R : N, sizeof(T)) && aligned(w, slot, sizeof(T));
  const int vo = aligned(out, ldo, sizeof(T)) && (!y || aligned(y, ldy, sizeof(T)));
  // Ranges of columns: six blocks a multiprocessor (three at a time), so that a
  // block has several tiles to overlap and the last wave is short.
  int parts = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(col_tiles, 6ll * device_sm_count() / tiles)));
  const int per = (col_tiles + parts - 1) / parts;
  parts = (col_tiles + per - 1) / per;
  const dim3 grid(static_cast<unsigned>(tiles * parts), 1, parts_of(rows.M, rows.S, parts));
  cudaError_t e = cudaSuccess;
#define EXPAND(RANK)                                                                              \
  {                                                                                               \
    auto k = expand_kernel<T, RANK, kWCols>;                                                      \
    constexpr int bytes = ExpandTile<T, RANK, kWCols>::kBytes;                                    \
    if (int rc = prepare(k, bytes)) return rc;                                                    \
    e = launch_chained(true, k, grid, kThreads, bytes, stream, y, ldy, part, splits, w, slot, scaling, rows, N, R, parts, \
                                         per * kBN, vw, vo, out, ldo);                            \
  }
  switch (pad_rank(R)) {
    case 16: EXPAND(16) break;
    case 32: EXPAND(32) break;
    case 64: EXPAND(64) break;
    default: EXPAND(128) break;
  }
#undef EXPAND
  return chained("lora expand", e);
}

template <typename TX, typename T>
int tokens_pair(const TokensArgs<TX>& a, const TokensArgs<T>& b, const float* scaling, const Rows& rows, int R,
                cudaStream_t stream) {
  const dim3 grid(a.chunks * a.count + b.chunks * b.count, 1, rows.S);
  cudaError_t e = cudaSuccess;
#define TOKENS(RANK)                                                       \
  {                                                                        \
    auto k = tokens_pair_kernel<TX, T, RANK>;                              \
    constexpr int bytes = std::max(TokensTile<TX, T, RANK, false>::kBytes, TokensTile<T, T, RANK, true>::kBytes); \
    if (int rc = prepare(k, bytes)) return rc;                             \
    e = launch_chained(true, k, grid, kThreads, bytes, stream, a, b, scaling, rows, R); \
  }
  BY_RANK(TOKENS)
#undef TOKENS
  return chained("lora tokens", e);
}

// Whether up to one tile of rows goes row by row: each reads its adapter again, M R (K + N) elements
// of weights through L2, where a tile reads an adapter once but goes through its adapters, of which
// it has min(S, M) at most, one after another.  Captured calls, memory cold, 4096 -> 12288
// in bf16, us (rows / tiles):
//   one adapter   16 rows  rank 16 10 / 14, rank 64 20 / 16;  64 rows  rank 16 18 / 16, rank 32 23 / 16, rank 128 86 / 29
//   four          16 rows  rank 64 21 / 23, rank 128 31 / 33;  64 rows  rank 16 18 / 21, rank 64 49 / 27
//   thirty-two    64 rows  rank 16 18 / 55, rank 32 27 / 64, rank 128 92 / 203
// f16 and fp32 tiles multiply pieces and pay later, 4096 -> 4096, one adapter: 32 rows of rank 128
// 31 / 33 (fp32 37 / 55), 64 rows of rank 64 27 / 27 (37 / 37), of rank 128 46 / 39 (66 / 62).
bool few_rows(const LoraArgs& g) {
  if (g.M > kBM) return false;
  const int64_t adapters = std::min(g.S, g.M);
  return g.M * g.R <= (g.dtype == W8A8_BF16 ? 256 * (adapters + 3) : 512 * (adapters + 8));
}

template <typename T>
int add_few_rows(const LoraArgs& g, const Rows& rows, float* h, cudaStream_t stream) {
  const int K = static_cast<int>(g.K), N = static_cast<int>(g.N), R = static_cast<int>(g.R);
  const T* x = static_cast<const T*>(g.x);
  const T* a = static_cast<const T*>(g.a);
  const T* b = static_cast<const T*>(g.b);
  const T* y = static_cast<const T*>(g.y);
  const int vec = aligned(x, g.ldx, sizeof(T)) && aligned(a, K, sizeof(T)) && aligned(a, g.lda, sizeof(T));
  const unsigned m = static_cast<unsigned>(g.M);
  shrink_row_kernel<T><<<dim3(R, m), kThreads, 0, stream>>>(x, g.ldx, a, g.lda, rows, K, R, vec, h);
  if (int rc = launched("lora shrink")) return rc;
  const bool whole = R % 8 == 0 && aligned(b, R, sizeof(T)) && aligned(b, g.ldb, sizeof(T));
  return chained("lora expand",
                 launch_chained(true, whole ? expand_row_kernel<T, true> : expand_row_kernel<T, false>,
                                dim3((N + kThreads - 1) / kThreads, m), kThreads, 0, stream, y, g.ldy,
                                static_cast<const float*>(h), b, g.ldb, g.scaling, rows, N, R,
                                static_cast<T*>(g.out), g.ldo));
}

template <typename T>
int add_typed(const LoraArgs& g, cudaStream_t stream) {
  const Rows rows{g.adapter, g.adapter64, g.rows_per_index, g.M, static_cast<int>(g.S)};
  const int K = static_cast<int>(g.K), N = static_cast<int>(g.N), R = static_cast<int>(g.R);
  float* part = static_cast<float*>(g.workspace);
  if (few_rows(g)) return add_few_rows<T>(g, rows, part, stream);
  Split sp = shrink_split(g.M, K);
  int* counts = nullptr;
  if (tc_shape(g, false) && tc_x(g) && tc_weights(g.a, g.lda, K, g.S)) {
    sp = shrink_tc_split(g.M, K);
    counts = reinterpret_cast<int*>(part + sp.count * g.M * g.R);
    if (int rc = shrink_tc(g, g.x, g.ldx, false, nullptr, g.a, g.lda, true, K, sp, part, counts, true, stream)) return rc;
  } else if (int rc = shrink<T>(shrink_args<T, T, true>(static_cast<const T*>(g.x), g.ldx, nullptr,
                                                        static_cast<const T*>(g.a), g.lda, K, R, sp, part),
                                true, sp.count, rows, R, stream)) {
    return rc;
  }
  if (counts && tc_rows(g.y, g.ldy, 2) && tc_rows(g.out, g.ldo, 2) && tc_weights(g.b, g.ldb, R, g.S)) {
    return lora_expand_tc({g.y, g.ldy, counts, part, sp.count, g.b, 1, g.ldb, g.scaling, g.out, g.ldo, g.M, g.N, g.S, g.R},
                          {g.adapter, g.adapter64, g.rows_per_index, g.M, g.S}, stream);
  }
  return expand<T, true>(static_cast<const T*>(g.y), g.ldy, part, sp.count,
                         static_cast<const T*>(g.b), g.ldb, g.scaling, rows, N, R,
                         static_cast<T*>(g.out), g.ldo, stream);
}

struct BackwardPlan {
  Split h, g;
  RowSplit a, b;
  int64_t off_g, off_counts, off_a, off_b, off_found, off_pa, off_pb, off_info, bytes;  // dx alone: up to off_a
};
BackwardPlan backward_plan(int64_t M, int64_t N, int64_t K, int64_t S, int64_t R, bool tc, bool weights) {
  BackwardPlan p;
  const int r = static_cast<int>(R), s = static_cast<int>(S), k = static_cast<int>(K), n = static_cast<int>(N);
  if (tc || !weights) {
    p.h = tc ? shrink_tc_split(M, k) : shrink_split(M, k);
    p.g = tc ? shrink_tc_split(M, n) : shrink_split(M, n);
  } else {
    shrink_pair_split(M, n, k, p.g, p.h);
  }
  p.a = tc ? tokens_tc_split(M, k, s, r) : tokens_split(M, k, s, r);
  p.b = tc ? tokens_tc_split(M, n, s, r) : tokens_split(M, n, s, r);
  p.off_g = up(p.h.count * M * R * 4);
  p.off_counts = p.off_g + up(p.g.count * M * R * 4);
  p.off_a = p.off_counts + (tc ? up((M + 127) / 128 * 4) : 0);
  p.off_b = p.off_a + up(p.a.count * S * R * K * 4);
  p.off_found = p.off_b + up(p.b.count * S * R * N * 4);
  p.off_pa = p.off_found + up((p.a.count + p.b.count) * S * 4);
  const int64_t tiles = (M + kBM - 1) / kBM;
  const int64_t pieces = tc ? up(2 * pad_rank(r) * tiles * kBM * 2) : 0;
  p.off_pb = p.off_pa + pieces;
  p.off_info = p.off_pb + pieces;
  p.bytes = p.off_info + (tc ? up(S * tiles) : 0);
  return p;
}

template <typename T, typename TX>
int backward_typed(const LoraArgs& g, cudaStream_t stream) {
  const Rows rows{g.adapter, g.adapter64, g.rows_per_index, g.M, static_cast<int>(g.S)};
  const int K = static_cast<int>(g.K), N = static_cast<int>(g.N), R = static_cast<int>(g.R);
  const bool tc = tc_shape(g, true) && tc_x(g) && tc_rows(g.y, g.ldy, 2) && tc_weights(g.a, g.lda, g.K, g.S) &&
                  tc_weights(g.b, g.ldb, g.R, g.S);
  const BackwardPlan p = backward_plan(g.M, g.N, g.K, g.S, g.R, tc, g.da != nullptr);
  uint8_t* ws = static_cast<uint8_t*>(g.workspace);
  float* ph = reinterpret_cast<float*>(ws);
  float* pg = reinterpret_cast<float*>(ws + p.off_g);
  float* pa = reinterpret_cast<float*>(ws + p.off_a);
  float* pb = reinterpret_cast<float*>(ws + p.off_b);
  int* fa = reinterpret_cast<int*>(ws + p.off_found);
  int* fb = fa + p.a.count * g.S;
  int* counts = reinterpret_cast<int*>(ws + p.off_counts);
  const TX* x = static_cast<const TX*>(g.x);
  const T* dy = static_cast<const T*>(g.y);
  const T* a = static_cast<const T*>(g.a);
  const T* b = static_cast<const T*>(g.b);
  if (g.M > 0) {
    if (tc) {
      if (int rc = shrink_tc(g, dy, g.ldy, false, nullptr, b, g.ldb, false, N, p.g, pg, counts, true, stream)) return rc;
    } else {
      const auto sg = shrink_args<T, T, false>(dy, g.ldy, nullptr, b, g.ldb, N, R, p.g, pg);
      const auto sh = shrink_args<TX, T, true>(x, g.ldx, g.x_scale, a, g.lda, K, R, p.h, ph);
      if (int rc = g.da ? shrink_pair<TX, T>(sg, p.g.count, sh, p.h.count, rows, R, stream)
                        : shrink<T>(sg, false, p.g.count, rows, R, stream)) {
        return rc;
      }
    }
    if (g.out && tc && tc_rows(g.out, g.ldo, 2)) {
      if (int rc = lora_expand_tc({g.accumulate ? g.out : nullptr, g.ldo, counts, pg, p.g.count, a, 0, g.lda, g.scaling,
                                   g.out, g.ldo, g.M, g.K, g.S, g.R},
                                  {g.adapter, g.adapter64, g.rows_per_index, g.M, g.S}, stream)) {
        return rc;
      }
    } else if (g.out) {
      if (int rc = expand<T, false>(g.accumulate ? static_cast<const T*>(g.out) : nullptr, g.ldo, pg,
                                    p.g.count, a, g.lda, g.scaling, rows, K, R,
                                    static_cast<T*>(g.out), g.ldo, stream)) {
        return rc;
      }
    }
  }
  if (!g.da) return 0;
  if (tc) {
    const LoraRows lr{g.adapter, g.adapter64, g.rows_per_index, g.M, g.S};
    void *qa = ws + p.off_pa, *qb = ws + p.off_pb;
    uint8_t* info = ws + p.off_info;
    if (int rc = shrink_tc(g, x, g.ldx, g.x_scale != nullptr, g.x_scale, a, g.lda, true, K, p.h, ph, nullptr, false, stream)) return rc;
    if (int rc = lora_rank_pieces({pg, p.g.count, g.x_scale, qa, ph, p.h.count, qb, g.scaling, R, info}, lr, stream)) {
      return rc;
    }
    const int per_a = static_cast<int>(p.a.per / kBM), per_b = static_cast<int>(p.b.per / kBM);
    if (int rc = lora_tokens_tc({x, g.x_scale != nullptr, g.ldx, qa, g.M, g.K, g.S, g.R, 0, p.a.count, per_a,
                                 info, pa, fa}, lr, stream)) {
      return rc;
    }
    if (int rc = lora_tokens_tc({dy, 0, g.ldy, qb, g.M, g.N, g.S, g.R, 1, p.b.count, per_b, info, pb, fb}, lr,
                                stream)) {
      return rc;
    }
  } else {
    const TokensArgs<TX> ta{x, g.ldx, g.x_scale, pg, p.g.count, K, p.a.per, p.a.count, (K + kBN - 1) / kBN,
                            aligned(x, g.ldx, sizeof(TX)), pa, fa};
    const TokensArgs<T> tb{dy, g.ldy, nullptr, ph, p.h.count, N, p.b.per, p.b.count, (N + kBN - 1) / kBN,
                           aligned(dy, g.ldy, sizeof(T)), pb, fb};
    if (int rc = tokens_pair<TX, T>(ta, tb, g.scaling, rows, R, stream)) return rc;
  }
  const SumArgs sa{pa, fa, p.a.count, g.R * g.K, g.da}, sb{pb, fb, p.b.count, g.R * g.N, g.db};
  const int64_t most = std::max(sa.per, sb.per);
  const int64_t want = (most + 4 * kThreads - 1) / (4 * kThreads);
  const int64_t cap = std::max<int64_t>(1, 8ll * device_sm_count() / g.S);
  return chained("lora gradient sum",
                 launch_chained(true, sum_splits_kernel<T>,
                                dim3(static_cast<unsigned>(std::min(want, cap)), static_cast<unsigned>(g.S), 2),
                                kThreads, 0, stream, sa, sb, static_cast<int>(g.S)));
}

}  // namespace

int64_t lora_workspace_bytes(int64_t M, int64_t N, int64_t K, int64_t S, int64_t R, int backward) {
  // either form of the kernels may run: which one depends on pointers and strides too
  const int k = static_cast<int>(K);
  if (!backward) {
    return up(std::max(shrink_split(M, k).count, shrink_tc_split(M, k).count) * M * R * 4 + (M + 127) / 128 * 4);
  }
  const bool weights = backward == 1;
  const BackwardPlan plain = backward_plan(M, N, K, S, R, false, weights);
  const bool tc = tc_work(M, N, K, S, true);
  const BackwardPlan other = tc ? backward_plan(M, N, K, S, R, true, weights) : plain;
  return !weights ? std::max(plain.off_a, other.off_a) : std::max(plain.bytes, other.bytes);
}

int lora_add_launch(const LoraArgs& g, cudaStream_t stream) {
  switch (g.dtype) {
    case W8A8_BF16: return add_typed<__nv_bfloat16>(g, stream);
    case W8A8_F16: return add_typed<__half>(g, stream);
    default: return add_typed<float>(g, stream);
  }
}

int lora_backward_launch(const LoraArgs& g, cudaStream_t stream) {
  const bool codes = g.x_scale != nullptr;
  switch (g.dtype) {
    case W8A8_BF16:
      return codes ? backward_typed<__nv_bfloat16, int8_t>(g, stream)
                   : backward_typed<__nv_bfloat16, __nv_bfloat16>(g, stream);
    case W8A8_F16:
      return codes ? backward_typed<__half, int8_t>(g, stream)
                   : backward_typed<__half, __half>(g, stream);
    default:
      return codes ? backward_typed<float, int8_t>(g, stream)
                   : backward_typed<float, float>(g, stream);
  }
}

}  // namespace w8a8
