// Softmax cross entropy of features against every row of a vocabulary table,
// without keeping the logits, and its gradients.
//
//   s_ij = c <h_i, w_j>,  loss_i = log sum_j exp s_ij - s_{i, t_i}
//   ds_ij = g_i (exp(s_ij) / sum_k exp s_ik - [j = t_i])
//   dh_i = c sum_j ds_ij w_j,  dw_j = c sum_i ds_ij h_i
//
// Forward: one product kernel over tiles of (vocabulary x rows) reduces each
// tile of logits in its accumulators to a (maximum, sum of exponentials) per
// row; a second kernel joins the tiles' pairs.  Backward: a piece of the
// vocabulary (and of the rows) at a time, the logits are formed again, turned
// into ds in the epilogue and stored in 16 bits, and two products turn the
// piece into its parts of the gradients.  Nothing of rows x vocabulary exists
// beyond one piece.
#include "gs_capi.h"
#include "gs_resident.h"
#include "gs_tile.h"
#include "gs_xent.h"

#include <algorithm>
#include <type_traits>

namespace gs_xent {

using gs_tile::Accumulators;
using gs_tile::kBK;
using gs_tile::Operand;

// The tile shapes (BM, BN, waves along each, stages).  Big has twice Mid's reuse
// of what it loads and one workgroup a CU (forward of 16384 x 8192 x 512 bf16: 158
// us, Mid 182); Mid wastes less on small sides and two of its workgroups overlap
// (512 x 4096: 16 us, Big 25).  256 x 128 and 128 x 256 tiles were slower than both
// (65536 x 32768 x 512 with gradients: 13.6 to 14 ms, Mid 12.2, Big 11).  Thin: few
// tiles, where what counts is how many bytes are under way (two workgroups a CU,
// four or five steps each); see kThinTiles.
typedef gs_tile::Shape<256, 256, 2, 4> Big;
typedef gs_tile::Shape<128, 128, 2, 2> Mid;
typedef gs_tile::Shape<64, 32, 2, 1, 6> Thin32;
typedef gs_tile::Shape<64, 64, 2, 1, 5> Thin64;

constexpr float kLog2e = 1.4426950408889634f;
constexpr double kLn2 = 0.6931471805599453;
constexpr int kJoinThreads = 256;
// ds of one piece, all planes: 65536 x 32768 x 512 bf16 takes 13.3, 11.1, 10.3, 10.0
// and 9.8 ms at 128, 256, 512, 1024 and 2048 MiB (fewer sums of dh and dw go through memory).
constexpr int64_t kPieceBytes = 1ll << 30;
constexpr int64_t kLeastSide = 4096;         // rows or vocabulary of a piece, at least (a multiple of the tiles')
constexpr int64_t kStatBytes = 256ll << 20;  // the tiles' pairs of one piece (forward)

// ------------------------------------------------------------------ packing
// A matrix and where its layout for the tile loads goes: rows of dp = ceil(dim /
// 8) * 8 16-bit values, zero past dim, from dst (null: it is read in place);
// fp32 as the planes hi and lo of value / unit, `plane` apart.  Only for fp32 and
// for rows that the 16-byte loads cannot take (dim or ld not a multiple of 8).
struct Matrix {
  const void* src;
  int64_t ld, rows;
  uint16_t* dst;
  int64_t plane;
};

// The order of the rows (struct Order), where it is worth a copy of them: the rows
// that count are counted by workgroups of `share` rows (counts[b]), then each puts
// its rows behind those of the workgroups before it.  5 us each for 640000 rows.
constexpr int kOrderBlocks = 1024;
__device__ __forceinline__ bool row_is_used(const Targets& targets, int64_t row, int64_t end) {
  return row < end && targets.at(row) != targets.ignore;
}

__global__ __launch_bounds__(256) void used_kernel(Targets targets, int64_t rows, int64_t share,
                                                   int* __restrict__ counts) {
  __shared__ int lds[4];
  const int64_t begin = blockIdx.x * share, end = min(rows, begin + share);
  int n = 0;
  for (int64_t r = begin; r < end; r += 256)
    n += __builtin_popcountll(__ballot(row_is_used(targets, r + threadIdx.x, end)));
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = n;
  __syncthreads();
  if (threadIdx.x == 0) counts[blockIdx.x] = lds[0] + lds[1] + lds[2] + lds[3];
}

__global__ __launch_bounds__(256) void order_kernel(Targets targets, int64_t rows, int64_t share,
                                                    const int* __restrict__ counts, int* __restrict__ order,
                                                    int* __restrict__ count) {
  __shared__ int before_lds[4], all_lds[4], wave_lds[2][4];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  int before = 0, all = 0;
  for (int b = threadIdx.x; b < (int)gridDim.x; b += 256) {
    all += counts[b];
    if (b < (int)blockIdx.x) before += counts[b];
  }
#pragma unroll
  for (int off = 32; off; off >>= 1) {
    before += __shfl_xor(before, off);
    all += __shfl_xor(all, off);
  }
  if (lane == 0) {
    before_lds[wave] = before;
    all_lds[wave] = all;
  }
  __syncthreads();
  before = before_lds[0] + before_lds[1] + before_lds[2] + before_lds[3];  // used rows before this one
  all = all_lds[0] + all_lds[1] + all_lds[2] + all_lds[3];
  if (blockIdx.x == 0 && threadIdx.x == 0) *count = all;
  const int64_t begin = blockIdx.x * share, end = min(rows, begin + share);
  int turn = 0;
  for (int64_t r = begin; r < end; r += 256, turn ^= 1) {
    const int64_t row = r + threadIdx.x;
    const bool use = row_is_used(targets, row, end);
    const uint64_t who = __ballot(use);
    if (lane == 0) wave_lds[turn][wave] = __builtin_popcountll(who);
    __syncthreads();  // (two places in turn: one barrier does)
    int rank = before + __builtin_popcountll(who & ((1ull << lane) - 1));
    for (int w = 0; w < 4; ++w) {
      const int n = wave_lds[turn][w];
      if (w < wave) rank += n;
      before += n;
    }
    if (row < end) order[use ? (int64_t)rank : all + row - rank] = (int)row;
  }
}

// Bound by its read: 640000 x 64 fp32 (164 MB) in 48 us, and their layout, 164 MB
// to 131 MB of the rows that count, in 75 us (3.5 and 3.7 TB/s).
// fp32: the largest finite magnitudes of the features (of the rows that count
// only, so that what ignored rows hold does not reach the unit of the others) and
// of the table, one value a block, the features' blocks first.  A group of
// `lanes` lanes reads a row, V values a lane at a time.
constexpr int kLargestBlocks = 1024;
template <int V>
__global__ __launch_bounds__(256) void magnitude_kernel(Matrix features, int features_blocks, Matrix table, int dim,
                                                        int lanes, Targets targets, float* __restrict__ largest) {
  __shared__ float lds[4];
  struct __attribute__((aligned(4 * V))) Vec {
    float v[V];
  };
  constexpr int kRows = 8;  // rows in flight
  const bool of_table = (int)blockIdx.x >= features_blocks;
  const Matrix m = of_table ? table : features;
  const float* src = (const float*)m.src;
  const int block = of_table ? blockIdx.x - features_blocks : blockIdx.x;
  const int blocks = of_table ? gridDim.x - features_blocks : features_blocks;
  const int lane = threadIdx.x % lanes;
  const int64_t groups = (int64_t)blocks * (256 / lanes);
  float top = 0.0f;
  for (int64_t r0 = (int64_t)block * (256 / lanes) + threadIdx.x / lanes; r0 < m.rows; r0 += groups * kRows) {
    bool use[kRows];
#pragma unroll
    for (int j = 0; j < kRows; ++j) {
      const int64_t row = r0 + j * groups;
      use[j] = row < m.rows && (of_table || targets.at(row) != targets.ignore);
    }
    for (int c = lane * V; c < dim; c += lanes * V) {
      Vec v[kRows];
#pragma unroll
      for (int j = 0; j < kRows; ++j)
        v[j] = *reinterpret_cast<const Vec*>(src + min(r0 + j * groups, m.rows - 1) * m.ld + c);
#pragma unroll
      for (int j = 0; j < kRows; ++j)
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float x = fabsf(v[j].v[e]);
          if (use[j] && x < INFINITY) top = fmaxf(top, x);
        }
    }
  }
#pragma unroll
  for (int off = 32; off; off >>= 1) top = fmaxf(top, __shfl_xor(top, off));
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = top;
  __syncthreads();
  if (threadIdx.x == 0) largest[blockIdx.x] = fmaxf(fmaxf(lds[0], lds[1]), fmaxf(lds[2], lds[3]));
}

// The unit of a matrix from its blocks' magnitudes: the power of two 2^e that
// brings the largest to [2^13, 2^14).
__device__ __forceinline__ float unit_of(const float* __restrict__ largest, int n) {
  __shared__ float lds[4];
  float top = 0.0f;
  for (int i = threadIdx.x; i < n; i += 256) top = fmaxf(top, largest[i]);
#pragma unroll
  for (int off = 32; off; off >>= 1) top = fmaxf(top, __shfl_xor(top, off));
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = top;
  __syncthreads();
  top = fmaxf(fmaxf(lds[0], lds[1]), fmaxf(lds[2], lds[3]));
  int e = 14;
  if (top > 0.0f) frexpf(top, &e);
  return ldexpf(1.0f, max(e - 14, -126));
}

// Lays two matrices out, the first's blocks first, the first's rows in their order;
// fp32: their units, from largest (the first's magnitudes, then the second's), go to
// units[0] and units[1].
template <typename T>
__global__ __launch_bounds__(256) void layout_kernel(Matrix first, Order order, int first_blocks, Matrix second,
                                                     int dim, int dp,
                                                     const float* __restrict__ largest, int first_n, int second_n,
                                                     float* __restrict__ units) {
  const bool other = (int)blockIdx.x >= first_blocks;
  const Matrix m = other ? second : first;
  const int block = other ? blockIdx.x - first_blocks : blockIdx.x;
  const int blocks = other ? gridDim.x - first_blocks : first_blocks;
  float scale = 1.0f;
  if constexpr (sizeof(T) == 4) {
    const float unit = unit_of(largest + (other ? first_n : 0), other ? second_n : first_n);
    if (block == 0 && threadIdx.x == 0) units[other] = unit;
    scale = 1.0f / unit;
  }
  const T* src = (const T*)m.src;
  const uint32_t vectors = dp / 8;
  const int64_t total = (other ? m.rows : (int64_t)order.used((int)m.rows)) * vectors;
  const bool whole = sizeof(T) == 2 && dim % 8 == 0 && m.ld % 8 == 0 && (uintptr_t)src % 16 == 0;
  for (int64_t v = (int64_t)block * 256 + threadIdx.x; v < total; v += (int64_t)blocks * 256) {
    const int64_t row = v / vectors;
    const int col = (int)(v - row * vectors) * 8;
    const T* s = src + (other ? row : order.row((int)row)) * m.ld + col;
    uint16_t* d = m.dst + row * dp + col;
    if constexpr (sizeof(T) == 4) {
      gs_tile::f16x8 hi, lo;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float x = (col + e < dim ? s[e] : 0.0f) * scale;
        hi[e] = (_Float16)x;
        // nothing is left of infinities and NaN
        lo[e] = fabsf(x) < INFINITY ? (_Float16)gs_tile::behind(x, hi[e]) : (_Float16)0.0f;
      }
      *reinterpret_cast<gs_tile::f16x8*>(d) = hi;
      *reinterpret_cast<gs_tile::f16x8*>(d + m.plane) = lo;
    } else if (whole) {
      *reinterpret_cast<gs_tile::u32x4*>(d) = *reinterpret_cast<const gs_tile::u32x4*>(s);
    } else {
      uint16_t out[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) out[e] = col + e < dim ? __builtin_bit_cast(uint16_t, s[e]) : (uint16_t)0;
      *reinterpret_cast<gs_tile::u32x4*>(d) = *reinterpret_cast<const gs_tile::u32x4*>(out);
    }
  }
}

// m of element e of accumulator block a, from the lane's first m.
__device__ __forceinline__ constexpr int block_m(int a, int e) { return 32 * a + 8 * (e >> 2) + (e & 3); }

// A target as a distance from the lane's first m (base: the piece's first row of
// the table, vocab: the piece's rows); -1 outside the piece or the wave's part of
// the tile (a distance may still belong to the other half of the wave).
__device__ __forceinline__ int from_first(int64_t target, int64_t base, int first, int wave_m, int vocab) {
  if (target < base || target >= base + vocab) return -1;
  const int d = (int)(target - base) - first;
  return d >= 0 && d < wave_m ? d : -1;
}

// (x, sum over all but x) of a set from its largest and the sum that the fma formed (0, or NaN, where that is -inf).
__device__ __forceinline__ float2 pair_of(float x, float scale, float sum) {
  return make_float2(x, x == -INFINITY ? sum - 1.0f : settled(x, scale, sum));
}

// ------------------------------------------------------------------ forward
// The logits of a tile (vocabulary m x rows n), reduced to one pair per row:
// stats[tile * rows + row] = (x, sum over all but x), see settled().  The tile that holds a row's
// target also writes its dot product, upright.  Bound by the matrix cores (and the
// power they may draw) where rows are many, 65536 x 32768 x 512 bf16 at 880 TFLOP/s;
// by the read of the table where they are few, one row x 32000 x 512 in 11 us (3 TB/s).
template <class S, typename T>
__global__ __launch_bounds__(S::kThreads) void logits_fwd_kernel(Operand table, Operand features, int dim,
                                                                 int products, float logit_scale2,
                                                                 const float* __restrict__ units, Targets targets,
                                                                 Order order, int tiles_m,
                                                                 float2* __restrict__ stats,
                                                                 float* __restrict__ label_dot) {
  __shared__ __attribute__((aligned(16))) char lds[S::kLdsBytes];
  const int used_n = (order.used(features.extent) + S::BN - 1) / S::BN;
  const gs_tile::TileAt tile = gs_tile::tile_at(tiles_m, used_n);
  if (tile.n >= used_n) return;
  const int m0 = tile.m * S::BM, n0 = tile.n * S::BN;
  Accumulators<S> acc;
  gs_tile::product<S, T, true, true>(acc, table, features, m0, n0, 0, dim, products, nullptr, lds);

  float scale2 = scale_of(logit_scale2, units);
  const int lane = threadIdx.x & 63;
  const int wm = gs_tile::wave_m<S>(), wn = gs_tile::wave_n<S>();
  float2* red = reinterpret_cast<float2*>(lds);  // [kWavesM][BN]
  // under a negative scale the dot products change their signs first
  if (scale2 < 0.0f) {
    scale2 = -scale2;
#pragma unroll
    for (int a = 0; a < S::kMB; ++a)
#pragma unroll
      for (int b = 0; b < S::kNB; ++b) acc.c[a][b] = -acc.c[a][b];
  }
  const int first = m0 + wm + 4 * (lane >> 5);  // the lane's first m
#pragma unroll
  for (int b = 0; b < S::kNB; ++b) {
    const int n = n0 + wn + 32 * b + (lane & 31);
    const int64_t target = n < features.extent ? targets.at(order.row(n)) : -1;
    const int label_at = from_first(target, 0, first, S::kWaveM, table.extent);
    if (__any(label_at >= 0)) {
      float label = 0.0f;
      bool mine = false;
#pragma unroll
      for (int a = 0; a < S::kMB; ++a)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (label_at == block_m(a, e)) {
            label = acc.c[a][b][e];
            mine = true;
          }
      if (mine) label_dot[n] = label;
    }
    if (m0 + S::BM > table.extent) {
#pragma unroll
      for (int a = 0; a < S::kMB; ++a)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (first + block_m(a, e) >= table.extent) acc.c[a][b][e] = -INFINITY;
    }
    float raw = acc.c[0][b][0];
#pragma unroll
    for (int a = 0; a < S::kMB; ++a)
#pragma unroll
      for (int e = 0; e < 16; ++e) raw = fmaxf(raw, acc.c[a][b][e]);
    raw = fmaxf(raw, __shfl_xor(raw, 32));
    const float top = raw * scale2;
    const float ref = top == -INFINITY ? 0.0f : top;
    // four sums, so that no addition waits for the one before
    float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int a = 0; a < S::kMB; ++a)
#pragma unroll
      for (int e = 0; e < 16; ++e)
        sum[e & 3] += __builtin_amdgcn_exp2f(__builtin_fmaf(acc.c[a][b][e], scale2, -ref));
    float all = (sum[0] + sum[1]) + (sum[2] + sum[3]);
    all += __shfl_xor(all, 32);
    if (lane < 32) red[(wm / S::kWaveM) * S::BN + wn + 32 * b + lane] = pair_of(raw, scale2, all);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < S::BN; i += S::kThreads) {
    if (n0 + i >= features.extent) break;
    float2 r = red[i];
#pragma unroll
    for (int w = 1; w < S::kWavesM; ++w) {
      r = joined(r, red[w * S::BN + i], scale2);
    }
    stats[(int64_t)tile.m * features.extent + n0 + i] = r;
  }
}

// Sums over the rows of a block: the losses in 64 bits, and how many rows count.
struct Sum {
  double loss;
  int64_t count;
};

__device__ __forceinline__ Sum block_sum(Sum s, Sum* lds) {
#pragma unroll
  for (int off = 32; off; off >>= 1) {
    s.loss += __shfl_xor(s.loss, off);
    s.count += __shfl_xor(s.count, off);
  }
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = s;
  __syncthreads();
  s = lds[0];
  for (int w = 1; w < kJoinThreads / 64; ++w) {
    s.loss += lds[w].loss;
    s.count += lds[w].count;
  }
  return s;
}

__device__ __forceinline__ void write_total(Sum s, int reduction, float* loss, int64_t* count) {
  *count = s.count;
  if (reduction == GS_REDUCE_SUM) *loss = (float)s.loss;
  // the mean over no rows is 0 / 0
  if (reduction == GS_REDUCE_MEAN) *loss = (float)(s.loss / (double)s.count);
}

// Joins the tiles' pairs of each row (kLanes lanes a row, in a fixed order):
// norm = (x, 1 / sum, the label's dot product) for the backward, at the row's place
// in the order, and the loss at its own; ignored rows give 0, targets outside the
// vocabulary NaN.  With a reduction the block's sum goes to partial[block], or, when
// there is one block in all, to the result.
template <int kLanes>
__global__ __launch_bounds__(kJoinThreads) void join_kernel(const float2* __restrict__ stats,
                                                            const float* __restrict__ label_dot, int rows,
                                                            int tiles, int vocab, float logit_scale2,
                                                            const float* __restrict__ units, Targets targets,
                                                            Order order, int reduction, float4* __restrict__ norm,
                                                            float* __restrict__ loss_rows,
                                                            Sum* __restrict__ partial, bool last,
                                                            float* __restrict__ loss, int64_t* __restrict__ count) {
  __shared__ Sum lds[kJoinThreads / 64];
  const int sub = threadIdx.x % kLanes;
  const int64_t row = (int64_t)blockIdx.x * (kJoinThreads / kLanes) + threadIdx.x / kLanes;
  // the sum in 64 bits: tiles far below a row's maximum count, however many they are
  const float scale = fabsf(scale_of(logit_scale2, units));
  float x = -INFINITY;
  double sum = 0.0;
  auto add = [&](float ox, double osum) {
    const float all = fmaxf(x, ox);
    sum = sum * (double)weight(x, all, scale) + osum * (double)weight(ox, all, scale);
    x = all;
  };
  if (row < order.used(rows)) {
    // (eight pairs on their way: 65536 rows of 128 tiles take 23 us, and 45 one by one)
    constexpr int kBatch = 8;
    for (int t0 = sub; t0 < tiles; t0 += kBatch * kLanes) {
      float2 o[kBatch];
#pragma unroll
      for (int j = 0; j < kBatch; ++j) o[j] = stats[(int64_t)min(t0 + j * kLanes, tiles - 1) * rows + row];
#pragma unroll
      for (int j = 0; j < kBatch; ++j)
        if (t0 + j * kLanes < tiles) add(o[j].x, 1.0 + (double)o[j].y);
    }
  }
#pragma unroll
  for (int off = kLanes / 2; off; off >>= 1) add(__shfl_xor(x, off), __shfl_xor(sum, off));
  Sum mine = {0.0, 0};
  if (row < rows && sub == 0) {
    const int64_t from = order.row((int)row), t = targets.at(from);
    float value = 0.0f;
    if (t != targets.ignore) {
      value = t >= 0 && t < vocab ? (float)(log(sum) + kLn2 * (double)scale * ((double)x - (double)label_dot[row]))
                                  : __builtin_nanf("");
      mine = {(double)value, 1};
    }
    if (norm) norm[row] = make_float4(x, (float)(1.0 / sum), label_dot[row], 0.0f);
    if (loss_rows) loss_rows[from] = value;
  }
  if (reduction == GS_REDUCE_NONE) return;
  const Sum s = block_sum(mine, lds);
  if (threadIdx.x == 0) {
    if (last) write_total(s, reduction, loss, count);
    else partial[blockIdx.x] = s;
  }
}

__global__ __launch_bounds__(kJoinThreads) void total_kernel(const Sum* __restrict__ partial, int64_t n,
                                                             int reduction, float* loss, int64_t* count) {
  __shared__ Sum lds[kJoinThreads / 64];
  Sum mine = {0.0, 0};
  for (int64_t i = threadIdx.x; i < n; i += kJoinThreads) {
    mine.loss += partial[i].loss;
    mine.count += partial[i].count;
  }
  const Sum s = block_sum(mine, lds);
  if (threadIdx.x == 0) write_total(s, reduction, loss, count);
}

// ------------------------------------------------------------------ backward
// The largest finite |g_i| of the rows that count, one value a block.
__global__ __launch_bounds__(256) void largest_kernel(const float* __restrict__ grad, int64_t rows, Targets targets,
                                                      float* __restrict__ largest) {
  __shared__ float lds[4];
  float top = 0.0f;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < rows; i += (int64_t)gridDim.x * 256) {
    const float g = fabsf(grad[i]);
    if (g < INFINITY && targets.at(i) != targets.ignore) top = fmaxf(top, g);
  }
#pragma unroll
  for (int off = 32; off; off >>= 1) top = fmaxf(top, __shfl_xor(top, off));
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = top;
  __syncthreads();
  if (threadIdx.x == 0) largest[blockIdx.x] = fmaxf(fmaxf(lds[0], lds[1]), fmaxf(lds[2], lds[3]));
}

// Per row of the order: its RowInfo, and one bit: does the row count.  With a gradient for
// each row the factors are g_i / G, G the largest, so that ds stays in the 16-bit
// type's range; alpha holds the rest.
__global__ __launch_bounds__(256) void rows_kernel(const float* __restrict__ grad, int64_t rows, int vocab,
                                                   Targets targets, Order order, int reduction,
                                                   const int64_t* __restrict__ count,
                                                   const float4* __restrict__ norm, float logit_scale,
                                                   float logit_scale2, const float* __restrict__ units,
                                                   float held_scale, const float* __restrict__ largest, int largest_n,
                                                   RowInfo* __restrict__ info, uint64_t* __restrict__ counts,
                                                   double* __restrict__ alpha) {
  __shared__ float lds[4];
  const int lane = threadIdx.x & 63;
  float G = 1.0f;
  if (reduction == GS_REDUCE_NONE) {
    float top = 0.0f;
    for (int i = threadIdx.x; i < largest_n; i += 256) top = fmaxf(top, largest[i]);
#pragma unroll
    for (int off = 32; off; off >>= 1) top = fmaxf(top, __shfl_xor(top, off));
    if (lane == 0) lds[threadIdx.x >> 6] = top;
    __syncthreads();
    top = fmaxf(fmaxf(lds[0], lds[1]), fmaxf(lds[2], lds[3]));
    G = top > 0.0f ? top : 1.0f;
  }
  const int64_t row = (int64_t)blockIdx.x * 256 + threadIdx.x;
  bool use = false;
  if (row < rows) {
    const int64_t from = order.row((int)row), t = targets.at(from);
    const float4 z = norm[row];
    use = t != targets.ignore;
    RowInfo r = {0.0f, 0.0f, 0.0f, -1};
    if (use) {
      const bool in = t >= 0 && t < vocab;
      const float f = (reduction == GS_REDUCE_NONE ? grad[from] / G : 1.0f) * (in ? held_scale : __builtin_nanf(""));
      const float scale = fabsf(scale_of(logit_scale2, units));
      r.top = z.x * scale;
      const float off = __builtin_fmaf(z.x, scale, -r.top);
      r.share = f * z.y * (1.0f - off * kLn2f);
      r.label = (weight(z.z, z.x, scale) * z.y - 1.0f) * f;
      r.target = in ? (int)t : -1;
    }
    info[row] = r;
  }
  const uint64_t bits = __ballot(use);
  if (lane == 0 && row < rows) counts[row / 64] = bits;
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    double g = G;
    if (reduction == GS_REDUCE_SUM) g = grad[0];
    if (reduction == GS_REDUCE_MEAN) g = *count ? (double)grad[0] / (double)*count : 0.0;  // no row counts: zeros
    *alpha = g * (double)logit_scale;
  }
}

__device__ __forceinline__ bool row_counts(const uint64_t* counts, int64_t row) {
  return (counts[row >> 6] >> (row & 63)) & 1;
}

// ds of a piece: tiles of (vocabulary m x rows n) like the forward's, stored as
// ds[row * ld + m] (planes for fp32); rows that do not count and vocabulary
// past the end are zeros.  As the forward, with an epilogue that the one workgroup
// of a CU does not hide: 65536 x 32768 x 512 bf16 in 3.0 ms where the forward takes 2.5.
template <class S, typename T, int kPlanes>
__global__ __launch_bounds__(S::kThreads) void logits_bwd_kernel(Operand table, Operand features, int dim,
                                                                 int products, float logit_scale2,
                                                                 const float* __restrict__ units, int32_t m_base,
                                                                 Order order, int tiles_m,
                                                                 const RowInfo* __restrict__ info,
                                                                 const uint64_t* __restrict__ counts,
                                                                 uint16_t* __restrict__ ds, int64_t ld,
                                                                 int64_t plane) {
  __shared__ __attribute__((aligned(16))) char lds[S::kLdsBytes];
  const int used_n = (order.used(features.extent) + S::BN - 1) / S::BN;
  const gs_tile::TileAt tile = gs_tile::tile_at(tiles_m, used_n);
  if (tile.n >= used_n) return;
  const int m0 = tile.m * S::BM, n0 = tile.n * S::BN;
  Accumulators<S> acc;
  gs_tile::product<S, T, true, true>(acc, table, features, m0, n0, 0, dim, products, nullptr, lds);
  const float scale2 = scale_of(logit_scale2, units);
  const int lane = threadIdx.x & 63;
  const int wm = gs_tile::wave_m<S>(), wn = gs_tile::wave_n<S>();
  const int first = m0 + wm + 4 * (lane >> 5);  // the lane's first m
#pragma unroll
  for (int b = 0; b < S::kNB; ++b) {
    const int n = min(n0 + wn + 32 * b + (lane & 31), features.extent - 1);
    const RowInfo r = info[n];
    const int label_at = from_first(r.target, m_base, first, S::kWaveM, table.extent);
#pragma unroll
    for (int a = 0; a < S::kMB; ++a)
#pragma unroll
      for (int e = 0; e < 16; ++e)
        acc.c[a][b][e] = r.share * __builtin_amdgcn_exp2f(__builtin_fmaf(acc.c[a][b][e], scale2, -r.top));
    if (__any(label_at >= 0)) {
#pragma unroll
      for (int a = 0; a < S::kMB; ++a)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc.c[a][b][e] = label_at == block_m(a, e) ? r.label : acc.c[a][b][e];
    }
    if (m0 + S::BM > table.extent) {
#pragma unroll
      for (int a = 0; a < S::kMB; ++a)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (first + block_m(a, e) >= table.extent) acc.c[a][b][e] = 0.0f;
    }
  }
  // Through LDS, so that the stores are 16 bytes of whole rows: for each column
  // block the waves' rows of BM values, 16 bytes apart from a multiple of the
  // banks, which keeps both sides free of conflicts.
  constexpr int kPitch = S::BM * 2 + 16;
  constexpr int kRows = 32 * S::kWavesN;
  static_assert(kRows * kPitch <= S::kLdsBytes, "a column block of ds fits where the operands were");
#pragma unroll
  for (int b = 0; b < S::kNB; ++b) {
#pragma unroll
    for (int p = 0; p < kPlanes; ++p) {
      if (p > 0 || b > 0) __syncthreads();
      const int n = n0 + wn + 32 * b + (lane & 31);
      const uint32_t use = n < features.extent && row_counts(counts, n) ? ~0u : 0u;
      char* to = lds + (wn / S::kWaveN * 32 + (lane & 31)) * kPitch + (wm + 4 * (lane >> 5)) * 2;
#pragma unroll
      for (int a = 0; a < S::kMB; ++a)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          typename gs_tile::Pack<T>::v4 held;
#pragma unroll
          for (int j = 0; j < 4; j += 2) {
            T pair[2];
            gs_tile::round_pair(acc.c[a][b][4 * q + j], acc.c[a][b][4 * q + j + 1], p + 1 < kPlanes, pair);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              held[j + i] = pair[i];
              if (p + 1 < kPlanes) acc.c[a][b][4 * q + j + i] = gs_tile::behind(acc.c[a][b][4 * q + j + i], pair[i]);
            }
          }
          // a row that does not count holds zeros whatever came out above
          gs_tile::u32x2 bits = __builtin_bit_cast(gs_tile::u32x2, held);
          bits &= use;
          *reinterpret_cast<gs_tile::u32x2*>(to + (32 * a + 8 * q) * 2) = bits;
        }
      __syncthreads();
      constexpr int kRowVectors = S::BM / 8;
#pragma unroll
      for (int j = 0; j < kRows * kRowVectors / S::kThreads; ++j) {
        const int i = threadIdx.x + j * S::kThreads;
        const int slot = i / kRowVectors, v = i % kRowVectors;
        const int row = n0 + slot / 32 * S::kWaveN + 32 * b + slot % 32;
        if (row < features.extent)
          *reinterpret_cast<gs_tile::u32x4*>(ds + p * plane + (int64_t)row * ld + m0 + v * 8) =
              *reinterpret_cast<const gs_tile::u32x4*>(lds + slot * kPitch + v * 16);
      }
    }
  }
}

// A gradient's product: out(n, m) of `N x D` elements, n the rows (of the
// features or of the table), m the D columns.  kTableGrad: dw (both operands in
// K rows, K the rows of the piece); else dh (ds along K, K the vocabulary).
// With `part` set the tile goes, in fp32, to plane blockIdx.y of part (added to
// what is there if `add`); else out = the gradient of the tile's sums in the
// result's type (alpha, unit: see factor_of).
// counts (dh): rows that do not count are zero; order: of the features, K (dw) or n (dh).
// Bound by the matrix cores: 1000 TFLOP/s for either gradient of 65536 x 32768 x 512 bf16.
template <class S, typename T, typename Out, bool kTableGrad>
__global__ __launch_bounds__(S::kThreads) void grad_kernel(Operand x, Operand ds, int32_t K,
                                                           int products, const uint64_t* __restrict__ counts,
                                                           Order order, int tiles_m,
                                                           float* __restrict__ part, int64_t part_plane,
                                                           bool add, const double* __restrict__ alpha,
                                                           const float* __restrict__ unit, Out* __restrict__ out) {
  __shared__ __attribute__((aligned(16))) char lds[S::kLdsBytes];
  const int used_n = (int)(((int64_t)(kTableGrad ? ds.extent : order.used(ds.extent)) + S::BN - 1) / S::BN);
  const gs_tile::TileAt tile = gs_tile::tile_at(tiles_m, used_n);
  const int m0 = tile.m * S::BM, n0 = tile.n * S::BN;
  const int D = x.extent;
  // The parts share what there is of K in whole steps; one past the end has nothing
  // to add, and neither has a tile of features that do not count.
  const int32_t k_used = kTableGrad ? order.used(K) : tile.n >= used_n ? 0 : K;
  const int64_t k_part = (((int64_t)k_used + gridDim.y - 1) / gridDim.y + kBK - 1) / kBK * kBK;
  const int32_t k_begin = (int32_t)min((int64_t)k_used, blockIdx.y * k_part);
  const int32_t k_end = (int32_t)min((int64_t)k_used, k_begin + k_part);
  Accumulators<S> acc;
  gs_tile::product<S, T, false, !kTableGrad>(acc, x, ds, m0, n0, k_begin, k_end, products,
                                             kTableGrad ? counts : nullptr, lds);
  const int lane = threadIdx.x & 63;
  const int wm = gs_tile::wave_m<S>(), wn = gs_tile::wave_n<S>();
  const float factor = part ? 0.0f : factor_of(alpha, unit);
#pragma unroll
  for (int b = 0; b < S::kNB; ++b) {
    const int n = n0 + wn + 32 * b + (lane & 31);
    if (n >= ds.extent) continue;
    const bool use = kTableGrad || row_counts(counts, n);
#pragma unroll
    for (int a = 0; a < S::kMB; ++a)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int m = m0 + wm + 32 * a + 8 * q + 4 * (lane >> 5);
        if (part) {
          float* p = part + (int64_t)blockIdx.y * part_plane + (int64_t)n * D + m;
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (m + j < D) p[j] = acc.c[a][b][4 * q + j] + (add ? p[j] : 0.0f);
        } else {
          const int64_t at = (kTableGrad ? (int64_t)n : order.row(n)) * D + m;
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (m + j < D) out[at + j] = (Out)(use ? gradient_of<T>(acc.c[a][b][4 * q + j], factor) : 0.0f);
        }
      }
  }
}

// out = the gradient of the planes' sum.  dh: rows that do not count (counts) are
// zero, and order says where a row goes; dw: counts null.  A thread has V
// consecutive elements of a row; kGroups threads share their planes, the sums
// joined in order.  Bound by the planes' read: four planes of 4096 x 1024 to bf16
// (76 MB) in 17 us, 29 with an element a thread.
template <int kGroups, int V, typename T, typename Out>
__global__ __launch_bounds__(256) void finish_kernel(const float* __restrict__ part, int planes, int64_t plane,
                                                     int64_t n, int D, const uint64_t* __restrict__ counts,
                                                     Order order, const double* __restrict__ alpha,
                                                     const float* __restrict__ unit,
                                                     Out* __restrict__ out) {
  static_assert(kGroups == 1 || V == 1, "the groups' sums are joined element by element");
  constexpr int kElements = 256 / kGroups;
  struct __attribute__((aligned(4 * V))) Floats {
    float v[V];
  };
  struct __attribute__((aligned(sizeof(Out) * V))) Outs {
    Out v[V];
  };
  __shared__ float lds[256];
  const float factor = factor_of(alpha, unit);
  const int element = threadIdx.x % kElements, group = threadIdx.x / kElements;
  for (int64_t i0 = (int64_t)blockIdx.x * kElements * V; i0 < n; i0 += (int64_t)gridDim.x * kElements * V) {
    const int64_t i = i0 + element * V;
    float s[V] = {};
    if (i < n) {
#pragma unroll 4
      for (int p = group; p < planes; p += kGroups) {
        const Floats x = *reinterpret_cast<const Floats*>(part + (int64_t)p * plane + i);
#pragma unroll
        for (int e = 0; e < V; ++e) s[e] += x.v[e];
      }
    }
    if constexpr (kGroups > 1) {
      __syncthreads();
      lds[threadIdx.x] = s[0];
      __syncthreads();
      if (group > 0) continue;
      for (int g = 1; g < kGroups; ++g) s[0] += lds[g * kElements + element];
    }
    if (i < n) {
      const int64_t row = counts ? i / D : 0;
      const int64_t at = counts ? order.row((int)row) * D + (i - row * D) : i;
      const bool use = !counts || row_counts(counts, row);
      Outs x;
#pragma unroll
      for (int e = 0; e < V; ++e) x.v[e] = (Out)(use ? gradient_of<T>(s[e], factor) : 0.0f);
      *reinterpret_cast<Outs*>(out + at) = x;
    }
  }
}

// ------------------------------------------------------------------ host
static inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
static inline int64_t round_up(int64_t a, int64_t b) { return ceil_div(a, b) * b; }

// Takes parts of a workspace, each on 256 bytes; with a null base it only adds up.
struct Carve {
  char* base;
  size_t at = 0;
  template <typename P>
  P* take(int64_t n) {
    const size_t here = at;
    at += (size_t)round_up(n * (int64_t)sizeof(P), 256);
    return base ? reinterpret_cast<P*>(base + here) : nullptr;
  }
};

struct Problem {
  int64_t rows;
  int32_t vocab, dim, dtype;
  const void* features;
  int64_t ld_features;
  const void* table;
  int64_t ld_table;
  int planes() const { return dtype == GS_FP32 ? gs_tile::kSplitPlanes : 1; }
  int products() const { return dtype == GS_FP32 ? gs_tile::kSplitProducts : 1; }
  // Small problems of 16 bits hold ds in two planes: where few of its values decide a
  // gradient their rounding does not average out (it came to 1.8 times the result's
  // own), and there the products are not what takes the time: 38 x 8192 x 768 bf16
  // with gradients 73 us in one plane, 78 in two.  Less so for short rows, which the
  // kernels that hold them in registers have in one plane: 512 x 1024 x 64 39 and 62 us.
  bool fine() const {
    const int64_t logits = rows * vocab;
    return dtype != GS_FP32 && logits <= 1ll << (dp() <= 128 ? 16 : 19) && logits * dim <= 1ll << 28;
  }
  int ds_planes() const { return dtype == GS_FP32 ? gs_tile::kWidePlanes : fine() ? gs_tile::kFinePlanes : 1; }
  int ds_products() const { return dtype == GS_FP32 ? gs_tile::kWideProducts : fine() ? gs_tile::kFineProducts : 1; }
  int64_t dp() const { return round_up(dim, 8); }
  bool packs(int64_t ld) const { return dtype == GS_FP32 || dim % 8 || ld % 8 || ld > gs_tile::kMaxLd; }
  size_t element() const { return dtype == GS_FP32 ? 4 : 2; }
  // Are the features' rows put in an order (struct Order)?  It takes two small
  // kernels and, for rows that the loads can take in place, a copy of them, whether
  // rows are ignored or not.  With gradients, without and with it, at 0, 10 and 40 %
  // of rows ignored: 65536 x 1024 x 64 fp32 202 / 208, 200 / 197, 190 / 165 us (half
  // the vocabulary: 145 / 149, 139 / 140, 131 / 121); 32768 x 8192 x 512 bf16, in
  // place, 1286 / 1305, 1291 / 1216, 1273 / 922 us.
  bool orders() const {
    const int64_t logits = rows * vocab;
    return packs(ld_features) ? logits >= 1ll << 26 : vocab >= 8192 && logits >= 1ll << 28;
  }
  bool packs_features() const { return packs(ld_features) || orders(); }
};

constexpr int64_t kMaxRows = (1ll << 31) - 1024;
constexpr int64_t kMaxVocab = 1ll << 29;

static int check(const Problem& p) {
  if (p.rows < 0 || p.vocab <= 0 || p.dim <= 0 || p.dtype < GS_FP32 || p.dtype > GS_FP16)
    return GS_ERR_INVALID_ARGUMENT;
  if (p.ld_features < p.dim || p.ld_table < p.dim) return GS_ERR_INVALID_ARGUMENT;
  // (indices of rows, rounded up to a tile, are int32, and a launch has fewer than 2^32 threads)
  if (p.rows > kMaxRows || p.vocab > kMaxVocab || p.dim > gs_tile::kMaxLd - 8) return GS_ERR_OVERFLOW;
  return GS_OK;
}

static int check_pointers(const Problem& p) {
  if (!p.table || (p.rows > 0 && !p.features)) return GS_ERR_INVALID_ARGUMENT;
  if (!p.packs(p.ld_features) && ((uintptr_t)p.features & 15)) return GS_ERR_MISALIGNED;
  if (!p.packs(p.ld_table) && ((uintptr_t)p.table & 15)) return GS_ERR_MISALIGNED;
  return GS_OK;
}

// Both matrices as the kernels read them: in place, or laid out (struct Matrix).
// The layouts of a forward whose backward may follow are of all rows and go to its
// state, where the backward finds them; else the features are laid out a piece
// of the rows at a time, in the workspace.
struct Layouts {
  uint16_t *features_space, *table_space;
  float *units, *largest;
  int *order_space, *used, *order_counts;
  int64_t rows;  // that features_space holds
  int features_n, table_n;

  Layouts() = default;
  Layouts(const Problem& p, int64_t rows_held, Carve& c) : rows(rows_held), features_n(0), table_n(0) {
    const bool fp32 = p.dtype == GS_FP32;
    features_space = c.take<uint16_t>(p.packs_features() ? rows * p.dp() * p.planes() : 0);
    table_space = c.take<uint16_t>(p.packs(p.ld_table) ? p.vocab * p.dp() * p.planes() : 0);
    units = c.take<float>(fp32 ? 2 : 0);
    if (!fp32) units = nullptr;
    order_space = c.take<int>(p.orders() ? p.rows : 0);
    used = c.take<int>(p.orders() ? 1 : 0);
    if (!p.orders()) order_space = used = nullptr;
  }
  Order order() const { return {order_space, used, 0}; }
  const float* features_unit() const { return units; }
  const float* table_unit() const { return units ? units + 1 : nullptr; }

  // Lays out the table and, where all rows are held, the features.
  void prepare(const Problem& p, Targets targets, hipStream_t s) {
    const Matrix f = {p.features, p.ld_features, p.rows, features_space, rows * p.dp()};
    const Matrix t = {p.table, p.ld_table, p.vocab, table_space, p.vocab * p.dp()};
    if (order_space) {
      const int64_t share = round_up(ceil_div(p.rows, kOrderBlocks), 256);
      const int blocks = (int)ceil_div(p.rows, share);
      used_kernel<<<blocks, 256, 0, s>>>(targets, p.rows, share, order_counts);
      order_kernel<<<blocks, 256, 0, s>>>(targets, p.rows, share, order_counts, order_space, used);
    }
    if (units) {
      auto fits = [](const Matrix& m) { return m.ld % 4 == 0 && (uintptr_t)m.src % 16 == 0; };
      const int V = p.dim % 4 == 0 && fits(f) && fits(t) ? 4 : 1;
      int lanes = 1;
      while (lanes < 64 && lanes * V < p.dim) lanes *= 2;
      auto blocks = [&](int64_t n) { return (int)std::min(ceil_div(n, 8 * (256 / lanes)), (int64_t)kLargestBlocks); };
      features_n = blocks(p.rows);
      table_n = blocks(p.vocab);
      auto* kernel = V == 4 ? magnitude_kernel<4> : magnitude_kernel<1>;
      kernel<<<features_n + table_n, 256, 0, s>>>(f, features_n, t, p.dim, lanes, targets, largest);
    }
    lay_out(p, rows == p.rows && p.packs_features() ? f : Matrix{}, order(), p.packs(p.ld_table) ? t : Matrix{}, s);
  }
  void lay_out(const Problem& p, const Matrix& f, const Order& order, const Matrix& t, hipStream_t s) const {
    auto blocks = [&](const Matrix& m) { return (int)std::min(ceil_div(m.rows * (p.dp() / 8), 256), (int64_t)4096); };
    const int fn = blocks(f), tn = blocks(t);
    if (fn + tn == 0) return;
    auto* kernel = p.dtype == GS_FP32 ? layout_kernel<float> : layout_kernel<_Float16>;
    kernel<<<fn + tn, 256, 0, s>>>(f, order, fn, t, p.dim, (int)p.dp(), largest, features_n, table_n, units);
  }
  Operand features(const Problem& p, int64_t first, int64_t n, hipStream_t s) const {
    if (!p.packs_features()) return {(const uint16_t*)p.features + first * p.ld_features, p.ld_features, 0, (int32_t)n};
    const int64_t plane = rows * p.dp();
    if (rows == p.rows) return {features_space + first * p.dp(), p.dp(), plane, (int32_t)n};
    lay_out(p, {p.features, p.ld_features, n, features_space, plane}, order().from(first), Matrix{}, s);
    return {features_space, p.dp(), plane, (int32_t)n};
  }
  Operand table(const Problem& p) const {
    if (!p.packs(p.ld_table)) return {(const uint16_t*)p.table, p.ld_table, 0, p.vocab};
    return {table_space, p.dp(), p.vocab * p.dp(), p.vocab};
  }
};

// What a forward leaves for its backward.
struct State {
  float4* norm;  // see join_kernel
  Layouts layouts;
  size_t bytes;
  State(const Problem& p, void* at) {
    Carve c{(char*)at};
    norm = c.take<float4>(p.rows);
    layouts = Layouts(p, p.rows, c);
    bytes = c.at;
  }
};

// Short rows: the kernels that hold one operand in registers (gs_resident.h).
// The forward alone needs fewer of them, and goes twice as far.
static bool resident(const Problem& p) { return p.dp() <= (p.dtype == GS_FP32 ? 64 : 128) && !p.fine(); }
// Against tiles it needs logits enough to fill its parts: 4096 x 4096 bf16 17 and 18
// us at D = 64, 25 and 22 at 256; 65536 x 1024 24 and 42, 48 and 61.
static bool resident_forward(const Problem& p) {
  const int64_t blocks = ceil_div(p.dp(), 64) * p.planes();
  return blocks <= 4 && p.rows * p.vocab >= blocks * (3ll << 22);
}
// Two workgroups of a forward on rows of one or two 128-byte blocks (counting planes) share a CU, else one has it.
static int resident_forward_slots(const Problem& p) { return ceil_div(p.dp(), 64) * p.planes() <= 2 ? 512 : 256; }

// Parts along the streamed operand for `slots` workgroups at a time: whole rounds
// of the chip, each a part's tiles and about six tiles' time to begin and end;
// and what it costs to write and add the parts' fp32 sums (sum_bytes a part) at
// a tile's microsecond.
static int resident_parts(int64_t held, int64_t stream, int64_t slots, double sum_bytes) {
  const int64_t blocks = ceil_div(held, gs_resident::kHeldRows), tiles = ceil_div(stream, gs_resident::kTileRows);
  const int64_t most = std::min(std::max((int64_t)1, tiles / 4), std::max((int64_t)4, 2 * ceil_div(slots, blocks)));
  int64_t best = 1;
  double least = 1e300;
  for (int64_t n = 1; n <= most; ++n) {
    const double cost = (double)(ceil_div(blocks * n, slots) * (ceil_div(tiles, n) + 6)) +
                        (n > 1 ? (double)n * sum_bytes / 2.0e6 : 0.0);
    if (cost < least) {
      least = cost;
      best = n;
    }
  }
  return (int)best;
}

template <typename T, int kKind>
static void launch_resident(const Problem& p, const gs_resident::Args& a, int parts, hipStream_t s) {
  const dim3 grid((unsigned)ceil_div(a.held.extent, gs_resident::kHeldRows), (unsigned)parts);
  auto launch = [&](auto* kernel) { kernel<<<grid, gs_resident::kThreads, 0, s>>>(a); };
  constexpr bool kForward = kKind == gs_resident::kForward;
  if constexpr (std::is_same<T, _Float16>::value) {
    if (p.dtype == GS_FP32) {
      if constexpr (kForward)
        if (a.dim > 64) return launch(gs_resident::resident_kernel<T, 2, gs_tile::kSplitPlanes, kKind>);
      return launch(gs_resident::resident_kernel<T, 1, gs_tile::kSplitPlanes, kKind>);
    }
  }
  if constexpr (kForward)
    if (a.dim > 128) return launch(gs_resident::resident_kernel<T, 4, 1, kKind>);
  if (a.dim <= 64) launch(gs_resident::resident_kernel<T, 1, 1, kKind>);
  else launch(gs_resident::resident_kernel<T, 2, 1, kKind>);
}

// Big or Mid tiles for a product of M x N (parts: copies of it side by side):
// the time of whole rounds of the chip's 256 CUs, one Big workgroup each or two
// Mid ones, a Mid tile of a quarter of the work taking 1.15 times its share.
static bool takes_big(int64_t M, int64_t N) {
  const int64_t big = ceil_div(M, Big::BM) * ceil_div(N, Big::BN), mid = ceil_div(M, Mid::BM) * ceil_div(N, Mid::BN);
  const int64_t mid_rounds = mid <= 256 ? 1 : 2 * ceil_div(mid, 512);
  return 400 * ceil_div(big, 256) <= 115 * mid_rounds;
}

// Calls f with a value of the shape for the tiles of ds.
template <bool kBig, class F>
static void with_logits_shape(int64_t vocab, int64_t rows, F f) {
  if constexpr (kBig)
    if (takes_big(vocab, rows)) return f(Big{});
  f(Mid{});
}

template <class S>
static int64_t tiles_of(const Problem& p) {
  return ceil_div(p.vocab, S::BM) * ceil_div(p.rows, S::BN);
}
// Thin tiles, where a launch of them fits the chip at once: 200 rows x 1203 x 512 bf16
// take 12.5 us in 32-wide, 13.6 in 64-wide and 16.1 in Mid tiles, 64 x 32000 20.7,
// 17.0 (500 tiles) and 17.4, 100 x 32000 30.2, 22.7 (1000 tiles) and 17.9.
constexpr int64_t kThinTiles = 512;

struct ForwardPlan {
  enum { kThin32, kThin64, kResident, kMid, kBig } shape;
  int64_t rows_piece, tiles_m, blocks;
  int lanes;
  Layouts layouts;
  float2* stats;
  float* label;
  Sum* partial;
  size_t bytes;

  // kept: the layouts lie in a state
  ForwardPlan(const Problem& p, bool kept, void* ws) {
    shape = tiles_of<Thin32>(p) <= kThinTiles ? kThin32 : tiles_of<Thin64>(p) <= kThinTiles ? kThin64
            : resident_forward(p) ? kResident : takes_big(p.vocab, p.rows) ? kBig : kMid;
    const int bm = shape == kBig ? Big::BM : shape == kMid ? Mid::BM : Thin32::BM;
    tiles_m = shape == kResident ? resident_parts(p.rows, p.vocab, resident_forward_slots(p), 0.0)
                                 : ceil_div(p.vocab, bm);
    rows_piece = std::max((int64_t)256, kStatBytes / (tiles_m * (int64_t)sizeof(float2)) / 256 * 256);
    rows_piece = std::min(p.rows, std::min(rows_piece, (int64_t)1 << 20));
    // of a row, in the kernel that joins (1024 rows x 32768 x 256 in all: 35 us with 64
    // lanes, 55 with one; 8192 rows 155 and 146)
    lanes = p.rows <= 4096 && tiles_m >= 16 ? 64 : 1;
    blocks = 0;
    for (int64_t r = 0; r < p.rows; r += rows_piece)
      blocks += ceil_div(std::min(rows_piece, p.rows - r), kJoinThreads / lanes);
    Carve c{(char*)ws};
    if (!kept) layouts = Layouts(p, rows_piece, c);
    layouts.largest = c.take<float>(p.dtype == GS_FP32 ? 2 * kLargestBlocks : 0);
    layouts.order_counts = c.take<int>(p.orders() ? kOrderBlocks : 0);
    stats = c.take<float2>(tiles_m * rows_piece);
    label = c.take<float>(rows_piece);
    partial = c.take<Sum>(blocks);
    bytes = c.at;
  }
};

template <class S, typename T>
static void launch_logits_fwd(const Problem& p, const ForwardPlan& f, const Operand& table, const Operand& features,
                              float scale2, Targets targets, const Order& order, hipStream_t s) {
  const int64_t tiles_n = ceil_div(features.extent, S::BN);
  logits_fwd_kernel<S, T><<<(unsigned)(f.tiles_m * tiles_n), S::kThreads, 0, s>>>(
      table, features, (int)p.dp(), p.products(), scale2, f.layouts.units, targets, order, (int)f.tiles_m,
      f.stats, f.label);
}

template <typename T>
static int forward(const Problem& p, Targets targets, float logit_scale, int reduction, float* loss, float4* norm,
                   int64_t* count, ForwardPlan& f, hipStream_t s) {
  const float scale2 = logit_scale * kLog2e;
  f.layouts.prepare(p, targets, s);
  const Operand table = f.layouts.table(p);
  int64_t block = 0;
  for (int64_t r = 0; r < p.rows; r += f.rows_piece) {
    const int64_t rows = std::min(f.rows_piece, p.rows - r);
    const Operand features = f.layouts.features(p, r, rows, s);
    const Order order = f.layouts.order().from(r);
    switch (f.shape) {
      case ForwardPlan::kThin32: launch_logits_fwd<Thin32, T>(p, f, table, features, scale2, targets, order, s); break;
      case ForwardPlan::kThin64: launch_logits_fwd<Thin64, T>(p, f, table, features, scale2, targets, order, s); break;
      case ForwardPlan::kResident: {
        gs_resident::Args a = {};
        a.held = features;
        a.stream = table;
        a.dim = (int32_t)p.dp();
        a.logit_scale2 = scale2;
        a.units = f.layouts.units;
        a.targets = targets;
        a.order = order;
        a.stats = f.stats;
        a.label_dot = f.label;
        launch_resident<T, gs_resident::kForward>(p, a, (int)f.tiles_m, s);
        break;
      }
      case ForwardPlan::kMid: launch_logits_fwd<Mid, T>(p, f, table, features, scale2, targets, order, s); break;
      case ForwardPlan::kBig: launch_logits_fwd<Big, T>(p, f, table, features, scale2, targets, order, s); break;
    }
    const int64_t blocks = ceil_div(rows, kJoinThreads / f.lanes);
    auto* join = f.lanes == 64 ? join_kernel<64> : join_kernel<1>;
    join<<<(unsigned)blocks, kJoinThreads, 0, s>>>(f.stats, f.label, (int)rows, (int)f.tiles_m, p.vocab, scale2,
                                                   f.layouts.units, targets, order, reduction,
                                                   norm ? norm + r : nullptr,
                                                   reduction == GS_REDUCE_NONE ? loss : nullptr,
                                                   f.partial + block, f.blocks == 1, loss, count);
    block += blocks;
  }
  if (f.blocks > 1 && reduction != GS_REDUCE_NONE)
    total_kernel<<<1, kJoinThreads, 0, s>>>(f.partial, f.blocks, reduction, loss, count);
  return gs_status_from_hip(hipGetLastError());
}

// How a gradient's product of (N x D) over K is done: in which tiles, and in how
// many parts along K.  The time in microseconds: whole rounds of the chip's 256
// CUs (one Big workgroup each, or two Mid ones), each a part's steps and about
// four steps' time to begin and end; and what it takes to write and add the parts'
// fp32 sums.  Of all tiles and parts it takes the fastest or one within 6 % for dh
// and dw of 15 sizes from 16 x 32000 x 512 to 65536 x 64 x 512, where the worst are 2
// to 4 times slower.
struct Split {
  bool big;
  int parts;
};
static Split split_of(int64_t N, int64_t D, int64_t K, int products) {
  Split best = {true, 1};
  double least = 1e300;
  const int64_t steps = ceil_div(K, kBK) * products;
  for (int big = 0; big < 2; ++big) {
    const int64_t tiles = big ? ceil_div(N, Big::BN) * ceil_div(D, Big::BM)
                              : ceil_div(N, Mid::BN) * ceil_div(D, Mid::BM);
    const int64_t most = std::max((int64_t)1, std::min(K / (4 * kBK), (int64_t)256));
    for (int64_t n = 1; n <= most; ++n) {
      const int64_t blocks = tiles * n;
      const double round = big ? 2.1 * ceil_div(blocks, 256) : blocks <= 256 ? 0.8 : 1.24 * ceil_div(blocks, 512);
      const double sums = n > 1 ? 3.0 + (double)n * N * D * 8.0 / 4.0e6 : 0.0;
      const double cost = round * (double)(ceil_div(steps, n) + 4) + sums;
      if (cost < least) {
        least = cost;
        best = {big == 1, (int)n};
      }
    }
  }
  return best;
}

// Calls f with a value of the shape.
template <class F>
static void with_shape(bool big, F f) {
  if (big) f(Big{});
  else f(Mid{});
}

struct BackwardPlan {
  int64_t rows_piece, cols_piece, ld, row_pieces, col_pieces;
  int parts_h, parts_t;  // parts along K of dh and dw, and their tiles
  bool big_h, big_t;
  bool direct_h, direct_t;  // one part and one piece: no fp32 sums in between
  uint16_t* ds;
  RowInfo* info;
  double* alpha;
  float *largest, *part_h, *part_t;
  uint64_t* counts;
  size_t bytes;

  BackwardPlan(const Problem& p, bool want_h, bool want_t, void* ws) {
    if (resident(p)) {  // one piece of everything, and no ds
      rows_piece = p.rows;
      cols_piece = p.vocab;
      ld = 0;
      parts_h = want_h ? resident_parts(p.rows, p.vocab, 256, 4.0 * p.rows * p.dim) : 1;
      parts_t = want_t ? resident_parts(p.vocab, p.rows, 256, 4.0 * p.vocab * p.dim) : 1;
      carve(p, want_h, want_t, ws);
      return;
    }
    // The piece: a part of the longer side against (if it fits) the whole of the
    // shorter, whose gradient's sums then wait from piece to piece; that one is the smaller.
    const int64_t most = kPieceBytes / (2 * p.ds_planes());  // elements of ds
    if (p.rows > p.vocab) {
      cols_piece = std::min((int64_t)p.vocab, most / kLeastSide / 256 * 256);
      rows_piece = std::min(p.rows, most / round_up(cols_piece, 256) / 256 * 256);
    } else {
      rows_piece = std::min(p.rows, most / kLeastSide / 256 * 256);
      cols_piece = std::min((int64_t)p.vocab, most / rows_piece / 256 * 256);
    }
    ld = round_up(cols_piece, 256);
    const Split h = split_of(rows_piece, p.dim, cols_piece, p.ds_products());
    const Split t = split_of(cols_piece, p.dim, rows_piece, p.ds_products());
    big_h = h.big;
    big_t = t.big;
    parts_h = want_h ? h.parts : 1;
    parts_t = want_t ? t.parts : 1;
    carve(p, want_h, want_t, ws);
  }

  void carve(const Problem& p, bool want_h, bool want_t, void* ws) {
    row_pieces = ceil_div(p.rows, rows_piece);
    col_pieces = ceil_div(p.vocab, cols_piece);
    direct_h = parts_h == 1 && col_pieces == 1;
    direct_t = parts_t == 1 && row_pieces == 1;
    Carve c{(char*)ws};
    ds = c.take<uint16_t>(rows_piece * ld * p.ds_planes());
    info = c.take<RowInfo>(p.rows);
    counts = c.take<uint64_t>(ceil_div(p.rows, 64));
    alpha = c.take<double>(1);
    largest = c.take<float>(kLargestBlocks);
    part_h = c.take<float>(want_h && !direct_h ? parts_h * rows_piece * p.dim : 0);
    const int64_t table_rows = row_pieces > 1 ? (int64_t)p.vocab : cols_piece;
    part_t = c.take<float>(want_t && !direct_t ? parts_t * table_rows * p.dim : 0);
    bytes = c.at;
  }
};

static unsigned finish_blocks(int64_t n) { return (unsigned)std::min(ceil_div(n, 256), (int64_t)8192); }

template <typename T, typename Out>
static void finish(const float* part, int planes, int64_t plane, int64_t n, int D, const uint64_t* counts,
                   const Order& order, const double* alpha, const float* unit, Out* out, hipStream_t s) {
  // many planes of few elements (a small table's) do not fill the chip by their
  // elements alone: 65536 x 512 x 64 with gradients 69 us, and 100 with a thread an element
  const bool many = planes >= 16, wide = D % 4 == 0;
  auto* kernel = many ? finish_kernel<8, 1, T, Out> : wide ? finish_kernel<1, 4, T, Out> : finish_kernel<1, 1, T, Out>;
  kernel<<<finish_blocks(many ? n * 8 : wide ? n / 4 : n), 256, 0, s>>>(part, planes, plane, n, D, counts, order, alpha,
                                                                       unit, out);
}

template <typename T, typename Out, int kPlanes>
static int backward(const Problem& p, Targets targets, float logit_scale, int reduction, const State& state,
                    const int64_t* count, const float* grad_loss, Out* grad_features, Out* grad_table,
                    BackwardPlan& b, hipStream_t s) {
  const float scale2 = logit_scale * kLog2e;
  const int D = p.dim;
  int largest_n = 0;
  if (reduction == GS_REDUCE_NONE) {
    largest_n = (int)std::min(ceil_div(p.rows, 256), (int64_t)kLargestBlocks);
    largest_kernel<<<largest_n, 256, 0, s>>>(grad_loss, p.rows, targets, b.largest);
  }
  const Layouts& layouts = state.layouts;
  const float *unit_h = layouts.features_unit(), *unit_w = layouts.table_unit();
  rows_kernel<<<(unsigned)ceil_div(p.rows, 256), 256, 0, s>>>(
      grad_loss, p.rows, p.vocab, targets, layouts.order(), reduction, count, state.norm, logit_scale, scale2,
      layouts.units, Held<T>::kScale, b.largest, largest_n, b.info, b.counts, b.alpha);
  const Operand table = layouts.table(p);
  if (resident(p)) {
    const Operand features = layouts.features(p, 0, p.rows, s);
    gs_resident::Args a = {};
    a.dim = (int32_t)p.dp();
    a.logit_scale2 = scale2;
    a.units = layouts.units;
    a.order = layouts.order();
    a.info = b.info;
    a.counts = b.counts;
    a.alpha = b.alpha;
    a.D = D;
    auto run = [&](auto kind, const Operand& held, const Operand& stream, int parts, float* sums, const float* unit,
                   Out* out, const uint64_t* counts) {
      a.held = held;
      a.stream = stream;
      a.part_sums = parts > 1 ? sums : nullptr;
      a.part_plane = (int64_t)held.extent * D;
      a.unit = unit;
      a.out = out;
      launch_resident<T, decltype(kind)::value>(p, a, parts, s);
      if (parts > 1)
        finish<T>(sums, parts, a.part_plane, a.part_plane, D, counts, layouts.order(), b.alpha, unit, out, s);
    };
    if (grad_features)
      run(std::integral_constant<int, gs_resident::kFeatures>{}, features, table, b.parts_h, b.part_h, unit_w,
          grad_features, b.counts);
    if (grad_table)
      run(std::integral_constant<int, gs_resident::kTable>{}, table, features, b.parts_t, b.part_t, unit_h,
          grad_table, nullptr);
    return gs_status_from_hip(hipGetLastError());
  }
  for (int64_t r = 0; r < p.rows; r += b.rows_piece) {
    const int32_t rows = (int32_t)std::min(b.rows_piece, p.rows - r);
    const Operand features = layouts.features(p, r, rows, s);
    const uint64_t* counts = b.counts + r / 64;
    const Order order = layouts.order().from(r);
    const int64_t ds_plane = rows * b.ld;
    for (int64_t c = 0; c < p.vocab; c += b.cols_piece) {
      const int32_t cols = (int32_t)std::min(b.cols_piece, p.vocab - c);
      Operand piece = table;  // the piece's rows of the table
      piece.p += c * table.ld;
      piece.extent = cols;
      // fp32 always in Mid tiles: the planes of a Big one's ds do not fit its registers
      with_logits_shape<kPlanes == 1>(cols, rows, [&](auto shape) {
        typedef decltype(shape) S;
        const int tiles_m = (int)ceil_div(cols, S::BM), tiles_n = (int)ceil_div(rows, S::BN);
        logits_bwd_kernel<S, T, kPlanes><<<(unsigned)((int64_t)tiles_m * tiles_n), S::kThreads, 0, s>>>(
            piece, features, (int)p.dp(), p.products(), scale2, layouts.units, (int32_t)c, order, tiles_m,
            b.info + r, counts, b.ds, b.ld, ds_plane);
      });
      if (grad_features) {
        with_shape(b.big_h, [&](auto shape) {
          typedef decltype(shape) S;
          const int tiles_m = (int)ceil_div(D, S::BM);
          const Operand ds = {b.ds, b.ld, ds_plane, rows};
          Operand x = piece;  // D columns of the piece's rows
          x.extent = D;
          const int tiles_n = (int)ceil_div(rows, S::BN);
          grad_kernel<S, T, Out, false><<<dim3((unsigned)((int64_t)tiles_m * tiles_n), b.parts_h), S::kThreads, 0, s>>>(
              x, ds, cols, p.ds_products(), counts, order, tiles_m, b.direct_h ? nullptr : b.part_h,
              (int64_t)rows * D, c > 0, b.alpha, unit_w, grad_features);
        });
      }
      if (grad_table) {
        with_shape(b.big_t, [&](auto shape) {
          typedef decltype(shape) S;
          const int tiles_m = (int)ceil_div(D, S::BM);
          const Operand ds = {b.ds, b.ld, ds_plane, cols};
          Operand x = features;
          x.extent = D;
          const int tiles_n = (int)ceil_div(cols, S::BN);
          float* part = b.direct_t ? nullptr : b.part_t + (b.row_pieces > 1 ? c * D : 0);
          const int64_t part_plane = (b.row_pieces > 1 ? (int64_t)p.vocab : cols) * D;
          grad_kernel<S, T, Out, true><<<dim3((unsigned)((int64_t)tiles_m * tiles_n), b.parts_t), S::kThreads, 0, s>>>(
              x, ds, rows, p.ds_products(), counts, order, tiles_m, part, part_plane, r > 0, b.alpha, unit_h,
              grad_table + c * D);
          if (part && b.row_pieces == 1)
            finish<T>(part, b.parts_t, part_plane, (int64_t)cols * D, D, nullptr, Order{}, b.alpha, unit_h,
                      grad_table + c * D, s);
        });
      }
    }
    if (grad_features && !b.direct_h)
      finish<T>(b.part_h, b.parts_h, (int64_t)rows * D, (int64_t)rows * D, D, counts, order, b.alpha, unit_w,
                grad_features, s);
  }
  if (grad_table && b.row_pieces > 1)
    finish<T>(b.part_t, b.parts_t, (int64_t)p.vocab * D, (int64_t)p.vocab * D, D, nullptr, Order{}, b.alpha, unit_h,
              grad_table, s);
  return gs_status_from_hip(hipGetLastError());
}

// No rows: the table's gradient is zero.
__global__ __launch_bounds__(256) void zero_kernel(uint16_t* out, int64_t n) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) out[i] = 0;
}

static bool options_valid(int32_t target_bits, float logit_scale, int32_t reduction) {
  return (target_bits == 32 || target_bits == 64) && logit_scale == logit_scale && fabsf(logit_scale) < INFINITY &&
         reduction >= GS_REDUCE_NONE && reduction <= GS_REDUCE_MEAN;
}

}  // namespace gs_xent

using gs_xent::Problem;

extern "C" size_t gs_xent_state_bytes(int64_t rows, int32_t vocab, int32_t dim, int32_t dtype, int64_t ld_features,
                                      int64_t ld_table) {
  const Problem p = {rows, vocab, dim, dtype, nullptr, ld_features, nullptr, ld_table};
  if (gs_xent::check(p) != GS_OK || rows == 0) return 0;
  return gs_xent::State(p, nullptr).bytes;
}

extern "C" size_t gs_xent_fwd_workspace_bytes(int64_t rows, int32_t vocab, int32_t dim, int32_t dtype,
                                              int64_t ld_features, int64_t ld_table) {
  const Problem p = {rows, vocab, dim, dtype, nullptr, ld_features, nullptr, ld_table};
  if (gs_xent::check(p) != GS_OK || rows == 0) return 0;
  return gs_xent::ForwardPlan(p, false, nullptr).bytes;
}

extern "C" int gs_xent_fwd(int64_t rows, int32_t vocab, int32_t dim, int32_t dtype, const void* features,
                           int64_t ld_features, const void* table, int64_t ld_table, const void* targets,
                           int32_t target_bits, int64_t ignore_index, float logit_scale, int32_t reduction, float* loss,
                           void* state, int64_t* count, void* workspace, size_t workspace_bytes, void* stream) {
  const Problem p = {rows, vocab, dim, dtype, features, ld_features, table, ld_table};
  int status = gs_xent::check(p);
  if (status != GS_OK) return status;
  if (!gs_xent::options_valid(target_bits, logit_scale, reduction) || !count || (rows > 0 && !targets) ||
      (!loss && (rows > 0 || reduction != GS_REDUCE_NONE)))
    return GS_ERR_INVALID_ARGUMENT;
  if ((status = gs_xent::check_pointers(p)) != GS_OK) return status;
  hipStream_t s = (hipStream_t)stream;
  if (rows == 0) {
    if (reduction == GS_REDUCE_NONE) return GS_OK;
    gs_xent::total_kernel<<<1, gs_xent::kJoinThreads, 0, s>>>(nullptr, 0, reduction, loss, count);
    return gs_status_from_hip(hipGetLastError());
  }
  if (((uintptr_t)workspace & 255) || ((uintptr_t)state & 255)) return GS_ERR_MISALIGNED;
  if (!workspace || workspace_bytes < gs_xent::ForwardPlan(p, state != nullptr, nullptr).bytes)
    return GS_ERR_SCRATCH_TOO_SMALL;
  gs_xent::ForwardPlan f(p, state != nullptr, workspace);
  float4* norm = nullptr;
  if (state) {
    const gs_xent::State kept(p, state);
    const gs_xent::Layouts scratch = f.layouts;
    f.layouts = kept.layouts;
    f.layouts.largest = scratch.largest;
    f.layouts.order_counts = scratch.order_counts;
    norm = kept.norm;
  }
  const gs_xent::Targets t = {targets, target_bits, ignore_index};
  auto* run = dtype == GS_BF16 ? gs_xent::forward<__bf16> : gs_xent::forward<_Float16>;  // fp32: planes of fp16
  return run(p, t, logit_scale, reduction, loss, norm, count, f, s);
}

extern "C" size_t gs_xent_bwd_workspace_bytes(int64_t rows, int32_t vocab, int32_t dim, int32_t dtype,
                                              int64_t ld_features, int64_t ld_table, int32_t want_features,
                                              int32_t want_table) {
  const Problem p = {rows, vocab, dim, dtype, nullptr, ld_features, nullptr, ld_table};
  if (gs_xent::check(p) != GS_OK || rows == 0) return 0;
  return gs_xent::BackwardPlan(p, want_features != 0, want_table != 0, nullptr).bytes;
}

extern "C" int gs_xent_bwd(int64_t rows, int32_t vocab, int32_t dim, int32_t dtype, const void* features,
                           int64_t ld_features, const void* table, int64_t ld_table, const void* targets,
                           int32_t target_bits, int64_t ignore_index, float logit_scale, int32_t reduction,
                           const void* state, const int64_t* count, const float* grad_loss, void* grad_features,
                           void* grad_table, void* workspace, size_t workspace_bytes, void* stream) {
  const Problem p = {rows, vocab, dim, dtype, features, ld_features, table, ld_table};
  int status = gs_xent::check(p);
  if (status != GS_OK) return status;
  if (!gs_xent::options_valid(target_bits, logit_scale, reduction)) return GS_ERR_INVALID_ARGUMENT;
  if (!grad_features && !grad_table) return GS_OK;
  hipStream_t s = (hipStream_t)stream;
  if (rows == 0) {
    if (grad_table) {
      const int64_t n = (int64_t)vocab * dim * (int64_t)(p.element() / 2);
      gs_xent::zero_kernel<<<gs_xent::finish_blocks(n), 256, 0, s>>>((uint16_t*)grad_table, n);
    }
    return gs_status_from_hip(hipGetLastError());
  }
  if (!targets || !state || !grad_loss || !count) return GS_ERR_INVALID_ARGUMENT;
  if ((status = gs_xent::check_pointers(p)) != GS_OK) return status;
  if (((uintptr_t)grad_features & 15) || ((uintptr_t)grad_table & 15)) return GS_ERR_MISALIGNED;
  if (((uintptr_t)workspace & 255) || ((uintptr_t)state & 255)) return GS_ERR_MISALIGNED;
  const bool want_h = grad_features != nullptr, want_t = grad_table != nullptr;
  if (!workspace || workspace_bytes < gs_xent::BackwardPlan(p, want_h, want_t, nullptr).bytes)
    return GS_ERR_SCRATCH_TOO_SMALL;
  gs_xent::BackwardPlan b(p, want_h, want_t, workspace);
  const gs_xent::State kept(p, const_cast<void*>(state));
  const gs_xent::Targets t = {targets, target_bits, ignore_index};
  if (dtype == GS_FP32)
    return gs_xent::backward<_Float16, float, gs_tile::kWidePlanes>(
        p, t, logit_scale, reduction, kept, count, grad_loss, (float*)grad_features, (float*)grad_table, b, s);
  auto run = [&](auto* to_features, auto* to_table) {
    typedef std::remove_pointer_t<decltype(to_table)> T;
    auto* call = p.fine() ? gs_xent::backward<T, T, gs_tile::kFinePlanes> : gs_xent::backward<T, T, 1>;
    return call(p, t, logit_scale, reduction, kept, count, grad_loss, to_features, to_table, b, s);
  };
  if (dtype == GS_BF16) return run((__bf16*)grad_features, (__bf16*)grad_table);
  return run((_Float16*)grad_features, (_Float16*)grad_table);
}
