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
#include "gs_tile.h"

#include <type_traits>

namespace gs_xent {

using gs_tile::Accumulators;
using gs_tile::kBK;
using gs_tile::Operand;

typedef gs_tile::Shape<128, 128, 2, 2> Tile;

constexpr float kLog2e = 1.4426950408889634f;
constexpr double kLn2 = 0.6931471805599453;
constexpr int kJoinThreads = 256;
constexpr int64_t kRowsPiece = 65536;          // rows of a piece (a multiple of 64 and of the tile)
constexpr int64_t kPieceBytes = 512ll << 20;   // ds of one piece, all planes
constexpr int64_t kStatBytes = 256ll << 20;    // the tiles' pairs of one piece (forward)
// fp16 has 2^-14 as its least normal number: ds (at most 1 in magnitude after
// the division by the largest g) is held times 2^15, so that probabilities down to 2^-29 keep all
// their bits.  bf16 has fp32's exponents and needs no scale.
template <typename T>
struct Held {
  static constexpr float kScale = 1.0f;
};
template <>
struct Held<_Float16> {
  static constexpr float kScale = 32768.0f;
};

struct Targets {
  const void* p;
  int bits;
  int64_t ignore;
  __device__ __forceinline__ int64_t at(int64_t i) const {
    return bits == 64 ? ((const int64_t*)p)[i] : (int64_t)((const int32_t*)p)[i];
  }
  __host__ __device__ Targets from(int64_t row) const {
    return {(const char*)p + row * (bits / 8), bits, ignore};
  }
};

// ------------------------------------------------------------------ packing
// A matrix laid out for the tile loads: rows of dp = ceil(dim / 8) * 8 16-bit
// values, zero past dim; fp32 as three bf16 planes.  Only for fp32 and for
// rows that the 16-byte loads cannot take (dim or ld not a multiple of 8).
template <typename T>
__global__ __launch_bounds__(256) void pack_kernel(const T* __restrict__ src, int64_t ld, int64_t rows, int dim,
                                                   int dp, uint16_t* __restrict__ dst, int64_t plane) {
  const int64_t total = rows * (dp / 8);
  for (int64_t v = (int64_t)blockIdx.x * 256 + threadIdx.x; v < total; v += (int64_t)gridDim.x * 256) {
    const int64_t row = v / (dp / 8);
    const int col = (int)(v - row * (dp / 8)) * 8;
    const T* s = src + row * ld + col;
    uint16_t out[3][8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if constexpr (sizeof(T) == 4) {
        const float x = col + e < dim ? s[e] : 0.0f;
        float left = x;
#pragma unroll
        for (int p = 0; p < 3; ++p) {
          // the nearest bf16, or x cut short where that would be infinite; nothing is
          // left of infinities and NaN
          __bf16 part = (__bf16)left;
          if (__builtin_isinf((float)part) && __builtin_isfinite(left))
            part = __builtin_bit_cast(__bf16, (uint16_t)(__builtin_bit_cast(uint32_t, left) >> 16));
          out[p][e] = __builtin_bit_cast(uint16_t, part);
          left = __builtin_isfinite(x) ? left - (float)part : 0.0f;
        }
      } else {
        out[0][e] = col + e < dim ? __builtin_bit_cast(uint16_t, s[e]) : (uint16_t)0;
      }
    }
    constexpr int kPlanes = sizeof(T) == 4 ? 3 : 1;
#pragma unroll
    for (int p = 0; p < kPlanes; ++p)
      *reinterpret_cast<gs_tile::u32x4*>(dst + p * plane + row * dp + col) =
          *reinterpret_cast<const gs_tile::u32x4*>(out[p]);
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

// ------------------------------------------------------------------ forward
// The logits of a tile (vocabulary m x rows n), reduced to one pair per row:
// stats[tile * rows + row] = (max, sum of 2^(s log2 e - max)), max the largest
// s log2 e rounded to fp32 (the exponents are formed from the unrounded product).
// The tile that holds a row's target also writes its dot product.  scale2 > 0;
// flip: the dot products change their signs first (a negative scale).
template <class S, typename T>
__global__ __launch_bounds__(S::kThreads) void logits_fwd_kernel(Operand table, Operand features, int dim,
                                                                 int products, float scale2, bool flip,
                                                                 Targets targets, int tiles_m, int tiles_n,
                                                                 float2* __restrict__ stats,
                                                                 float* __restrict__ label_logit) {
  __shared__ __attribute__((aligned(16))) char lds[S::kLdsBytes];
  const gs_tile::TileAt tile = gs_tile::tile_at(tiles_m, tiles_n);
  const int m0 = tile.m * S::BM, n0 = tile.n * S::BN;
  Accumulators<S> acc;
  gs_tile::product<S, T, true, true>(acc, table, features, m0, n0, 0, dim, products, nullptr, lds);

  const int lane = threadIdx.x & 63;
  const int wm = gs_tile::wave_m<S>(), wn = gs_tile::wave_n<S>();
  float2* red = reinterpret_cast<float2*>(lds);  // [kWavesM][BN]
  if (flip) {
#pragma unroll
    for (int a = 0; a < S::kMB; ++a)
#pragma unroll
      for (int b = 0; b < S::kNB; ++b) acc.c[a][b] = -acc.c[a][b];
  }
  const int first = m0 + wm + 4 * (lane >> 5);  // the lane's first m
#pragma unroll
  for (int b = 0; b < S::kNB; ++b) {
    const int n = n0 + wn + 32 * b + (lane & 31);
    const int label_at = from_first(n < features.extent ? targets.at(n) : -1, 0, first, S::kWaveM, table.extent);
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
      if (mine) label_logit[n] = label;
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
    if (lane < 32) red[(wm / S::kWaveM) * S::BN + wn + 32 * b + lane] = make_float2(top, all);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < S::BN; i += S::kThreads) {
    if (n0 + i >= features.extent) break;
    float2 r = red[i];
#pragma unroll
    for (int w = 1; w < S::kWavesM; ++w) {
      const float2 o = red[w * S::BN + i];
      const float top = fmaxf(r.x, o.x), ref = top == -INFINITY ? 0.0f : top;
      r.y = r.y * __builtin_amdgcn_exp2f(r.x - ref) + o.y * __builtin_amdgcn_exp2f(o.x - ref);
      r.x = top;
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
// norm = (maximum, 1 / sum), from which the backward forms the probabilities
// 2^(s log2 e - maximum) / sum to fp32's relative precision, and the loss; ignored rows give 0, targets outside the
// vocabulary NaN.  The block's sum goes to partial[block], or, when there is one block in all, to the result.
template <int kLanes>
__global__ __launch_bounds__(kJoinThreads) void join_kernel(const float2* __restrict__ stats,
                                                            const float* __restrict__ label_logit, int rows,
                                                            int tiles, int vocab, float scale2, Targets targets,
                                                            int reduction, float2* __restrict__ norm,
                                                            float* __restrict__ loss_rows,
                                                            Sum* __restrict__ partial, bool last,
                                                            float* __restrict__ loss, int64_t* __restrict__ count) {
  __shared__ Sum lds[kJoinThreads / 64];
  const int sub = threadIdx.x % kLanes;
  const int64_t row = (int64_t)blockIdx.x * (kJoinThreads / kLanes) + threadIdx.x / kLanes;
  // the sum in 64 bits: tiles far below a row's maximum count, however many they are
  float top = -INFINITY;
  double sum = 0.0;
  auto add = [&](float otop, double osum) {
    const float m = fmaxf(top, otop), ref = m == -INFINITY ? 0.0f : m;
    sum = sum * (double)__builtin_amdgcn_exp2f(top - ref) + osum * (double)__builtin_amdgcn_exp2f(otop - ref);
    top = m;
  };
  if (row < rows) {
    for (int t = sub; t < tiles; t += kLanes) {
      const float2 o = stats[(int64_t)t * rows + row];
      add(o.x, (double)o.y);
    }
  }
#pragma unroll
  for (int off = kLanes / 2; off; off >>= 1) add(__shfl_xor(top, off), __shfl_xor(sum, off));
  Sum mine = {0.0, 0};
  if (row < rows && sub == 0) {
    const int64_t t = targets.at(row);
    float value = 0.0f;
    if (t != targets.ignore) {
      // in 64 bits, the maximum kept apart: small losses do not drown in the logits' size
      value = t >= 0 && t < vocab
                  ? (float)(log(sum) + kLn2 * ((double)top - (double)label_logit[row] * (double)scale2))
                  : __builtin_nanf("");
      mine = {(double)value, 1};
    }
    if (norm) norm[row] = make_float2(top, (float)(1.0 / sum));
    if (loss_rows) loss_rows[row] = value;
  }
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

// Per row: the factor that ds takes in the piece's products, and one bit: does
// the row count.  With a gradient for each row the factors are g_i / G, G the
// largest, so that ds stays in the 16-bit type's range; alpha, applied to the
// sums, holds the rest.
constexpr int kLargestBlocks = 256;
__global__ __launch_bounds__(256) void factors_kernel(const float* __restrict__ grad, int64_t rows, int vocab,
                                                      Targets targets, int reduction, const int64_t* __restrict__ count,
                                                      float logit_scale, float held_scale,
                                                      const float* __restrict__ largest, int largest_n,
                                                      float* __restrict__ factor, uint64_t* __restrict__ counts,
                                                      float* __restrict__ alpha) {
  __shared__ float lds[4];
  const int lane = threadIdx.x & 63;
  float G = 1.0f;
  if (reduction == GS_REDUCE_NONE) {
    float top = (int)threadIdx.x < largest_n ? largest[threadIdx.x] : 0.0f;
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
    const int64_t t = targets.at(row);
    use = t != targets.ignore;
    float f = reduction == GS_REDUCE_NONE ? grad[row] / G : 1.0f;
    if (use && (t < 0 || t >= vocab)) f = __builtin_nanf("");
    factor[row] = use ? f * held_scale : 0.0f;
  }
  const uint64_t bits = __ballot(use);
  if (lane == 0 && row < rows) counts[row / 64] = bits;
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    float g = G;
    if (reduction == GS_REDUCE_SUM) g = grad[0];
    if (reduction == GS_REDUCE_MEAN) g = *count ? grad[0] / (float)*count : 0.0f;  // no row counts: zeros
    *alpha = g * logit_scale / held_scale;
  }
}

__device__ __forceinline__ bool row_counts(const uint64_t* counts, int64_t row) {
  return (counts[row >> 6] >> (row & 63)) & 1;
}

// ds of a piece: tiles of (vocabulary m x rows n) like the forward's, stored as
// ds[row * ld + m] (planes for fp32); rows that do not count and vocabulary
// past the end are zeros.
template <class S, typename T, int kPlanes>
__global__ __launch_bounds__(S::kThreads) void logits_bwd_kernel(Operand table, Operand features, int dim,
                                                                 int products, float scale2, Targets targets,
                                                                 int64_t m_base, int tiles_m, int tiles_n,
                                                                 const float2* __restrict__ norm,
                                                                 const float* __restrict__ factor,
                                                                 const uint64_t* __restrict__ counts,
                                                                 uint16_t* __restrict__ ds, int64_t ld,
                                                                 int64_t plane) {
  __shared__ __attribute__((aligned(16))) char lds[S::kLdsBytes];
  const gs_tile::TileAt tile = gs_tile::tile_at(tiles_m, tiles_n);
  const int m0 = tile.m * S::BM, n0 = tile.n * S::BN;
  Accumulators<S> acc;
  gs_tile::product<S, T, true, true>(acc, table, features, m0, n0, 0, dim, products, nullptr, lds);
  const int lane = threadIdx.x & 63;
  const int wm = gs_tile::wave_m<S>(), wn = gs_tile::wave_n<S>();
  const int first = m0 + wm + 4 * (lane >> 5);  // the lane's first m
#pragma unroll
  for (int b = 0; b < S::kNB; ++b) {
    const int n = min(n0 + wn + 32 * b + (lane & 31), features.extent - 1);
    const int label_at = from_first(targets.at(n), m_base, first, S::kWaveM, table.extent);
    const float2 z = norm[n];
    const float f = factor[n], share = f * z.y;
#pragma unroll
    for (int a = 0; a < S::kMB; ++a)
#pragma unroll
      for (int e = 0; e < 16; ++e)
        acc.c[a][b][e] = share * __builtin_amdgcn_exp2f(__builtin_fmaf(acc.c[a][b][e], scale2, -z.x));
    if (__any(label_at >= 0)) {
#pragma unroll
      for (int a = 0; a < S::kMB; ++a)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc.c[a][b][e] -= label_at == block_m(a, e) ? f : 0.0f;
    }
    if (m0 + S::BM > table.extent) {
#pragma unroll
      for (int a = 0; a < S::kMB; ++a)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (first + block_m(a, e) >= table.extent) acc.c[a][b][e] = 0.0f;
    }
  }
  // Through LDS, so that the stores are 16 bytes of whole rows: BN rows of BM
  // values, 16 bytes apart from a multiple of the banks, which keeps both sides free of conflicts.
  constexpr int kPitch = S::BM * 2 + 16;
  static_assert(S::BN * kPitch <= S::kLdsBytes, "the tile of ds fits where the operands were");
#pragma unroll
  for (int p = 0; p < kPlanes; ++p) {
    if (p > 0) __syncthreads();
#pragma unroll
    for (int b = 0; b < S::kNB; ++b) {
      const int row = wn + 32 * b + (lane & 31);
      const uint32_t use = n0 + row < features.extent && row_counts(counts, n0 + row) ? ~0u : 0u;
#pragma unroll
      for (int a = 0; a < S::kMB; ++a)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          typename gs_tile::Pack<T>::v4 held;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float v = acc.c[a][b][4 * q + j];
            held[j] = (T)v;
            if (kPlanes > 1) acc.c[a][b][4 * q + j] = v - (float)held[j];
          }
          // a row that does not count holds zeros whatever came out above
          gs_tile::u32x2 bits = __builtin_bit_cast(gs_tile::u32x2, held);
          bits &= use;
          *reinterpret_cast<gs_tile::u32x2*>(lds + row * kPitch + (wm + 32 * a + 8 * q + 4 * (lane >> 5)) * 2) = bits;
        }
    }
    __syncthreads();
    constexpr int kRowVectors = S::BM / 8;
    for (int i = threadIdx.x; i < S::BN * kRowVectors; i += S::kThreads) {
      const int row = i / kRowVectors, v = i % kRowVectors;
      if (n0 + row >= features.extent) break;
      *reinterpret_cast<gs_tile::u32x4*>(ds + p * plane + (int64_t)(n0 + row) * ld + m0 + v * 8) =
          *reinterpret_cast<const gs_tile::u32x4*>(lds + row * kPitch + v * 16);
    }
  }
}

// A gradient's product: out(n, m) of `N x D` elements, n the rows (of the
// features or of the table), m the D columns.  kTableGrad: dw (both operands in
// K rows, K the rows of the piece); else dh (ds along K, K the vocabulary).
// With `part` set the tile goes, in fp32, to plane blockIdx.y of part (added to
// what is there if `add`); else out = alpha * tile in the result's type.
// rows_count (dh): rows that do not count are zero.
template <class S, typename T, typename Out, bool kTableGrad>
__global__ __launch_bounds__(S::kThreads) void grad_kernel(Operand x, Operand ds, int32_t K, int32_t k_part,
                                                           int products, const uint64_t* __restrict__ counts,
                                                           int tiles_m, int tiles_n, float* __restrict__ part, int64_t part_plane,
                                                           bool add, const float* __restrict__ alpha,
                                                           Out* __restrict__ out) {
  __shared__ __attribute__((aligned(16))) char lds[S::kLdsBytes];
  const gs_tile::TileAt tile = gs_tile::tile_at(tiles_m, tiles_n);
  const int m0 = tile.m * S::BM, n0 = tile.n * S::BN;
  const int D = x.extent;
  // a part past the end (k_part is rounded up) has nothing to add
  const int32_t k_begin = (int32_t)min((int64_t)K, (int64_t)blockIdx.y * k_part);
  const int32_t k_end = (int32_t)min((int64_t)K, (int64_t)k_begin + k_part);
  Accumulators<S> acc;
  gs_tile::product<S, T, false, !kTableGrad>(acc, x, ds, m0, n0, k_begin, k_end, products,
                                             kTableGrad ? counts : nullptr, lds);
  const int lane = threadIdx.x & 63;
  const int wm = gs_tile::wave_m<S>(), wn = gs_tile::wave_n<S>();
  const float al = part ? 0.0f : *alpha;
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
        const int64_t at = (int64_t)n * D + m;
        if (part) {
          float* p = part + (int64_t)blockIdx.y * part_plane + at;
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (m + j < D) p[j] = acc.c[a][b][4 * q + j] + (add ? p[j] : 0.0f);
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (m + j < D) out[at + j] = (Out)(use ? acc.c[a][b][4 * q + j] * al : 0.0f);
        }
      }
  }
}

// out = alpha * sum of the planes; counts (dh): rows that do not count are zero.
template <typename Out>
__global__ __launch_bounds__(256) void finish_kernel(const float* __restrict__ part, int planes, int64_t plane,
                                                     int64_t n, int D, const uint64_t* __restrict__ counts,
                                                     const float* __restrict__ alpha, Out* __restrict__ out) {
  const float al = *alpha;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    float s = 0.0f;
    for (int p = 0; p < planes; ++p) s += part[(int64_t)p * plane + i];
    out[i] = (Out)(!counts || row_counts(counts, i / D) ? s * al : 0.0f);
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
  int64_t dp() const { return round_up(dim, 8); }
  bool packs(int64_t ld) const { return dtype == GS_FP32 || dim % 8 || ld % 8 || ld > gs_tile::kMaxLd; }
  size_t element() const { return dtype == GS_FP32 ? 4 : 2; }
};

static int check(const Problem& p) {
  if (p.rows < 0 || p.vocab <= 0 || p.dim <= 0 || p.dtype < GS_FP32 || p.dtype > GS_FP16)
    return GS_ERR_INVALID_ARGUMENT;
  if (p.ld_features < p.dim || p.ld_table < p.dim) return GS_ERR_INVALID_ARGUMENT;
  if (p.rows > 0x7fffffffll || p.dim > gs_tile::kMaxLd - 8) return GS_ERR_OVERFLOW;
  return GS_OK;
}

static int check_pointers(const Problem& p) {
  if (!p.table || (p.rows > 0 && !p.features)) return GS_ERR_INVALID_ARGUMENT;
  if (!p.packs(p.ld_features) && ((uintptr_t)p.features & 15)) return GS_ERR_MISALIGNED;
  if (!p.packs(p.ld_table) && ((uintptr_t)p.table & 15)) return GS_ERR_MISALIGNED;
  return GS_OK;
}

static void pack(const Problem& p, const void* src, int64_t ld, int64_t rows, uint16_t* dst, hipStream_t s) {
  const int64_t vectors = rows * (p.dp() / 8);
  if (vectors == 0) return;
  const int blocks = (int)min(ceil_div(vectors, 256), (int64_t)16384);
  const int64_t plane = rows * p.dp();
  if (p.dtype == GS_FP32)
    pack_kernel<<<blocks, 256, 0, s>>>((const float*)src, ld, rows, p.dim, (int)p.dp(), dst, plane);
  else
    pack_kernel<<<blocks, 256, 0, s>>>((const _Float16*)src, ld, rows, p.dim, (int)p.dp(), dst, plane);
}

// The operand of `rows` rows from row `first` of a matrix: in place, or packed into `space`.
static Operand operand(const Problem& p, const void* src, int64_t ld, int64_t first, int64_t rows, uint16_t* space,
                       hipStream_t s) {
  const char* at = (const char*)src + first * ld * (int64_t)p.element();
  if (!p.packs(ld)) return {(const uint16_t*)at, ld, 0, (int32_t)rows};
  pack(p, at, ld, rows, space, s);
  return {space, p.dp(), rows * p.dp(), (int32_t)rows};
}

// The logits' scale in base 2.  Zero becomes the least normal number: the same
// flat distribution, and minus infinity (what lies past the vocabulary) stays that.
static float base2_scale(float logit_scale) {
  const float scale2 = logit_scale * kLog2e;
  return scale2 == 0.0f ? 1.17549435e-38f : scale2;
}

struct ForwardPlan {
  int64_t rows_piece, tiles_m, blocks;
  int lanes;
  uint16_t *table, *features;
  float2* stats;
  float* label;
  Sum* partial;
  size_t bytes;

  ForwardPlan(const Problem& p, void* ws) {
    tiles_m = ceil_div(p.vocab, Tile::BM);
    rows_piece = kStatBytes / (tiles_m * (int64_t)sizeof(float2)) / Tile::BN * Tile::BN;
    if (rows_piece < Tile::BN) rows_piece = Tile::BN;
    if (rows_piece > (1 << 20)) rows_piece = 1 << 20;
    if (rows_piece > p.rows) rows_piece = p.rows;
    lanes = p.rows <= 4096 ? 64 : 1;
    blocks = 0;
    for (int64_t r = 0; r < p.rows; r += rows_piece)
      blocks += ceil_div(min(rows_piece, p.rows - r), kJoinThreads / lanes);
    Carve c{(char*)ws};
    table = c.take<uint16_t>(p.packs(p.ld_table) ? p.vocab * p.dp() * p.planes() : 0);
    features = c.take<uint16_t>(p.packs(p.ld_features) ? rows_piece * p.dp() * p.planes() : 0);
    stats = c.take<float2>(tiles_m * rows_piece);
    label = c.take<float>(rows_piece);
    partial = c.take<Sum>(blocks);
    bytes = c.at;
  }
};

template <typename T>
static void launch_logits_fwd(const Problem& p, const ForwardPlan& f, const Operand& table, const Operand& features,
                              float scale2, Targets targets, hipStream_t s) {
  const int64_t tiles = f.tiles_m * ceil_div(features.extent, Tile::BN);
  logits_fwd_kernel<Tile, T><<<(unsigned)tiles, Tile::kThreads, 0, s>>>(
      table, features, (int)p.dp(), p.products(), fabsf(scale2), scale2 < 0.0f, targets, (int)f.tiles_m, (int)ceil_div(features.extent, Tile::BN), f.stats, f.label);
}

static int forward(const Problem& p, Targets targets, float logit_scale, int reduction, float* loss, float2* norm,
                   int64_t* count, const ForwardPlan& f, hipStream_t s) {
  if (p.rows == 0) {
    total_kernel<<<1, kJoinThreads, 0, s>>>(nullptr, 0, reduction, loss, count);
    return gs_status_from_hip(hipGetLastError());
  }
  const float scale2 = base2_scale(logit_scale);
  const Operand table = operand(p, p.table, p.ld_table, 0, p.vocab, f.table, s);
  int64_t block = 0;
  for (int64_t r = 0; r < p.rows; r += f.rows_piece) {
    const int64_t rows = min(f.rows_piece, p.rows - r);
    const Operand features = operand(p, p.features, p.ld_features, r, rows, f.features, s);
    if (p.dtype == GS_FP16) launch_logits_fwd<_Float16>(p, f, table, features, scale2, targets.from(r), s);
    else launch_logits_fwd<__bf16>(p, f, table, features, scale2, targets.from(r), s);
    const int64_t blocks = ceil_div(rows, kJoinThreads / f.lanes);
    auto* join = f.lanes == 64 ? join_kernel<64> : join_kernel<1>;
    join<<<(unsigned)blocks, kJoinThreads, 0, s>>>(f.stats, f.label, (int)rows, (int)f.tiles_m, p.vocab, fabsf(scale2),
                                                   targets.from(r), reduction, norm ? norm + r : nullptr,
                                                   reduction == GS_REDUCE_NONE ? loss + r : nullptr,
                                                   f.partial + block, f.blocks == 1, loss, count);
    block += blocks;
  }
  if (f.blocks > 1) total_kernel<<<1, kJoinThreads, 0, s>>>(f.partial, f.blocks, reduction, loss, count);
  return gs_status_from_hip(hipGetLastError());
}

// How many parts a gradient's product of (N x D) over K is cut into along K, so
// that the launch fills the chip; a part has at least four steps.
static int parts_for(int64_t N, int64_t D, int64_t K) {
  const int64_t tiles = ceil_div(N, Tile::BN) * ceil_div(D, Tile::BM);
  const int64_t want = tiles >= 384 ? 1 : ceil_div(512, tiles);
  return (int)max((int64_t)1, min(want, K / (4 * kBK)));
}

struct BackwardPlan {
  int64_t rows_piece, cols_piece, ld, row_pieces, col_pieces;
  int parts_h, parts_t;  // parts along K of dh and dw
  bool direct_h, direct_t;  // one part and one piece: no fp32 sums in between
  uint16_t *table, *features, *ds;
  float *factor, *alpha, *largest, *part_h, *part_t;
  uint64_t* counts;
  size_t bytes;

  BackwardPlan(const Problem& p, bool want_h, bool want_t, void* ws) {
    const int64_t row_bytes = 2 * p.planes() * round_up(p.vocab, Tile::BM);
    rows_piece = min(p.rows, max(kRowsPiece, kPieceBytes / row_bytes / kRowsPiece * kRowsPiece));
    cols_piece = max((int64_t)Tile::BM, kPieceBytes / (rows_piece * 2 * p.planes()) / Tile::BM * Tile::BM);
    if (cols_piece > p.vocab) cols_piece = p.vocab;
    ld = round_up(cols_piece, Tile::BM);
    row_pieces = ceil_div(p.rows, rows_piece);
    col_pieces = ceil_div(p.vocab, cols_piece);
    parts_h = want_h ? parts_for(rows_piece, p.dim, cols_piece) : 1;
    parts_t = want_t ? parts_for(cols_piece, p.dim, rows_piece) : 1;
    direct_h = parts_h == 1 && col_pieces == 1;
    direct_t = parts_t == 1 && row_pieces == 1;
    Carve c{(char*)ws};
    table = c.take<uint16_t>(p.packs(p.ld_table) ? p.vocab * p.dp() * p.planes() : 0);
    features = c.take<uint16_t>(p.packs(p.ld_features) ? rows_piece * p.dp() * p.planes() : 0);
    ds = c.take<uint16_t>(rows_piece * ld * p.planes());
    factor = c.take<float>(p.rows);
    counts = c.take<uint64_t>(ceil_div(p.rows, 64));
    alpha = c.take<float>(1);
    largest = c.take<float>(kLargestBlocks);
    part_h = c.take<float>(want_h && !direct_h ? parts_h * rows_piece * p.dim : 0);
    part_t = c.take<float>(want_t && !direct_t ? parts_t * (row_pieces > 1 ? (int64_t)p.vocab : cols_piece) * p.dim : 0);
    bytes = c.at;
  }
};

static unsigned finish_blocks(int64_t n) { return (unsigned)min(ceil_div(n, 256), (int64_t)8192); }

template <typename T, typename Out, int kPlanes>
static int backward(const Problem& p, Targets targets, float logit_scale, int reduction, const float2* norm,
                    const int64_t* count, const float* grad_loss, Out* grad_features, Out* grad_table,
                    const BackwardPlan& b, hipStream_t s) {
  const float scale2 = base2_scale(logit_scale);
  const int D = p.dim;
  int largest_n = 0;
  if (reduction == GS_REDUCE_NONE) {
    largest_n = (int)min(ceil_div(p.rows, 256), (int64_t)kLargestBlocks);
    largest_kernel<<<largest_n, 256, 0, s>>>(grad_loss, p.rows, targets, b.largest);
  }
  factors_kernel<<<(unsigned)ceil_div(p.rows, 256), 256, 0, s>>>(grad_loss, p.rows, p.vocab, targets, reduction, count,
                                                                 logit_scale, Held<T>::kScale, b.largest, largest_n,
                                                                 b.factor, b.counts, b.alpha);
  const Operand table = operand(p, p.table, p.ld_table, 0, p.vocab, b.table, s);
  const int tiles_d = (int)ceil_div(D, Tile::BM);
  for (int64_t r = 0; r < p.rows; r += b.rows_piece) {
    const int64_t rows = min(b.rows_piece, p.rows - r);
    const Operand features = operand(p, p.features, p.ld_features, r, rows, b.features, s);
    const uint64_t* counts = b.counts + r / 64;
    const int64_t ds_plane = rows * b.ld;
    for (int64_t c = 0; c < p.vocab; c += b.cols_piece) {
      const int32_t cols = (int32_t)min(b.cols_piece, p.vocab - c);
      Operand piece = table;  // the piece's rows of the table
      piece.p += c * table.ld;
      piece.extent = cols;
      const int tiles_v = (int)ceil_div(cols, Tile::BM);
      logits_bwd_kernel<Tile, T, kPlanes><<<(unsigned)(tiles_v * ceil_div(rows, Tile::BN)), Tile::kThreads, 0, s>>>(
          piece, features, (int)p.dp(), p.products(), scale2, targets.from(r), c, tiles_v, (int)ceil_div(rows, Tile::BN), norm + r, b.factor + r,
          counts, b.ds, b.ld, ds_plane);
      if (grad_features) {
        const Operand ds = {b.ds, b.ld, ds_plane, (int32_t)rows};
        Operand x = piece;  // D columns of the piece's rows
        x.extent = D;
        const int32_t k_part = (int32_t)round_up(ceil_div(cols, b.parts_h), kBK);
        grad_kernel<Tile, T, Out, false><<<dim3((unsigned)(tiles_d * ceil_div(rows, Tile::BN)), b.parts_h),
                                           Tile::kThreads, 0, s>>>(
            x, ds, cols, k_part, p.products(), counts, tiles_d, (int)ceil_div(rows, Tile::BN), b.direct_h ? nullptr : b.part_h, rows * D, c > 0,
            b.alpha, grad_features + r * D);
      }
      if (grad_table) {
        const Operand ds = {b.ds, b.ld, ds_plane, cols};
        Operand x = features;
        x.extent = D;
        const int32_t k_part = (int32_t)round_up(ceil_div(rows, b.parts_t), kBK);
        float* part = b.direct_t ? nullptr : b.part_t + (b.row_pieces > 1 ? c * D : 0);
        const int64_t part_plane = (b.row_pieces > 1 ? (int64_t)p.vocab : cols) * D;
        grad_kernel<Tile, T, Out, true><<<dim3((unsigned)(tiles_d * ceil_div(cols, Tile::BN)), b.parts_t),
                                          Tile::kThreads, 0, s>>>(
            x, ds, (int32_t)rows, k_part, p.products(), counts, tiles_d, (int)ceil_div(cols, Tile::BN), part, part_plane, r > 0, b.alpha, grad_table + c * D);
        if (part && b.row_pieces == 1)
          finish_kernel<<<finish_blocks((int64_t)cols * D), 256, 0, s>>>(part, b.parts_t, part_plane, (int64_t)cols * D,
                                                                        D, nullptr, b.alpha, grad_table + c * D);
      }
    }
    if (grad_features && !b.direct_h)
      finish_kernel<<<finish_blocks(rows * D), 256, 0, s>>>(b.part_h, b.parts_h, rows * D, rows * D, D, counts, b.alpha,
                                                            grad_features + r * D);
  }
  if (grad_table && b.row_pieces > 1)
    finish_kernel<<<finish_blocks((int64_t)p.vocab * D), 256, 0, s>>>(b.part_t, b.parts_t, (int64_t)p.vocab * D,
                                                                     (int64_t)p.vocab * D, D, nullptr, b.alpha, grad_table);
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

extern "C" size_t gs_xent_fwd_workspace_bytes(int64_t rows, int32_t vocab, int32_t dim, int32_t dtype,
                                              int64_t ld_features, int64_t ld_table) {
  const Problem p = {rows, vocab, dim, dtype, nullptr, ld_features, nullptr, ld_table};
  if (gs_xent::check(p) != GS_OK || rows == 0) return 0;
  return gs_xent::ForwardPlan(p, nullptr).bytes;
}

extern "C" int gs_xent_fwd(int64_t rows, int32_t vocab, int32_t dim, int32_t dtype, const void* features,
                           int64_t ld_features, const void* table, int64_t ld_table, const void* targets,
                           int32_t target_bits, int64_t ignore_index, float logit_scale, int32_t reduction, float* loss,
                           float* norm, int64_t* count, void* workspace, size_t workspace_bytes, void* stream) {
  const Problem p = {rows, vocab, dim, dtype, features, ld_features, table, ld_table};
  int status = gs_xent::check(p);
  if (status != GS_OK) return status;
  if (!gs_xent::options_valid(target_bits, logit_scale, reduction) || !count || (rows > 0 && !targets) ||
      (!loss && (rows > 0 || reduction != GS_REDUCE_NONE)))
    return GS_ERR_INVALID_ARGUMENT;
  if ((status = gs_xent::check_pointers(p)) != GS_OK) return status;
  if (rows > 0 && ((uintptr_t)workspace & 255)) return GS_ERR_MISALIGNED;
  if (rows > 0 && (!workspace || workspace_bytes < gs_xent::ForwardPlan(p, nullptr).bytes)) return GS_ERR_SCRATCH_TOO_SMALL;
  if (rows == 0) workspace = nullptr;
  const gs_xent::ForwardPlan f(p, workspace);
  return gs_xent::forward(p, {targets, target_bits, ignore_index}, logit_scale, reduction, loss, (float2*)norm, count, f,
                          (hipStream_t)stream);
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
                           const float* norm, const int64_t* count, const float* grad_loss, void* grad_features,
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
  if (!targets || !norm || !grad_loss || !count) return GS_ERR_INVALID_ARGUMENT;
  if ((status = gs_xent::check_pointers(p)) != GS_OK) return status;
  if ((uintptr_t)workspace & 255) return GS_ERR_MISALIGNED;
  const bool want_h = grad_features != nullptr, want_t = grad_table != nullptr;
  if (!workspace || workspace_bytes < gs_xent::BackwardPlan(p, want_h, want_t, nullptr).bytes)
    return GS_ERR_SCRATCH_TOO_SMALL;
  const gs_xent::BackwardPlan b(p, want_h, want_t, workspace);
  const gs_xent::Targets t = {targets, target_bits, ignore_index};
  if (dtype == GS_FP32)
    return gs_xent::backward<__bf16, float, 3>(p, t, logit_scale, reduction, (const float2*)norm, count, grad_loss,
                                               (float*)grad_features, (float*)grad_table, b, s);
  if (dtype == GS_BF16)
    return gs_xent::backward<__bf16, __bf16, 1>(p, t, logit_scale, reduction, (const float2*)norm, count, grad_loss,
                                                (__bf16*)grad_features, (__bf16*)grad_table, b, s);
  return gs_xent::backward<_Float16, _Float16, 1>(p, t, logit_scale, reduction, (const float2*)norm, count, grad_loss,
                                                  (_Float16*)grad_features, (_Float16*)grad_table, b, s);
}
