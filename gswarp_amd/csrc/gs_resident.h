// The cross entropy's products for short rows (up to 128 values of 16 bits or 64
// of fp32, and twice that for the forward): one operand's rows stay in registers,
// the other's stream through LDS in tiles of 64 rows, and the logits of a tile never
// leave the registers of the wave that formed them.
//
//   kForward  features held, table streamed: the running maximum and sum of a
//             softmax over the tiles, one pair per row and part;
//   kFeatures features held, table streamed: ds = f (p - [label]), then
//             dh += ds W with the tile that is in LDS anyway;
//   kTable    table held, features streamed: ds, turned over through LDS, then
//             dw += ds^T H.
//
// Against the tiles of logits in memory this forms the logits once more (10 N V D
// flops in all instead of 8) and moves no logits: at D = 64 a logit costs 256
// flops and, there, 6 to 22 bytes.  Forward and gradients, this against tiles, in us:
//   16384 rows x 32768: bf16 D = 64 461 / 931, D = 128 678 / 1099; fp32 D = 64 1209 / 3365
//   1024 rows x 512:    bf16 D = 64 42 / 59, fp32 81 / 93
// What bounds it: the vector instructions, with the matrix ones (37 to 48 % busy).
// 640000 x 512 x 64 fp32, a fifth of the rows ignored: kForward 134 us, kFeatures
// 336, kTable 285 (the products alone would take 73, 171 and 171 at the rate of a
// large fp16 product).
//
// What the products bring per element is little, so the vector instructions
// count: an element takes an fma, an exponential and a multiplication.  The label
// is kept out of that: its logit is formed once per row (kForward), kFeatures
// looks for it only in the tiles that hold one of a wave's labels, and kTable
// writes f (p_t - 1), formed once per row in fp32, over p_t on its way through LDS.
#pragma once

#include "gs_tile.h"
#include "gs_xent.h"

#include <type_traits>

namespace gs_resident {

using gs_tile::f32x16;
using gs_tile::kPlaneStep;
using gs_tile::mfma;
using gs_tile::Operand;
using gs_tile::Pack;
using gs_xent::RowInfo;
using gs_xent::kLn2f;
using gs_xent::scale_of;
using gs_xent::settled;

enum Kind { kForward, kFeatures, kTable };

constexpr int kWaves = 8, kThreads = 64 * kWaves;
constexpr int kHeldRows = 32 * kWaves;  // held rows of a workgroup, 32 a wave
constexpr int kTileRows = 64;
constexpr int kStages = 4;

struct Args {
  Operand held, stream;
  int32_t dim;   // of the operands, padded to 8
  float logit_scale2;
  const float* units;
  gs_xent::Order order;  // of the features' rows
  // kForward: stats[part * rows + row], and the rows' labels' dot products, upright
  float* label_dot;
  gs_xent::Targets targets;
  float2* stats;
  // kFeatures, kTable
  const RowInfo* info;
  const uint64_t* counts;
  float* part_sums;  // fp32, part_plane apart; null: the gradients go to out
  int64_t part_plane;
  const double* alpha;
  const float* unit;
  int32_t D;
  void* out;
};

// The held rows' matrix-core operands: lane l holds row l % 32 of the wave's, columns 16 s + 8 (l / 32) ..+7.
template <typename T, int KB, int PL>
struct HeldRows {
  typename Pack<T>::v8 v[PL][4 * KB];
  // row: the lane's row of the operand (any; none: nothing but zeros)
  __device__ __forceinline__ void load(const Operand& o, int64_t row, bool some, int dim) {
    const int first = 8 * ((threadIdx.x & 63) >> 5);
#pragma unroll
    for (int p = 0; p < PL; ++p)
#pragma unroll
      for (int s = 0; s < 4 * KB; ++s) {
        v[p][s] = typename Pack<T>::v8{};
        if (some && 16 * s + first < dim)
          v[p][s] = *reinterpret_cast<const typename Pack<T>::v8*>(o.p + p * o.plane + row * o.ld + 16 * s + first);
      }
  }
};

// s = the 32 x 32 products of 32 rows x and 32 rows y, in the order of K (and of
// the planes) that gs_tile::product takes, so that a logit has the same bits wherever it is formed.
// x(plane, step) and y(plane, step) give the operands.
template <typename T, int KB, int PL, class X, class Y>
__device__ __forceinline__ void logits(f32x16& s, X x, Y y) {
  s = f32x16{};
  if (PL > 1) {
#pragma unroll
    for (int k = 0; k < 4 * KB; ++k) s = mfma(x(PL - 1, k), y(0, k), s);
#pragma unroll
    for (int k = 0; k < 4 * KB; ++k) s = mfma(x(0, k), y(PL - 1, k), s);
    s *= 1.0f / kPlaneStep;
  }
#pragma unroll
  for (int k = 0; k < 4 * KB; ++k) s = mfma(x(0, k), y(0, k), s);
}

// Element e of a 32 x 32 accumulator: its m from the lane's first.
__device__ __forceinline__ constexpr int block_m(int e) { return 8 * (e >> 2) + (e & 3); }

// acc[m] of the lane whose block holds column m - own (a lane's own number in 0..31): the diagonal.
__device__ __forceinline__ float diagonal(const f32x16& s) {
  const int lane = threadIdx.x & 63, n = lane & 31;
  float d = 0.0f;
#pragma unroll
  for (int e = 0; e < 16; ++e) d = block_m(e) + 4 * (lane >> 5) == n ? s[e] : d;
  const bool mine = ((n >> 2) & 1) == lane >> 5;
  const float other = __shfl_xor(d, 32);
  return mine ? d : other;
}

// Planes of eight consecutive accumulator elements (an operand of 16 rows as K).
template <typename T, int kPlanes>
__device__ __forceinline__ void planes_of(const f32x16& s, int from, typename Pack<T>::v8* out) {
  float v[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = s[from + e];
#pragma unroll
  for (int p = 0; p < kPlanes; ++p)
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      T pair[2];
      gs_tile::round_pair(v[e], v[e + 1], p + 1 < kPlanes, pair);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        out[p][e + i] = pair[i];
        if (p + 1 < kPlanes) v[e + i] = gs_tile::behind(v[e + i], pair[i]);
      }
    }
}

template <typename T, int KB, int PL, int kKind>
__global__ __launch_bounds__(kThreads, kKind == kForward && KB * PL <= 2 ? 4 : 2) void resident_kernel(Args a) {
  typedef gs_tile::Stage<true, kTileRows, kWaves> Stage;
  typedef typename Pack<T>::v8 v8;
  constexpr int kTile = PL * KB * Stage::kBytes;
  constexpr int kInfo = kKind == kTable ? kWaves * 1024 : 0;  // a copy of the tile's RowInfo for each wave
  constexpr int kTurn = kKind == kTable ? kWaves * 4096 : 0;  // a wave's ds, to be turned over
  constexpr int kDsPlanes = PL > 1 ? gs_tile::kWidePlanes : 1;
  constexpr int kSums = kKind == kForward ? 1 : PL > 1 ? 3 : 1;  // sums of one step down each
  constexpr int kDBlocks = kKind == kForward ? 1 : 2 * KB;
  // kFeatures forms the logits of a tile while those of the one before go through
  // the exponentials and the second product (133k x 1203 x 100 fp16: 136 -> 125 us);
  // the others gain nothing from it, or lack the registers.
  constexpr int kLag = kKind == kFeatures && PL == 1 ? 1 : 0;
  __shared__ __attribute__((aligned(16))) char lds[kStages * (kTile + kInfo) + kTurn];

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
  const float scale2 = scale_of(a.logit_scale2, a.units);
  const int held_row = blockIdx.x * kHeldRows + wave * 32 + (lane & 31);
  const bool held_in = held_row < a.held.extent;

  // what there is to do of the features; the parts (blockIdx.y) share the streamed rows in whole tiles
  const int held_used = kKind == kTable ? a.held.extent : a.order.used(a.held.extent);
  const int stream_used = kKind == kTable ? a.order.used(a.stream.extent) : a.stream.extent;
  const bool idle = (int)(blockIdx.x * kHeldRows) >= held_used;  // none of the held rows count
  if (kKind == kForward && idle) return;
  const int64_t part = (((int64_t)stream_used + gridDim.y - 1) / gridDim.y + kTileRows - 1) / kTileRows * kTileRows;

  HeldRows<T, KB, PL> held;
  RowInfo row = {0.0f, 0.0f, 0.0f, -1};
  bool counts = held_in;
  if (kKind == kForward) {
    const int64_t target = held_in ? a.targets.at(a.order.row(held_row)) : -1;
    const int label = target >= 0 && target < a.stream.extent ? (int)target : -1;
    counts = held_in && target != a.targets.ignore;
    held.load(a.held, held_row, counts, a.dim);
    if (blockIdx.y == 0) {
      // the label's logit: the diagonal of the labels' rows against the held ones
      HeldRows<T, KB, PL> at_label;
      at_label.load(a.stream, max(label, 0), label >= 0, a.dim);
      f32x16 s;
      logits<T, KB, PL>(s, [&](int p, int k) { return at_label.v[p][k]; }, [&](int p, int k) { return held.v[p][k]; });
      const float d = diagonal(s);
      if (held_in && half == 0) a.label_dot[held_row] = scale2 < 0.0f ? -d : d;
    }
  } else if (kKind == kFeatures) {
    counts = held_in && ((a.counts[held_row >> 6] >> (held_row & 63)) & 1);
    if (held_in) row = a.info[held_row];
    held.load(a.held, held_row, counts, a.dim);
  } else {
    held.load(a.held, held_row, held_in, a.dim);
  }

  // What the lanes hold is there before the ring starts: a wait for it in the
  // loop would be one for the ring's loads as well.  (vmcnt 0, nothing else)
  constexpr int kWaitLoads = 0x0f70;
  __builtin_amdgcn_s_waitcnt(kWaitLoads);
  const int begin = (int)min((int64_t)stream_used, blockIdx.y * part);
  const int end = (int)min((int64_t)stream_used, begin + part);
  const int tiles = idle ? 0 : (end - begin + kTileRows - 1) / kTileRows;

  Stage stage;
  stage.init(a.stream, 0);
  uint64_t masks = 0;  // kTable: of 64 tiles, a lane each
  int loaded = 0;
  auto load = [&]() {
    const int first = begin + loaded * kTileRows;
    char* to = lds + (loaded % kStages) * (kTile + kInfo);
    uint64_t mask = ~0ull;
    if (kKind == kTable) {
      if ((loaded & 63) == 0) {
        masks = loaded + lane < tiles ? a.counts[(begin >> 6) + loaded + lane] : 0;
        __builtin_amdgcn_s_waitcnt(kWaitLoads);
      }
      mask = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(masks >> 32), loaded & 63) << 32 |
             (uint32_t)__builtin_amdgcn_readlane((int)masks, loaded & 63);
    }
#pragma unroll
    for (int p = 0; p < PL; ++p)
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
        stage.load(a.stream, p, first, 64 * kb, a.dim, mask, to + (p * KB + kb) * Stage::kBytes);
    if (kKind == kTable) {
      const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(
          (void*)(a.info + first), 0, (uint32_t)min(kTileRows, end - first) * 16u, 0x00020000);
      typedef __attribute__((address_space(3))) void lds_void;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_void*)(to + kTile + wave * 1024), 16, lane * 16, 0, 0, 0);
    }
    ++loaded;
  };
  // (a block past dim is loaded too: as zeros)
  constexpr int kLoads = PL * KB * Stage::kLoads + (kKind == kTable ? 1 : 0), kAhead = kStages - 1 - kLag;
#pragma unroll
  for (int t = 0; t < kAhead; ++t)
    if (t < tiles) load();

  float x = -INFINITY, sum = -1.0f;  // kForward: the largest, and the sum over all but it; see settled()
  f32x16 acc[kSums][kDBlocks];
  if (kKind != kForward) {
#pragma unroll
    for (int i = 0; i < kSums; ++i)
#pragma unroll
      for (int d = 0; d < kDBlocks; ++d) acc[i][d] = f32x16{};
  }

  auto at = [&](int t) { return (const char*)lds + (t % kStages) * (kTile + kInfo); };
  // the logits of tile t
  auto form = [&](f32x16* s, const char* __restrict__ tile) {
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      auto streamed = [&](int p, int k) {
        return Stage::template fragment<T>(tile + (p * KB + k / 4) * Stage::kBytes, 32 * b, k % 4);
      };
      auto own = [&](int p, int k) { return held.v[p][k]; };
      // the table is always x
      if (kKind == kTable) logits<T, KB, PL>(s[b], own, streamed);
      else logits<T, KB, PL>(s[b], streamed, own);
    }
  };
  // and what becomes of them
  auto use = [&](f32x16* s, const char* __restrict__ tile, const char* __restrict__ infos, int first) {
    if constexpr (kKind == kForward) {
      if (scale2 < 0.0f) {
        s[0] = -s[0];
        s[1] = -s[1];
      }
      const float scale = fabsf(scale2);
      if (first + kTileRows > end) {
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (first + 32 * b + block_m(e) + 4 * half >= end) s[b][e] = -INFINITY;
      }
      float raw = s[0][0];
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int e = 0; e < 16; ++e) raw = fmaxf(raw, s[b][e]);
      const float now = fmaxf(x, raw), top = now == -INFINITY ? 0.0f : now * scale;
      float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int e = 0; e < 16; ++e) part[e & 3] += __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][e], scale, -top));
      const float all = (part[0] + part[1]) + (part[2] + part[3]);
      if (now > x) {  // the largest so far is among these
        sum = (1.0f + sum) * __builtin_amdgcn_exp2f((x - now) * scale) + settled(now, scale, all);
        x = now;
      } else {
        sum += all * (1.0f - (now == -INFINITY ? 0.0f : __builtin_fmaf(now, scale, -top)) * kLn2f);
      }
    } else if constexpr (kKind == kFeatures) {
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          s[b][e] = row.share * __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][e], scale2, -row.top));
      const int label_at = row.target - first - 4 * half;  // from the lane's first of the tile's rows
      if (__any(label_at >= 0 && label_at < kTileRows)) {
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int e = 0; e < 16; ++e) s[b][e] = label_at == 32 * b + block_m(e) ? row.label : s[b][e];
      }
      if (first + kTileRows > end) {
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (first + 32 * b + block_m(e) + 4 * half >= end) s[b][e] = 0.0f;
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {  // 16 rows of the tile
        v8 ds[kDsPlanes];
        planes_of<T, kDsPlanes>(s[u / 2], 8 * (u & 1), ds);
#pragma unroll
        for (int d = 0; d < kDBlocks; ++d) {
          const char* block = tile + d / 2 * Stage::kBytes;
          const v8 hi = Stage::template across<T, true>(block, 32 * (d & 1), 16 * u);
          acc[0][d] = mfma(hi, ds[0], acc[0][d]);
          if constexpr (PL > 1) {
            const v8 lo = Stage::template across<T, true>(block + KB * Stage::kBytes, 32 * (d & 1), 16 * u);
            acc[1][d] = mfma(lo, ds[0], acc[1][d]);
            acc[1][d] = mfma(hi, ds[1], acc[1][d]);
            acc[2][d] = mfma(hi, ds[2], acc[2][d]);
          }
        }
      }
    } else {
      // the lane's two rows of the tile
      char* turn = lds + kStages * (kTile + kInfo) + wave * 4096;
      RowInfo r[2];
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        r[b] = *reinterpret_cast<const RowInfo*>(infos + (32 * b + (lane & 31)) * 16);
#pragma unroll
        for (int e = 0; e < 16; ++e)
          s[b][e] = r[b].share * __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][e], scale2, -r[b].top));
      }
#pragma unroll
      for (int p = 0; p < kDsPlanes; ++p) {
        // Turned over: row n of the tile at n * 64, its values 4 u .. 4 u + 3 at
        // (u ^ (n / 4 & 7)) * 8, so that neither side meets a bank twice.  A
        // wave's own LDS accesses are carried out in order.
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          const int n = 32 * b + (lane & 31), swap = (n >> 2) & 7;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            typename Pack<T>::v4 held4;
#pragma unroll
            for (int j = 0; j < 4; j += 2) {
              T pair[2];
              gs_tile::round_pair(s[b][4 * q + j], s[b][4 * q + j + 1], p + 1 < kDsPlanes, pair);
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                held4[j + i] = pair[i];
                if (p + 1 < kDsPlanes) s[b][4 * q + j + i] = gs_tile::behind(s[b][4 * q + j + i], pair[i]);
              }
            }
            *reinterpret_cast<typename Pack<T>::v4*>(turn + n * 64 + (((2 * q + half) ^ swap) << 3)) = held4;
          }
          // the label's value, by the half of the wave that holds its column
          const int at = r[b].target - (int)(blockIdx.x * kHeldRows + wave * 32);
          if (at >= 0 && at < 32 && ((at >> 2) & 1) == half) {
            const T v = (T)r[b].label;
            *reinterpret_cast<T*>(turn + n * 64 + (((at >> 2) ^ swap) << 3) + (at & 3) * 2) = v;
            if (p + 1 < kDsPlanes) r[b].label = gs_tile::behind(r[b].label, v);
          }
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {  // 16 rows of the tile
          const int j = lane & 15, group = lane >> 4, n = 16 * u + 8 * (group >> 1) + (j >> 2);
          const int unit = 4 * (group & 1) + (j & 3);
          const gs_tile::s16x4 lo4 = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              (gs_tile::lds_s16x4*)(turn + n * 64 + ((unit ^ ((n >> 2) & 7)) << 3)));
          const gs_tile::s16x4 hi4 = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              (gs_tile::lds_s16x4*)(turn + (n + 4) * 64 + ((unit ^ (((n + 4) >> 2) & 7)) << 3)));
          const gs_tile::s16x8 both = __builtin_shufflevector(lo4, hi4, 0, 1, 2, 3, 4, 5, 6, 7);
          const v8 ds = __builtin_bit_cast(v8, both);
#pragma unroll
          for (int d = 0; d < kDBlocks; ++d) {
            const char* block = tile + d / 2 * Stage::kBytes;
            const v8 hi = Stage::template across<T, false>(block, 32 * (d & 1), 16 * u);
            acc[p][d] = mfma(hi, ds, acc[p][d]);
            if constexpr (PL > 1) {
              if (p == 0)
                acc[1][d] = mfma(Stage::template across<T, false>(block + KB * Stage::kBytes, 32 * (d & 1), 16 * u), ds,
                                 acc[1][d]);
            }
          }
        }
      }
    }
  };

  auto arrive = [&](int t) {
    if (t + kAhead <= tiles) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((kAhead - 1) * kLoads) : "memory");
    else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if (loaded < tiles) load();
  };
  auto finish = [&](f32x16* s, int t) { use(s, at(t), at(t) + kTile + wave * 1024, begin + t * kTileRows); };
  f32x16 s0[2], s1[2];
  if constexpr (kLag == 0) {
    for (int t = 0; t < tiles; ++t) {
      arrive(t);
      form(s0, at(t));
      finish(s0, t);
    }
  } else {
    int t = 1;
    if (tiles > 0) {
      arrive(0);
      form(s0, at(0));
    }
    for (; t + 1 < tiles; t += 2) {
      arrive(t);
      form(s1, at(t));
      finish(s0, t - 1);
      arrive(t + 1);
      form(s0, at(t + 1));
      finish(s1, t);
    }
    if (t < tiles) {
      arrive(t);
      form(s1, at(t));
      finish(s0, t - 1);
      finish(s1, t);
    } else if (tiles > 0) {
      finish(s0, t - 1);
    }
  }

  if constexpr (kKind == kForward) {
    // the two halves of the wave hold the same rows
    const float2 other = make_float2(__shfl_xor(x, 32), __shfl_xor(sum, 32));
    const float2 all = gs_xent::joined(make_float2(x, sum), other, fabsf(scale2));
    if (held_in && half == 0) a.stats[(int64_t)blockIdx.y * a.held.extent + held_row] = all;
  } else {
    if (!held_in) return;
    const float factor = a.part_sums ? 0.0f : gs_xent::factor_of(a.alpha, a.unit);
#pragma unroll
    for (int d = 0; d < kDBlocks; ++d)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int first = 32 * d + 8 * q + 4 * half;
        float v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          v[j] = acc[0][d][4 * q + j];
          if constexpr (PL > 1)
            v[j] += (acc[1][d][4 * q + j] + acc[2][d][4 * q + j] * (1.0f / kPlaneStep)) * (1.0f / kPlaneStep);
        }
        const int64_t to_row = kKind == kFeatures && !a.part_sums ? a.order.row(held_row) : (int64_t)held_row;
        const int64_t at = to_row * a.D + first;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          v[j] = !counts ? 0.0f : a.part_sums ? v[j] : gs_xent::gradient_of<T>(v[j], factor);
        if (a.part_sums) {
          float* to = a.part_sums + (int64_t)blockIdx.y * a.part_plane + at;
          if (a.D % 4 == 0 && first < a.D) *reinterpret_cast<float4*>(to) = make_float4(v[0], v[1], v[2], v[3]);
          else
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (first + j < a.D) to[j] = v[j];
        } else {
          typedef typename std::conditional<(PL > 1), float, T>::type Out;
          Out* to = (Out*)a.out + at;
          struct __attribute__((aligned(4 * sizeof(Out)))) Four {
            Out v[4];
          };
          if (a.D % 4 == 0 && first < a.D) {
            Four f;
#pragma unroll
            for (int j = 0; j < 4; ++j) f.v[j] = (Out)v[j];
            *reinterpret_cast<Four*>(to) = f;
          } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (first + j < a.D) to[j] = (Out)v[j];
          }
        }
      }
  }
}

}  // namespace gs_resident
