// Tiled matrix products on the matrix cores, shared by the vocabulary kernels.
//
// A workgroup computes out(m, n) = sum_k X(m, k) Y(n, k) for a BM x BN tile in
// fp32 accumulators.  The operands hold 16-bit values (bf16 or fp16) and each
// comes in one of two layouts:
//   K contiguous: element (i, k) at p[i * ld + k] (a matrix read along its rows);
//   K rows:       element (i, k) at p[k * ld + i] (the transposed read), turned
//                 on its way from LDS to registers by the transposing LDS load.
// So the three products of the cross entropy (features x table for the logits,
// and the two gradients) read the same row-major matrices, and nothing is ever
// transposed in memory.
//
// fp32 operands are held as fp16 planes, hi + lo / 2^11, of the values times a
// power of two that brings the matrix's largest magnitude to 2^13..2^14 (its
// unit; the results are multiplied by it).  Together they have 22 bits, down to
// 2^-28 of the largest magnitude, and below it an error of 2^-50 of that.  Three
// products of planes (lo hi and hi lo, whose sum is then divided by 2^11, and hi
// hi; lo lo is below 2^-24 of the product, as fp32's own rounding) run through
// the same kernel as three times the K steps.  The matrix cores' own fp32 form
// has a sixteenth of the fp16 rate, so this is faster by 16 / 3.  An operand Y of
// wider range (gradients of the logits: probabilities) adds a third plane, + tiny / 2^22, and a fourth product.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace gs_tile {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

constexpr int kBK = 64;  // K columns of a step: 128 bytes of a row
// Buffer offsets are 32-bit and the ones used as "out of range" start at 2^31:
// a tile's rows must span less than that.
constexpr int64_t kMaxLd = 1 << 21;
constexpr uint32_t kOutOfRange = 0x80000000u;

// A matrix operand.  extent: how many m (or n) there are; plane: elements
// between the planes of an fp32 operand.
struct Operand {
  const uint16_t* p;
  int64_t ld;
  int64_t plane;
  int32_t extent;
};

constexpr int kSplitPlanes = 2, kWidePlanes = 3;      // of an fp32 operand, of one of wide range
constexpr int kSplitProducts = 3, kWideProducts = 4;  // of two fp32 operands, with a wide Y
constexpr int kFinePlanes = 2, kFineProducts = 2;     // of a 16-bit X and a Y that is held more finely
constexpr float kPlaneStep = 2048.0f;                 // what each plane is held times more than the one before
// What is left of v behind its plane h, for the next one: exact, and two
// instructions (the second takes h in 16 bits).
__device__ __forceinline__ float behind(float v, _Float16 h) {
  return __builtin_fmaf((float)h, -kPlaneStep, v * kPlaneStep);
}
__device__ __forceinline__ float behind(float v, __bf16 h) {
  return __builtin_fmaf((float)h, -kPlaneStep, v * kPlaneStep);
}
// The planes of X and Y that product s of `products` takes: (hi, tiny) if there are
// four, (lo, hi), (hi, lo), (hi, hi); of two, the last two.  Before (lo, hi), if not the first, and
// before (hi, hi) the sums so far are divided by a step.
__device__ __forceinline__ int plane_x(int products, int s) { return products > 1 && s == products - 3; }
__device__ __forceinline__ int plane_y(int products, int s) {
  return products == 1 ? 0 : s == products - 2 ? 1 : s == products - 4 ? 2 : 0;
}
__device__ __forceinline__ bool steps_down(int products, int s) {
  return (s > 0 && s == products - 3) || (products > 1 && s == products - 1);
}

__device__ __forceinline__ f32x16 mfma(bf16x8 a, bf16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mfma(f16x8 a, f16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
template <typename T>
struct Pack;
template <>
struct Pack<__bf16> {
  typedef bf16x8 v8;
  typedef bf16x4 v4;
};
template <>
struct Pack<_Float16> {
  typedef f16x8 v8;
  typedef f16x4 v4;
};

// Two values in 16 bits.  As planes go on from what was rounded, the compiler would
// round for that once more, one by one, if it saw where the pair comes from.
template <typename T>
__device__ __forceinline__ void round_pair(float a, float b, bool goes_on, T* out) {
  typedef T pair __attribute__((ext_vector_type(2)));
  typedef float floats __attribute__((ext_vector_type(2)));
  uint32_t bits = __builtin_bit_cast(uint32_t, __builtin_convertvector(floats{a, b}, pair));
  if (goes_on) asm("" : "+v"(bits));
  const pair p = __builtin_bit_cast(pair, bits);
  out[0] = p[0];
  out[1] = p[1];
}

// One operand's part of a K step, BT rows (m or n) x 64 columns of K, loaded
// straight into LDS: each load instruction of a wave fills 1024 bytes, lane l
// the 16 bytes at 16 l, so the arrangement in LDS is made by the choice of what
// each lane reads.
//
// LDS layouts (bytes), 16-byte chunks permuted so that no read of a wave meets a
// bank twice:
//   K contiguous: row i at i * 128, its chunk c at (c ^ spread(i)) * 16: the 16
//     rows that one phase of a 16-byte read takes lie in 16 different chunks of
//     the 256 bytes of the banks, and so do four rows of 64 bytes, which a
//     transposing read takes;
//   K rows: K row k at k * 2 BT, its 32-byte chunk c at (c ^ turn(k)) * 32: the
//     four K rows that the transposing load takes per 16 lanes lie apart.
template <bool kAlongK, int BT, int kWaves>
struct Stage {
  static constexpr int kBytes = BT * 128;
  static constexpr int kLoads = kBytes / 1024 / kWaves;         // load instructions of a wave
  static constexpr int kRowVectors = kAlongK ? 8 : BT / 8;      // 16-byte chunks of a row of the layout
  static constexpr int kLoadRows = 64 / kRowVectors;            // rows of the layout that an instruction fills
  static_assert(kLoads * kWaves * 1024 == kBytes, "every wave issues the same loads");
  static_assert(kAlongK || BT >= 128, "the four K rows of a transposing load need four chunks to lie apart in");

  static __device__ __forceinline__ int spread(int i) { return ((i >> 2) & 3) | ((i << 1) & 4); }
  static __device__ __forceinline__ int turn(int k) { return 2 * (k & 3); }

  // Byte offsets of the lane's chunk from the step's first element, for
  // instructions of even and of odd number (the permutation repeats every two).
  uint32_t offset[2];
  int32_t chunk[2];  // the chunk's number in its row (K contiguous)

  __device__ __forceinline__ void init(const Operand& o, int i0) {
    const int lane = threadIdx.x & 63;
    const int row = lane / kRowVectors, at = lane % kRowVectors;
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const int r = p * kLoadRows + row;
      if (kAlongK) chunk[p] = at ^ spread(r);
      else chunk[p] = (((at >> 1) ^ turn(r)) << 1) | (at & 1);
      offset[p] = (uint32_t)row * (uint32_t)o.ld * 2u + chunk[p] * 16u;
      if (!kAlongK && i0 + chunk[p] * 8 >= o.extent) offset[p] = kOutOfRange;
    }
  }

  // Starts the loads of the K step at k0 of plane `plane` into lds; K and the
  // operand's extent bound what is read, and everything outside is zero.
  // row_mask: row r of the layout (of the tile, or K row k0 + r) counts as zero where bit r is clear.
  __device__ __forceinline__ void load(const Operand& o, int plane, int i0, int32_t k0, int32_t K, uint64_t row_mask,
                                       char* __restrict__ lds) const {
    typedef __attribute__((address_space(3))) void lds_void;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t ld2 = (uint32_t)o.ld * 2u;
    const uint16_t* base;
    uint32_t bytes, off[2] = {offset[0], offset[1]};
    if (kAlongK) {
      base = o.p + (int64_t)plane * o.plane + (int64_t)i0 * o.ld + k0;
      const int left = K - k0;
      bytes = (uint32_t)(min(BT, o.extent - i0) - 1) * ld2 + (uint32_t)min(kBK, (left + 7) & ~7) * 2u;
      if (left < kBK) {
#pragma unroll
        for (int p = 0; p < 2; ++p)
          if (chunk[p] * 8 >= left) off[p] = kOutOfRange;
      }
    } else {
      base = o.p + (int64_t)plane * o.plane + (int64_t)k0 * o.ld + i0;
      bytes = (uint32_t)(min(kBK, K - k0) - 1) * ld2 + (uint32_t)min(BT, (o.extent - i0 + 7) & ~7) * 2u;
    }
    const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, bytes, 0x00020000);
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
      const int number = wave * kLoads + j;
      uint32_t at = off[number & 1] + (uint32_t)(number * kLoadRows) * ld2;
      if (row_mask != ~0ull) {
        const int k = number * kLoadRows + (threadIdx.x & 63) / kRowVectors;
        if (!((row_mask >> k) & 1)) at = kOutOfRange;
      }
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_void*)(lds + number * 1024), 16, at, 0, 0, 0);
    }
  }

  // The other way round (K contiguous, BT rows x 64 columns): operand of 32
  // columns from i and the 16 rows from r0 as K, in their order, or (kHalves) as
  // accumulators hold them: rows 0-3 and 8-11 in the lower half of the wave, 4-7 and 12-15 in the upper.
  template <typename T, bool kHalves>
  static __device__ __forceinline__ typename Pack<T>::v8 across(const char* __restrict__ lds, int i, int r0) {
    const int lane = threadIdx.x & 63;
    const int j = lane & 15, group = lane >> 4;
    const int c = i + 16 * (group & 1) + 4 * (j & 3);
    const int lo_row = r0 + (kHalves ? 4 : 8) * (group >> 1) + (j >> 2), hi_row = lo_row + (kHalves ? 8 : 4);
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (lds_s16x4*)(lds + lo_row * 128 + (((c >> 3) ^ spread(lo_row)) << 4) + (c & 4) * 2));
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (lds_s16x4*)(lds + hi_row * 128 + (((c >> 3) ^ spread(hi_row)) << 4) + (c & 4) * 2));
    const s16x8 both = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    return __builtin_bit_cast(typename Pack<T>::v8, both);
  }

  // Matrix-core operand of 32 rows from i (a multiple of 32) and K columns
  // 16 ks .. 16 ks + 15 of the step: lane l holds row l % 32, columns 8 (l / 32) ..+7.
  template <typename T>
  static __device__ __forceinline__ typename Pack<T>::v8 fragment(const char* __restrict__ lds, int i, int ks) {
    const int lane = threadIdx.x & 63;
    if (kAlongK) {
      const int row = i + (lane & 31);
      const int c = 2 * ks + (lane >> 5);
      return *reinterpret_cast<const typename Pack<T>::v8*>(lds + row * 128 + ((c ^ spread(row)) << 4));
    } else {
      // The transposing load: in each group of 16 lanes, lane j gives the
      // address of 4 values of K row j / 4 and gets the 4 K rows of column j.
      const int j = lane & 15, group = lane >> 4;
      const int k = 16 * ks + 8 * (group >> 1) + (j >> 2);
      const int m = i + 16 * (group & 1);
      const char* at = lds + k * (BT * 2) + (((m >> 4) ^ turn(k)) << 5) + (j & 3) * 8;
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)at);
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(at + 4 * BT * 2));
      const s16x8 both = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
      return __builtin_bit_cast(typename Pack<T>::v8, both);
    }
  }
};

// The tile shape: kWavesM x kWavesN waves, each (BM / kWavesM) x (BN / kWavesN),
// kStages steps of K in LDS.
template <int kBM, int kBN, int kWavesM_, int kWavesN_, int kStages_ = 2>
struct Shape {
  static constexpr int BM = kBM, BN = kBN;
  static constexpr int kWavesM = kWavesM_, kWavesN = kWavesN_, kStages = kStages_;
  static constexpr int kWaves = kWavesM * kWavesN, kThreads = 64 * kWaves;
  static constexpr int kWaveM = BM / kWavesM, kWaveN = BN / kWavesN;
  static constexpr int kMB = kWaveM / 32, kNB = kWaveN / 32;
  static constexpr int kLdsBytes = kStages * (BM + BN) * 128;
};

// The accumulators of a wave.  Block (a, b) covers rows m = wave_m + 32 a and
// columns n = wave_n + 32 b on; of it lane l holds column l % 32 and, in
// element 4 q + j, row 8 q + 4 (l / 32) + j: four consecutive m for each q.
template <class S>
struct Accumulators {
  f32x16 c[S::kMB][S::kNB];
};
template <class S>
__device__ __forceinline__ int wave_m() {
  return (threadIdx.x >> 6) / S::kWavesN * S::kWaveM;
}
template <class S>
__device__ __forceinline__ int wave_n() {
  return (threadIdx.x >> 6) % S::kWavesN * S::kWaveN;
}

// acc += the step held at lds.  The fragments of 16 columns of K are read while
// the matrix cores work on the 16 before.
template <class S, typename T, class StageX, class StageY>
__device__ __forceinline__ void multiply(Accumulators<S>& acc, int wm, int wn, const char* __restrict__ lds) {
  typename Pack<T>::v8 fx[2][S::kMB], fy[2][S::kNB];
  auto read = [&](int ks) {
#pragma unroll
    for (int a = 0; a < S::kMB; ++a) fx[ks & 1][a] = StageX::template fragment<T>(lds, wm + 32 * a, ks);
#pragma unroll
    for (int b = 0; b < S::kNB; ++b)
      fy[ks & 1][b] = StageY::template fragment<T>(lds + StageX::kBytes, wn + 32 * b, ks);
  };
  read(0);
#pragma unroll
  for (int ks = 0; ks < kBK / 16; ++ks) {
    if (ks + 1 < kBK / 16) read(ks + 1);
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int a = 0; a < S::kMB; ++a)
#pragma unroll
      for (int b = 0; b < S::kNB; ++b) acc.c[a][b] = mfma(fx[ks & 1][a], fy[ks & 1][b], acc.c[a][b]);
    __builtin_amdgcn_s_setprio(0);
    __builtin_amdgcn_sched_barrier(0);
  }
}

// acc = the tile at (m0, n0), over K columns [k_begin, k_end) of
// `products` products of planes (1 to 4).  Every element outside the operands
// counts as zero.  x_rows (X in K rows only, may be null): one bit per K row
// (k_begin on a multiple of 64); rows whose bit is clear count as zero whatever
// they hold.  lds: S::kLdsBytes, free for the caller after a barrier.
//
// LDS holds a ring of kStages steps: while the matrix cores work on step t, the
// loads of the kStages - 1 steps behind it are on their way into the ring; one
// barrier per step, passed when the wave's own loads of step t have arrived.
template <class S, typename T, bool kXAlongK, bool kYAlongK>
__device__ __forceinline__ void product(Accumulators<S>& acc, const Operand& x, const Operand& y, int m0, int n0,
                                        int32_t k_begin, int32_t k_end, int products, const uint64_t* x_rows,
                                        char* lds) {
  typedef Stage<kXAlongK, S::BM, S::kWaves> StageX;
  typedef Stage<kYAlongK, S::BN, S::kWaves> StageY;
#pragma unroll
  for (int a = 0; a < S::kMB; ++a)
#pragma unroll
    for (int b = 0; b < S::kNB; ++b) acc.c[a][b] = f32x16{};
  const int steps = (k_end - k_begin + kBK - 1) / kBK;
  const int total = steps * products;
  if (total <= 0) return;
  StageX sx;
  StageY sy;
  sx.init(x, m0);
  sy.init(y, n0);
  int step = 0, prod = 0;
  constexpr int kBuffer = StageX::kBytes + StageY::kBytes;
  // the masks of 64 steps, a lane each
  uint64_t masks = 0;
  const bool masked = !kXAlongK && x_rows;
  auto load = [&](char* to) {
    const int32_t k0 = k_begin + step * kBK;
    const int px = plane_x(products, prod), py = plane_y(products, prod);
    uint64_t mask = ~0ull;
    if (masked) {
      if ((step & 63) == 0) {
        const int at = step + (threadIdx.x & 63);
        masks = at < steps ? x_rows[k_begin / kBK + at] : 0;
      }
      mask = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(masks >> 32), step & 63) << 32 |
             (uint32_t)__builtin_amdgcn_readlane((int)masks, step & 63);
    }
    sx.load(x, px, m0, k0, k_end, mask, to);
    sy.load(y, py, n0, k0, k_end, ~0ull, to + StageX::kBytes);
    if (++step == steps) {
      step = 0;
      ++prod;
    }
  };
  constexpr int kAhead = S::kStages - 1, kLoads = StageX::kLoads + StageY::kLoads;
  static_assert(S::kStages == 2 || (kXAlongK && kYAlongK), "the masks' loads would count among the steps'");
  int to = 0;  // the stage that the next loads fill
#pragma unroll
  for (int t = 0; t < kAhead; ++t)
    if (t < total) {
      load(lds + to * kBuffer);
      to = to + 1 == S::kStages ? 0 : to + 1;
    }
  const int wm = wave_m<S>(), wn = wave_n<S>();
  int at = 0, product_at = 0, next = 0;
  for (int t = 0; t < total; ++t) {
    // loads return in order: at most those of the steps behind step t may be under
    // way; and the reads of the stage that is filled next are over
    if (t + kAhead <= total) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((kAhead - 1) * kLoads) : "memory");
    else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if (t + kAhead < total) {
      load(lds + to * kBuffer);
      to = to + 1 == S::kStages ? 0 : to + 1;
    }
    if (t == next) {  // the first step of a product
      if (steps_down(products, product_at)) {
#pragma unroll
        for (int a = 0; a < S::kMB; ++a)
#pragma unroll
          for (int b = 0; b < S::kNB; ++b) acc.c[a][b] *= 1.0f / kPlaneStep;
      }
      ++product_at;
      next += steps;
    }
    multiply<S, T, StageX, StageY>(acc, wm, wn, lds + at * kBuffer);
    at = at + 1 == S::kStages ? 0 : at + 1;
  }
  __syncthreads();
}

// The tile of a block: blocks go to the 8 XCDs (each with an L2 of its own) in
// turn, so each XCD is given a run of consecutive tiles, in bands of 8 tiles
// of m, m first inside a band: tiles that run side by side share operands.  Those
// from used_n on have nothing to multiply and come last.
struct TileAt {
  int m, n;
};
__device__ __forceinline__ TileAt tile_at(int tiles_m, int used_n) {
  const int total = tiles_m * used_n;
  if ((int)blockIdx.x >= total) {
    const int rest = blockIdx.x - total;
    return {rest % tiles_m, used_n + rest / tiles_m};
  }
  const int id = blockIdx.x, q = total / 8, r = total % 8, xcd = id % 8;
  const int t = xcd * q + min(xcd, r) + id / 8;
  const int band = t / (8 * used_n);
  const int height = min(8, tiles_m - 8 * band), in = t - band * 8 * used_n;
  return {8 * band + in % height, in / height};
}

}  // namespace gs_tile
