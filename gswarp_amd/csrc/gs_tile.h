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
// fp32 operands are held as three bf16 planes whose sum is the value exactly
// (8 + 8 + 8 significant bits); the six products of planes that matter at fp32's
// precision (each dropped one is below 2^-26 of the product) run through the
// same kernel as six times the K steps, smallest first.  The matrix cores' own
// fp32 form has a sixteenth of the bf16 rate, so this is faster by 16 / 6.
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

// Which planes of X and Y the s-th product takes (4 bits each, low first).
__device__ __forceinline__ int product_plane(uint32_t planes, int s) { return (planes >> (4 * s)) & 15; }
constexpr uint32_t kPlanesX = 0x001012u;
constexpr uint32_t kPlanesY = 0x010210u;
constexpr int kSplitPlanes = 3;
constexpr int kSplitProducts = 6;

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

// One operand's part of a K step: BT rows (m or n) x 64 columns of K.
//
// LDS layouts (bytes), 16-byte chunks permuted so that no read or write of a
// wave meets a bank twice:
//   K contiguous: row i at i * 128, its chunk c at (c ^ ((i >> 1) & 7)) * 16:
//     the 16 rows that one phase of a 16-byte read takes lie in 16 different
//     chunks of the 256 bytes of the banks;
//   K rows: K row k at k * 2 BT, its 32-byte chunk c at (c ^ 2 (k & 3)) * 32:
//     the four K rows that the transposing load takes per 16 lanes lie apart.
template <bool kAlongK, int BT, int kThreads>
struct Stage {
  static constexpr int kVectors = BT * 8 / kThreads;  // 16-byte loads of a thread
  static constexpr int kBytes = BT * 128;
  static constexpr int kRowVectors = kAlongK ? 8 : BT / 8;
  u32x4 r[kVectors];

  // The K step at k0 of plane `plane`, rows (or columns) from i0; K and the
  // operand's extent bound what is read, and everything outside is zero.
  // row_mask (K rows only): bit k of it drops K row k0 + k when clear.
  __device__ __forceinline__ void load(const Operand& o, int plane, int i0, int64_t k0, int64_t K, uint64_t row_mask) {
    const int vec = threadIdx.x % kRowVectors;
    const int row = threadIdx.x / kRowVectors;
    constexpr int kRowStep = kThreads / kRowVectors;
    const uint16_t* base;
    uint32_t bytes;
    bool in;
    const uint32_t ld2 = (uint32_t)o.ld * 2u;
    if (kAlongK) {
      base = o.p + (int64_t)plane * o.plane + (int64_t)i0 * o.ld + k0;
      const int rows = min(BT, o.extent - i0);
      bytes = (uint32_t)(rows - 1) * ld2 + (uint32_t)min((int64_t)kBK, (K - k0 + 7) & ~7ll) * 2u;
      in = k0 + vec * 8 < K;
    } else {
      base = o.p + (int64_t)plane * o.plane + k0 * o.ld + i0;
      const int rows = (int)min((int64_t)kBK, K - k0);
      bytes = (uint32_t)(rows - 1) * ld2 + (uint32_t)min(BT, (o.extent - i0 + 7) & ~7) * 2u;
      in = i0 + vec * 8 < o.extent;
    }
    const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, bytes, 0x00020000);
#pragma unroll
    for (int j = 0; j < kVectors; ++j) {
      const int rr = row + j * kRowStep;
      uint32_t off = (uint32_t)rr * ld2 + vec * 16u;
      bool use = in;
      if (!kAlongK) use = use && ((row_mask >> rr) & 1);
      r[j] = __builtin_amdgcn_raw_buffer_load_b128(rsrc, use ? off : kOutOfRange, 0, 0);
    }
  }

  __device__ __forceinline__ void store(char* lds) const {
    const int vec = threadIdx.x % kRowVectors;
    const int row = threadIdx.x / kRowVectors;
    constexpr int kRowStep = kThreads / kRowVectors;
#pragma unroll
    for (int j = 0; j < kVectors; ++j) {
      const int rr = row + j * kRowStep;
      int at;
      if (kAlongK) at = rr * 128 + ((vec ^ ((rr >> 1) & 7)) << 4);
      else at = rr * (BT * 2) + ((((vec >> 1) ^ (2 * (rr & 3))) << 5) | ((vec & 1) << 4));
      *reinterpret_cast<u32x4*>(lds + at) = r[j];
    }
  }

  // Matrix-core operand of 32 rows from i (a multiple of 32) and K columns
  // 16 ks .. 16 ks + 15 of the step: lane l holds row l % 32, columns 8 (l / 32) ..+7.
  template <typename T>
  static __device__ __forceinline__ typename Pack<T>::v8 fragment(const char* lds, int i, int ks) {
    const int lane = threadIdx.x & 63;
    if (kAlongK) {
      const int row = i + (lane & 31);
      const int c = 2 * ks + (lane >> 5);
      return *reinterpret_cast<const typename Pack<T>::v8*>(lds + row * 128 + ((c ^ ((row >> 1) & 7)) << 4));
    } else {
      // The transposing load: in each group of 16 lanes, lane j gives the
      // address of 4 values of K row j / 4 and gets the 4 K rows of column j.
      const int j = lane & 15, group = lane >> 4;
      const int k = 16 * ks + 8 * (group >> 1) + (j >> 2);
      const int m = i + 16 * (group & 1);
      const char* at = lds + k * (BT * 2) + (((m >> 4) ^ (2 * (k & 3))) << 5) + (j & 3) * 8;
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)at);
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(at + 4 * BT * 2));
      const s16x8 both = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
      return __builtin_bit_cast(typename Pack<T>::v8, both);
    }
  }
};

// The tile shape: kWavesM x kWavesN waves, each (BM / kWavesM) x (BN / kWavesN).
template <int kBM, int kBN, int kWavesM_, int kWavesN_>
struct Shape {
  static constexpr int BM = kBM, BN = kBN;
  static constexpr int kWavesM = kWavesM_, kWavesN = kWavesN_;
  static constexpr int kThreads = 64 * kWavesM * kWavesN;
  static constexpr int kWaveM = BM / kWavesM, kWaveN = BN / kWavesN;
  static constexpr int kMB = kWaveM / 32, kNB = kWaveN / 32;
  static constexpr int kLdsBytes = 2 * (BM + BN) * 128;
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

// acc = the tile at (m0, n0), over K columns [k_begin, k_end) of products
// `products` (1, or 6 for fp32 planes).  Every element outside the operands
// counts as zero.  x_rows (X in K rows only, may be null): one bit per K row
// (k_begin on a multiple of 64); rows whose bit is clear count as zero whatever
// they hold.  lds: S::kLdsBytes, free for the caller after a barrier.
//
// Two LDS buffers: the loads of step t + 1 are in flight (in registers) while
// the matrix cores work on step t; one barrier per step.
template <class S, typename T, bool kXAlongK, bool kYAlongK>
__device__ __forceinline__ void product(Accumulators<S>& acc, const Operand& x, const Operand& y, int m0, int n0,
                                        int64_t k_begin, int64_t k_end, int products, const uint64_t* x_rows,
                                        char* lds) {
  typedef Stage<kXAlongK, S::BM, S::kThreads> StageX;
  typedef Stage<kYAlongK, S::BN, S::kThreads> StageY;
#pragma unroll
  for (int a = 0; a < S::kMB; ++a)
#pragma unroll
    for (int b = 0; b < S::kNB; ++b) acc.c[a][b] = f32x16{};
  const int steps = (int)((k_end - k_begin + kBK - 1) / kBK);
  const int total = steps * products;
  if (total <= 0) return;
  StageX sx;
  StageY sy;
  int step = 0, prod = 0;
  auto load = [&]() {
    const int64_t k0 = k_begin + (int64_t)step * kBK;
    const int px = products == 1 ? 0 : product_plane(kPlanesX, prod);
    const int py = products == 1 ? 0 : product_plane(kPlanesY, prod);
    const uint64_t mask = (!kXAlongK && x_rows) ? x_rows[k0 / kBK] : ~0ull;
    sx.load(x, px, m0, k0, k_end, mask);
    sy.load(y, py, n0, k0, k_end, ~0ull);
    if (++step == steps) {
      step = 0;
      ++prod;
    }
  };
  constexpr int kBuffer = StageX::kBytes + StageY::kBytes;
  load();
  sx.store(lds);
  sy.store(lds + StageX::kBytes);
  __syncthreads();
  const int wm = wave_m<S>(), wn = wave_n<S>();
  for (int t = 0; t < total; ++t) {
    const bool more = t + 1 < total;
    if (more) load();
    const char* lx = lds + (t & 1) * kBuffer;
    const char* ly = lx + StageX::kBytes;
#pragma unroll
    for (int ks = 0; ks < kBK / 16; ++ks) {
      typename Pack<T>::v8 fx[S::kMB], fy[S::kNB];
#pragma unroll
      for (int a = 0; a < S::kMB; ++a) fx[a] = StageX::template fragment<T>(lx, wm + 32 * a, ks);
#pragma unroll
      for (int b = 0; b < S::kNB; ++b) fy[b] = StageY::template fragment<T>(ly, wn + 32 * b, ks);
#pragma unroll
      for (int a = 0; a < S::kMB; ++a)
#pragma unroll
        for (int b = 0; b < S::kNB; ++b) acc.c[a][b] = mfma(fx[a], fy[b], acc.c[a][b]);
    }
    if (more) {
      char* next = lds + ((t + 1) & 1) * kBuffer;
      sx.store(next);
      sy.store(next + StageX::kBytes);
    }
    __syncthreads();
  }
}

}  // namespace gs_tile
