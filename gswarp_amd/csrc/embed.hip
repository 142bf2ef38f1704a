// Rows of a shared table looked up by token, and the table's gradient.
//
//   out[i, :] = scale table[t_i, :]
//   grad_table[v, :] = scale sum_{i: t_i = v} grad_out[i, :]
//
// The gradient is a sum over positions of equal token: the positions are sorted
// stably by token, and runs of equal tokens are summed in position order.  The
// sorted list is cut into groups of equal length whatever the runs are, so a
// token that holds most positions costs no more than a flat distribution: a
// group writes the rows of the runs that lie inside it, and hands the (at most
// two) that go on past its ends, as fp32 sums, to a next level that treats them
// as a sorted list in turn, 2 entries for each group.  The order of every sum
// is fixed by the tokens alone: no atomics, the same bits every time.
#include "gs_capi.h"

namespace gs_embed {

typedef unsigned u32;
constexpr u32 kNone = 0xffffffffu;  // an entry that holds nothing
constexpr int kThreads = 256;

static inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
static inline int64_t round_up(int64_t a, int64_t b) { return ceil_div(a, b) * b; }

struct Tokens {
  const void* p;
  int bits;
  __device__ __forceinline__ int64_t at(int64_t i) const {
    return bits == 64 ? ((const int64_t*)p)[i] : (int64_t)((const int32_t*)p)[i];
  }
};

template <typename T, int V>
struct __attribute__((aligned(sizeof(T) * V))) Vec {
  T v[V];
};

// ------------------------------------------------------------------ forward
// A thread moves kItems vectors of V elements, a block's vectors apart.
constexpr int kItems = 4;
template <typename T, int V>
__global__ __launch_bounds__(kThreads) void lookup_kernel(Tokens tokens, int64_t n, u32 vocab, u32 row_vectors,
                                                          const T* __restrict__ table, int64_t ld, float scale,
                                                          T* __restrict__ out) {
  // the block's first vector as (position, vector of its row); the threads' vectors follow in 32 bits
  const int64_t first = (int64_t)blockIdx.x * (kThreads * kItems);
  const int64_t row0 = first / row_vectors;
  const u32 rest = (u32)(first - row0 * row_vectors);
#pragma unroll
  for (int j = 0; j < kItems; ++j) {
    const u32 at = rest + threadIdx.x + j * kThreads;
    const u32 r = at / row_vectors, c = at - r * row_vectors;
    const int64_t row = row0 + r;
    if (row >= n) break;
    const int64_t t = tokens.at(row);
    Vec<T, V> x;
    if (t >= 0 && t < vocab) {
      x = *reinterpret_cast<const Vec<T, V>*>(table + t * ld + (int64_t)c * V);
      if (scale != 1.0f)
#pragma unroll
        for (int e = 0; e < V; ++e) x.v[e] = (T)((float)x.v[e] * scale);
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) x.v[e] = (T)__builtin_nanf("");
    }
    *reinterpret_cast<Vec<T, V>*>(out + (first + threadIdx.x + j * kThreads) * V) = x;
  }
}

// ------------------------------------------------------------------ gradient
// Sort input: the token, or vocab (sorted last, never read) where there is no gradient.
__global__ __launch_bounds__(kThreads) void keys_kernel(Tokens tokens, int64_t n, u32 vocab, int64_t padding,
                                                        u32* __restrict__ keys, int* __restrict__ positions) {
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < n; i += (int64_t)gridDim.x * kThreads) {
    const int64_t t = tokens.at(i);
    keys[i] = t >= 0 && t < vocab && t != padding ? (u32)t : vocab;
    positions[i] = (int)i;
  }
}

// Sums the runs of one level.  Entry e of n has key keys[e] (>= vocab: nothing)
// and its row at src + (positions ? positions[e] : e) * ld.  A group of `lanes`
// lanes takes entries [g length, (g + 1) length), lane l columns (blockIdx.y lanes + l) V on.
// next_keys / next (2 a group, rows of next_ld): the runs that go on past the
// group's ends, entry 2 g the one that comes in from the left, 2 g + 1 the one that only goes out to the right.
template <typename S, typename T, int V>
__global__ __launch_bounds__(kThreads) void runs_kernel(const u32* __restrict__ keys, const int* __restrict__ positions,
                                                        int64_t n, u32 vocab, const S* __restrict__ src, int64_t ld,
                                                        int D, int lanes, int length, float scale,
                                                        T* __restrict__ out, u32* __restrict__ next_keys,
                                                        float* __restrict__ next, int64_t next_ld) {
  constexpr int kBatch = 8;  // rows in flight
  const int lane = threadIdx.x % lanes;
  const int64_t g = (int64_t)blockIdx.x * (kThreads / lanes) + threadIdx.x / lanes;
  const int64_t begin = g * length;
  if (begin >= n) return;
  const int64_t end = min(n, begin + length);
  const int col = (blockIdx.y * lanes + lane) * V;
  const bool in = col < D;

  // the last key before the group: of the two entries before it, the second may be empty
  u32 before = kNone;
  if (begin > 0) {
    before = keys[begin - 1];
    if (before >= vocab && begin > 1) before = keys[begin - 2];
  }
  const u32 after = end < n ? keys[end] : kNone;

  u32 head_key = kNone, tail_key = kNone;
  u32 cur = kNone;
  bool from_left = false;
  float acc[V];
#pragma unroll
  for (int e = 0; e < V; ++e) acc[e] = 0.0f;

  auto to_next = [&](int slot) {
    if (!in) return;
    float* o = next + (2 * g + slot) * next_ld + col;
#pragma unroll
    for (int e = 0; e < V; ++e) o[e] = acc[e];
  };
  auto flush = [&](bool goes_on) {
    if (cur >= vocab) return;
    if (from_left) {
      head_key = cur;
      to_next(0);
    } else if (goes_on) {
      tail_key = cur;
      to_next(1);
    } else if (in) {
      Vec<T, V> x;
#pragma unroll
      for (int e = 0; e < V; ++e) x.v[e] = (T)(acc[e] * scale);
      *reinterpret_cast<Vec<T, V>*>(out + (int64_t)cur * D + col) = x;
    }
  };

  for (int64_t e0 = begin; e0 < end; e0 += kBatch) {
    u32 k[kBatch];
    Vec<S, V> x[kBatch];
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      k[j] = e0 + j < end ? keys[e0 + j] : kNone;
      if (k[j] < vocab && in) {
        const int64_t row = positions ? (int64_t)positions[e0 + j] : e0 + j;
        x[j] = *reinterpret_cast<const Vec<S, V>*>(src + row * ld + col);
      }
    }
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      if (k[j] >= vocab) continue;
      if (k[j] != cur) {
        flush(false);
        from_left = cur == kNone && before == k[j];
        cur = k[j];
#pragma unroll
        for (int e = 0; e < V; ++e) acc[e] = 0.0f;
      }
      if (in)
#pragma unroll
        for (int e = 0; e < V; ++e) acc[e] += (float)x[j].v[e];
    }
  }
  flush(cur == after);
  if (lane == 0 && blockIdx.y == 0 && next_keys) {
    next_keys[2 * g] = head_key;
    next_keys[2 * g + 1] = tail_key;
  }
}

// Zeros in the rows that no sorted key names: a wave looks 64 rows up, a lane each, by bisection.
template <typename T>
__global__ __launch_bounds__(kThreads) void absent_kernel(const u32* __restrict__ keys, int64_t n, u32 vocab, int D,
                                                          T* __restrict__ out) {
  const int lane = threadIdx.x & 63;
  const int64_t row0 = ((int64_t)blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6)) * 64;
  const int64_t v = row0 + lane;
  bool absent = false;
  if (v < vocab) {
    int64_t lo = 0, hi = n;  // the first key >= v lies in [lo, hi]
    while (lo < hi) {
      const int64_t mid = (lo + hi) >> 1;
      if (keys[mid] < (u32)v) lo = mid + 1;
      else hi = mid;
    }
    absent = lo == n || keys[lo] != (u32)v;
  }
  for (uint64_t left = __ballot(absent); left; left &= left - 1) {
    T* o = out + (row0 + __builtin_ctzll(left)) * D;
    for (int c = lane; c < D; c += 64) o[c] = (T)0.0f;
  }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void zero_kernel(T* __restrict__ out, int64_t n) {
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < n; i += (int64_t)gridDim.x * kThreads)
    out[i] = (T)0.0f;
}

// ------------------------------------------------------------------ host
// Elements of a vector access: 16 bytes where the rows allow it, else two or one elements.
template <typename T>
static int vector_of(int64_t D, int64_t ld, const void* a, const void* b) {
  auto fits = [&](int v) {
    const uintptr_t bytes = sizeof(T) * v;
    return D % v == 0 && ld % v == 0 && (uintptr_t)a % bytes == 0 && (uintptr_t)b % bytes == 0;
  };
  const int most = 16 / (int)sizeof(T);
  return fits(most) ? most : fits(2) ? 2 : 1;
}

template <typename T, int V>
static int lookup(int64_t n, int32_t vocab, int32_t dim, Tokens tokens, const T* table, int64_t ld, float scale, T* out,
                  hipStream_t s) {
  const int64_t vectors = n * (dim / V);
  const int64_t blocks = ceil_div(vectors, kThreads * kItems);
  if (blocks > 0x7fffffffll) return GS_ERR_OVERFLOW;
  lookup_kernel<T, V><<<(unsigned)blocks, kThreads, 0, s>>>(tokens, n, (u32)vocab, (u32)(dim / V), table, ld, scale, out);
  return gs_status_from_hip(hipGetLastError());
}

template <typename T>
static int forward(int64_t n, int32_t vocab, int32_t dim, Tokens tokens, const void* table, int64_t ld, float scale,
                   void* out, hipStream_t s) {
  const int v = vector_of<T>(dim, ld, table, out);
  if (v == 16 / (int)sizeof(T)) return lookup<T, 16 / sizeof(T)>(n, vocab, dim, tokens, (const T*)table, ld, scale, (T*)out, s);
  if (v == 2) return lookup<T, 2>(n, vocab, dim, tokens, (const T*)table, ld, scale, (T*)out, s);
  return lookup<T, 1>(n, vocab, dim, tokens, (const T*)table, ld, scale, (T*)out, s);
}

// Entries of a group: on the first level 8 to 64, by how many positions there are
// to fill the chip with; 64 above.
static int group_length(int64_t n, int level) {
  if (level > 0) return 64;
  int length = 8;
  while (length < 64 && n / length > 16384) length *= 2;
  return length;
}

struct BackwardPlan {
  u32 *keys, *keys_alt, *next_keys[2];
  int *positions, *positions_alt;
  float* next[2];
  int64_t next_ld;
  char* sort_scratch;
  size_t sort_bytes, bytes;

  BackwardPlan(int64_t n, int32_t dim, void* ws) {
    char* base = (char*)ws;
    size_t at = 0;
    auto take = [&](int64_t size) {
      char* p = base ? base + at : nullptr;
      at += (size_t)round_up(size, 256);
      return p;
    };
    next_ld = round_up(dim, 8);
    sort_bytes = gs_sort_scratch_bytes(n);
    keys = (u32*)take(n * 4);
    keys_alt = (u32*)take(n * 4);
    positions = (int*)take(n * 4);
    positions_alt = (int*)take(n * 4);
    sort_scratch = take((int64_t)sort_bytes);
    // the levels' entries, in turn in two places
    int64_t entries = n;
    for (int level = 0; level < 2; ++level) {
      entries = entries > 0 ? 2 * ceil_div(entries, group_length(entries, level)) : 0;
      next_keys[level] = (u32*)take(entries * 4);
      next[level] = (float*)take(entries * next_ld * 4);
    }
    bytes = at;
  }
};

template <typename S, typename T, int V>
static void runs(const u32* keys, const int* positions, int64_t n, int32_t vocab, const S* src, int64_t ld, int D,
                 int length, float scale, T* out, u32* next_keys, float* next, int64_t next_ld, hipStream_t s) {
  int lanes = 1;
  while (lanes < 64 && lanes * V < D) lanes *= 2;
  const dim3 grid((unsigned)ceil_div(ceil_div(n, length), kThreads / lanes), (unsigned)ceil_div(D, lanes * V));
  runs_kernel<S, T, V><<<grid, kThreads, 0, s>>>(keys, positions, n, (u32)vocab, src, ld, D, lanes, length, scale, out,
                                                 next_keys, next, next_ld);
}

template <typename T, int V>
static int gradient(int64_t n, int32_t vocab, int32_t dim, Tokens tokens, const T* grad, float scale, int64_t padding,
                    T* out, const BackwardPlan& b, hipStream_t s) {
  keys_kernel<<<(unsigned)min(ceil_div(n, kThreads), (int64_t)8192), kThreads, 0, s>>>(tokens, n, (u32)vocab, padding,
                                                                                     b.keys, b.positions);
  int passes = 0;
  const int status = gs_sort_pairs_u32_any(n, gs_bit_length(vocab), b.keys, b.positions, b.keys_alt, b.positions_alt,
                                           b.sort_scratch, b.sort_bytes, &passes, (void*)s);
  if (status != GS_OK) return status;
  const u32* keys = passes % 2 ? b.keys_alt : b.keys;
  const int* positions = passes % 2 ? b.positions_alt : b.positions;
  absent_kernel<T><<<(unsigned)ceil_div(vocab, kThreads), kThreads, 0, s>>>(keys, n, (u32)vocab, dim, out);
  int length = group_length(n, 0);
  int64_t groups = ceil_div(n, length);
  runs<T, T, V>(keys, positions, n, vocab, grad, dim, dim, length, scale, out, b.next_keys[0], b.next[0], b.next_ld, s);
  // a level of one group hands nothing on
  for (int level = 1; groups > 1; ++level) {
    const int from = (level - 1) & 1, to = level & 1;
    const int64_t entries = 2 * groups;
    length = group_length(entries, level);
    groups = ceil_div(entries, length);
    runs<float, T, V>(b.next_keys[from], nullptr, entries, vocab, b.next[from], b.next_ld, dim, length, scale, out,
                      b.next_keys[to], b.next[to], b.next_ld, s);
  }
  return gs_status_from_hip(hipGetLastError());
}

template <typename T>
static int backward(int64_t n, int32_t vocab, int32_t dim, Tokens tokens, const void* grad, float scale,
                    int64_t padding, void* out, const BackwardPlan& b, hipStream_t s) {
  if (n == 0) {
    const int64_t all = (int64_t)vocab * dim;
    zero_kernel<T><<<(unsigned)min(ceil_div(all, kThreads), (int64_t)8192), kThreads, 0, s>>>((T*)out, all);
    return gs_status_from_hip(hipGetLastError());
  }
  const int v = vector_of<T>(dim, dim, grad, out);
  if (v == 16 / (int)sizeof(T))
    return gradient<T, 16 / sizeof(T)>(n, vocab, dim, tokens, (const T*)grad, scale, padding, (T*)out, b, s);
  if (v == 2) return gradient<T, 2>(n, vocab, dim, tokens, (const T*)grad, scale, padding, (T*)out, b, s);
  return gradient<T, 1>(n, vocab, dim, tokens, (const T*)grad, scale, padding, (T*)out, b, s);
}

static int check(int64_t n, int32_t vocab, int32_t dim, int32_t dtype, const void* tokens, int32_t bits, float scale) {
  if (n < 0 || vocab <= 0 || dim <= 0 || dtype < GS_FP32 || dtype > GS_FP16 || (bits != 32 && bits != 64) ||
      (n > 0 && !tokens) || !(fabsf(scale) < INFINITY))
    return GS_ERR_INVALID_ARGUMENT;
  // positions are int32; the columns' blocks are a grid's second dimension (at most 65535)
  return n > 0x7fffffffll || dim > (1 << 21) ? GS_ERR_OVERFLOW : GS_OK;
}

}  // namespace gs_embed

extern "C" int gs_embed_fwd(int64_t n, int32_t vocab, int32_t dim, int32_t dtype, const void* tokens,
                            int32_t token_bits, const void* table, int64_t ld_table, float scale, void* out,
                            void* stream) {
  const int status = gs_embed::check(n, vocab, dim, dtype, tokens, token_bits, scale);
  if (status != GS_OK) return status;
  if (ld_table < dim || (n > 0 && (!table || !out))) return GS_ERR_INVALID_ARGUMENT;
  if (n == 0) return GS_OK;
  const gs_embed::Tokens t = {tokens, token_bits};
  hipStream_t s = (hipStream_t)stream;
  if (dtype == GS_FP32) return gs_embed::forward<float>(n, vocab, dim, t, table, ld_table, scale, out, s);
  if (dtype == GS_BF16) return gs_embed::forward<__bf16>(n, vocab, dim, t, table, ld_table, scale, out, s);
  return gs_embed::forward<_Float16>(n, vocab, dim, t, table, ld_table, scale, out, s);
}

extern "C" size_t gs_embed_bwd_workspace_bytes(int64_t n, int32_t vocab, int32_t dim, int32_t dtype) {
  if (n <= 0 || vocab <= 0 || dim <= 0 || dtype < GS_FP32 || dtype > GS_FP16 || n > 0x7fffffffll) return 0;
  return gs_embed::BackwardPlan(n, dim, nullptr).bytes;
}

extern "C" int gs_embed_bwd(int64_t n, int32_t vocab, int32_t dim, int32_t dtype, const void* tokens,
                            int32_t token_bits, const void* grad_out, float scale, int64_t padding_index,
                            void* grad_table, void* workspace, size_t workspace_bytes, void* stream) {
  const int status = gs_embed::check(n, vocab, dim, dtype, tokens, token_bits, scale);
  if (status != GS_OK) return status;
  if (!grad_table || (n > 0 && !grad_out)) return GS_ERR_INVALID_ARGUMENT;
  if (n > 0 && ((uintptr_t)workspace & 255)) return GS_ERR_MISALIGNED;
  if (n > 0 && (!workspace || workspace_bytes < gs_embed_bwd_workspace_bytes(n, vocab, dim, dtype)))
    return GS_ERR_SCRATCH_TOO_SMALL;
  const gs_embed::BackwardPlan b(n, dim, n > 0 ? workspace : nullptr);
  const gs_embed::Tokens t = {tokens, token_bits};
  hipStream_t s = (hipStream_t)stream;
  if (dtype == GS_FP32)
    return gs_embed::backward<float>(n, vocab, dim, t, grad_out, scale, padding_index, grad_table, b, s);
  if (dtype == GS_BF16)
    return gs_embed::backward<__bf16>(n, vocab, dim, t, grad_out, scale, padding_index, grad_table, b, s);
  return gs_embed::backward<_Float16>(n, vocab, dim, t, grad_out, scale, padding_index, grad_table, b, s);
}
