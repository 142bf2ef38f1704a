// Rows of a shared table looked up by token, and the table's gradient.
//
//   out[i, :] = scale table[t_i, :]
//   grad_table[v, :] = scale sum_{i: t_i = v} grad_out[i, :]
//
// The gradient is a sum over positions of equal token: the positions are sorted
// stably by token, and runs of equal tokens are summed in position order.  The
// sorted list is cut into chunks of equal length whatever the runs are, one a
// workgroup, and those into parts, one a group of lanes, so a token that holds
// most positions costs no more than a flat distribution.  A workgroup writes the
// rows of the runs that lie inside its chunk and hands the (at most two) that go
// on past its ends, as fp32 sums, to a next level that treats them as a sorted
// list in turn, 2 entries for each chunk.  The order of every sum is fixed by the
// tokens alone: no atomics, the same bits every time.  Few positions need no
// sort: see few_kernel.
#include "gs_capi.h"

#include <algorithm>
#include <type_traits>

namespace gs_embed {

typedef unsigned u32;
constexpr u32 kNone = 0xffffffffu;  // an entry that holds nothing
constexpr int kThreads = 256;
constexpr int64_t kMaxLookup = 1ll << 31;  // vectors of a launch of the lookup

static inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
static inline int64_t round_up(int64_t a, int64_t b) { return ceil_div(a, b) * b; }

struct Tokens {
  const void* p;
  int bits;
  __device__ __forceinline__ int64_t at(int64_t i) const {
    return bits == 64 ? ((const int64_t*)p)[i] : (int64_t)((const int32_t*)p)[i];
  }
  Tokens from(int64_t i) const { return {(const char*)p + i * (bits / 8), bits}; }
};

// Rows are moved in vectors of 16 bytes (V elements), or, shorter ones, element by
// element.  kWhole: rows are whole vectors, on 16 bytes.  Else they may lie
// anywhere (the memory unit takes any address), and a row's last vector ends with
// the row, over elements that the one before it holds too: both carry the same.
template <typename T, int V>
struct __attribute__((aligned(sizeof(T) * V < 16 ? sizeof(T) * V : 16))) Vec {
  T v[V];
};

template <int V>
__device__ __forceinline__ int column_of(int vector, int D) {
  return min(vector * V, D - V);
}

template <bool kWhole, typename T, int V>
__device__ __forceinline__ Vec<T, V> load_vector(const T* __restrict__ p) {
  if (kWhole) return *reinterpret_cast<const Vec<T, V>*>(p);
  Vec<T, V> x;
  __builtin_memcpy(&x, p, sizeof(x));
  return x;
}

// The same, of what nothing else will read.
template <bool kWhole, typename T, int V>
__device__ __forceinline__ Vec<T, V> load_once(const T* __restrict__ p) {
  if constexpr (kWhole && sizeof(T) * V == 16) {
    typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
    return __builtin_bit_cast(Vec<T, V>, __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p)));
  } else {
    return load_vector<kWhole, T, V>(p);
  }
}

template <bool kWhole, typename T, int V>
__device__ __forceinline__ void store_vector(T* __restrict__ p, const Vec<T, V>& x) {
  if (kWhole) *reinterpret_cast<Vec<T, V>*>(p) = x;
  else __builtin_memcpy(p, &x, sizeof(x));
}

// ------------------------------------------------------------------ forward
// A thread moves a vector of V elements.  What bounds it is the write of out, and
// the table's read where it does not stay in the caches.  Blocks go to the 8 XCDs in
// turn, so each XCD is given a run of consecutive blocks, and the stores bypass the
// caches: 5M x 48 fp32 from 8192 rows takes 155 us (6.2 TB/s written; cached stores
// in launch order reach 3.6), 65536 x 1024 bf16 from 32768 rows 40 us (6.7 TB/s of
// reads and writes).
template <typename T, int V, bool kWhole>
__global__ __launch_bounds__(kThreads) void lookup_kernel(Tokens tokens, int64_t n, u32 vocab, int D, u32 row_vectors,
                                                          const T* __restrict__ table, int64_t ld, float scale,
                                                          T* __restrict__ out) {
  const u32 share = gridDim.x / 8;
  const int64_t block = blockIdx.x < 8 * share ? blockIdx.x % 8 * (int64_t)share + blockIdx.x / 8 : blockIdx.x;
  // the block's first vector as (position, vector of its row); the threads' vectors follow in 32 bits
  const int64_t first = block * kThreads;
  const int64_t row0 = first / row_vectors;
  const u32 at = (u32)(first - row0 * row_vectors) + threadIdx.x;
  const u32 r = at / row_vectors;
  if (row0 + r >= n) return;
  const int64_t token = tokens.at(row0 + r);
  const int column = column_of<V>((int)(at - r * row_vectors), D);
  Vec<T, V> x;
  if (token >= 0 && token < vocab) {
    x = load_vector<kWhole, T, V>(table + token * ld + column);
    if (scale != 1.0f)
#pragma unroll
      for (int e = 0; e < V; ++e) x.v[e] = (T)((float)x.v[e] * scale);
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) x.v[e] = (T)__builtin_nanf("");
  }
  T* to = out + (row0 + r) * D + column;
  if constexpr (kWhole && sizeof(x) == 16) {
    typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
    __builtin_nontemporal_store(__builtin_bit_cast(u32x4, x), reinterpret_cast<u32x4*>(to));
  } else {
    store_vector<kWhole, T, V>(to, x);
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

// Rows [first, first + 64) of the table that no token names are zeroed by a wave;
// absent: bit r is set for such a row first + r.
template <typename T>
__device__ __forceinline__ void zero_rows(uint64_t absent, int64_t first, int D, T* __restrict__ out) {
  const int lane = threadIdx.x & 63;
  typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
  constexpr int kVector = 16 / sizeof(T);
  const bool wide = D % kVector == 0 && (uintptr_t)out % 16 == 0;
  for (; absent; absent &= absent - 1) {
    T* o = out + (first + __builtin_ctzll(absent)) * D;
    if (wide)
      for (int c = lane; c < D / kVector; c += 64) reinterpret_cast<u32x4*>(o)[c] = u32x4{0, 0, 0, 0};
    else
      for (int c = lane; c < D; c += 64) o[c] = (T)0.0f;
  }
}

// One level of sums.  Reading grad_out row by row in the tokens' order bounds it:
// 5M rows of 192 bytes take 290 us (3.3 TB/s, 4.4 of whole 128-byte lines), 65536
// rows of 2 KB 56 us with the 32768 rows that they are summed to (3.6 TB/s).  Each
// lane has two batches of rows on their way, at addresses that are in LDS before.
// Each row is read once, past the caches: what it would leave in them has to make
// way for the next lookup's writes (a step of 5M x 48 fp32 takes 547 us, and 660
// with cached reads; of 200000 x 64, which the caches hold, 81 and 79).
// Entry e of n has key keys[e] (>= vocab: nothing) and its
// row at src + (positions ? positions[e] : e) * ld.
struct Level {
  const u32* keys;
  const int* positions;
  int64_t n;
  u32 vocab;
  int64_t ld;
  int D, lanes, length;  // a group of `lanes` lanes takes `length` entries
  int chunks;            // workgroups of entries; on the first level those behind them zero the rows without a token
  float scale;
  u32* next_keys;  // 2 a chunk: the run that comes in from the left, the one that only goes out to the right
  float* next;     // their rows, next_ld apart
  int64_t next_ld;
};

constexpr int kRunThreads = 512;
constexpr int kMaxChunk = 2048;  // entries of a chunk at most

// blockIdx.y: vector blockIdx.y lanes + l of a row is lane l's.
template <typename S, typename T, int V, bool kWhole>
__global__ __launch_bounds__(kRunThreads, 4) void runs_kernel(Level v, const S* __restrict__ src, T* __restrict__ out) {
  constexpr int kBatch = sizeof(S) * V > 16 ? 4 : 8;  // rows of a batch; two are in flight
  __shared__ u32 lds_keys[kMaxChunk + 3];
  __shared__ int lds_positions[kMaxChunk];
  __shared__ float lds_head[kRunThreads * V], lds_tail[kRunThreads * V];
  __shared__ u32 head_key[kRunThreads], tail_key[kRunThreads];
  __shared__ bool head_open[kRunThreads];

  if ((int)blockIdx.x >= v.chunks) {
    // a wave looks 64 rows of the table up, a lane each, by bisection
    if (blockIdx.y > 0) return;
    const int64_t first = ((int64_t)(blockIdx.x - v.chunks) * (kRunThreads / 64) + (threadIdx.x >> 6)) * 64;
    const int64_t row = first + (threadIdx.x & 63);
    bool absent = false;
    if (row < v.vocab) {
      int64_t lo = 0, hi = v.n;  // the first key >= row lies in [lo, hi]
      while (lo < hi) {
        const int64_t mid = (lo + hi) >> 1;
        if (v.keys[mid] < (u32)row) lo = mid + 1;
        else hi = mid;
      }
      absent = lo == v.n || v.keys[lo] != (u32)row;
    }
    return zero_rows(__ballot(absent), first, v.D, out);
  }

  const int groups = kRunThreads / v.lanes, group = threadIdx.x / v.lanes, lane = threadIdx.x % v.lanes;
  const int64_t chunk = (int64_t)groups * v.length, begin = (int64_t)blockIdx.x * chunk;
  const int here = (int)min(chunk, v.n - begin);  // the chunk's entries
  // keys[2 + e]: entry e of the chunk, with the two before it and the one behind
  u32* keys = lds_keys;
  for (int e = (int)threadIdx.x - 2; e < here + 1; e += kRunThreads) {
    const int64_t at = begin + e;
    keys[2 + e] = at >= 0 && at < v.n ? v.keys[at] : kNone;
  }
  if (v.positions)
    for (int e = threadIdx.x; e < here; e += kRunThreads) lds_positions[e] = v.positions[begin + e];
  __syncthreads();

  const bool in = (int)(blockIdx.y * v.lanes + lane) * V < v.D;
  const int col = column_of<V>(blockIdx.y * v.lanes + lane, v.D);
  auto write = [&](u32 key, const float* acc) {
    if (!in) return;
    Vec<T, V> x;
#pragma unroll
    for (int e = 0; e < V; ++e) x.v[e] = (T)(acc[e] * v.scale);
    store_vector<kWhole, T, V>(out + (int64_t)key * v.D + col, x);
  };

  // the group's own part
  const int e_begin = min(here, group * v.length), e_end = min(here, e_begin + v.length);
  u32 my_head = kNone, my_tail = kNone;
  bool my_open = false;
  if (e_begin < e_end) {
    // the last key before it: of the two entries before, the nearer may be empty
    u32 before = keys[2 + e_begin - 1];
    if (before >= v.vocab) before = keys[2 + e_begin - 2];
    const u32 after = keys[2 + e_end];
    u32 cur = kNone;
    bool from_left = false;
    float acc[V];
#pragma unroll
    for (int e = 0; e < V; ++e) acc[e] = 0.0f;
    auto keep = [&](float* lds) {
#pragma unroll
      for (int e = 0; e < V; ++e) lds[e * kRunThreads + threadIdx.x] = acc[e];
    };
    auto flush = [&](bool goes_on) {
      if (cur >= v.vocab) return;
      if (from_left) {
        my_head = cur;
        my_open = goes_on;
        keep(lds_head);
      } else if (goes_on) {
        my_tail = cur;
        keep(lds_tail);
      } else {
        write(cur, acc);
      }
    };
    Vec<S, V> x[2][kBatch];
    auto load = [&](int e0, Vec<S, V>* to) {
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const int e = e0 + j;
        if (e < e_end && in && keys[2 + e] < v.vocab) {
          const int64_t row = v.positions ? (int64_t)lds_positions[e] : begin + e;
          to[j] = load_once<kWhole, S, V>(src + row * v.ld + col);
        }
      }
    };
    auto add = [&](int e0, const Vec<S, V>* from) {
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        const u32 k = e0 + j < e_end ? keys[2 + e0 + j] : kNone;
        if (k >= v.vocab) continue;
        if (k != cur) {
          flush(false);
          from_left = cur == kNone && before == k;
          cur = k;
#pragma unroll
          for (int e = 0; e < V; ++e) acc[e] = 0.0f;
        }
        if (in)
#pragma unroll
          for (int e = 0; e < V; ++e) acc[e] += (float)from[j].v[e];
      }
    };
    load(e_begin, x[0]);
    for (int e0 = e_begin; e0 < e_end; e0 += 2 * kBatch) {
      load(e0 + kBatch, x[1]);
      add(e0, x[0]);
      load(e0 + 2 * kBatch, x[0]);
      add(e0 + kBatch, x[1]);
    }
    flush(cur == after);
  }
  if (lane == 0) {
    head_key[group] = my_head;
    tail_key[group] = my_tail;
    head_open[group] = my_open;
  }
  __syncthreads();

  // The runs that cross groups, in order: the waves' first groups join those of
  // their wave, the first of all what the waves leave (what comes in from the
  // left and what goes on to the right, in their first group's place).  One after
  // the other, 512 groups of rows of 4 values took 65 us.
  u32 out_head = kNone, out_tail = kNone;
  auto merge = [&](int first, int count, int step, bool last) {
    u32 cur = kNone;
    bool from_left = true, out_open = false;
    float acc[V];
#pragma unroll
    for (int e = 0; e < V; ++e) acc[e] = 0.0f;
    // slot 0: the head, 1: the tail
    auto hand_on = [&](int slot) {
      if (!in) return;
      if (last) {
        float* o = v.next + (2 * (int64_t)blockIdx.x + slot) * v.next_ld + col;
#pragma unroll
        for (int e = 0; e < V; ++e) o[e] = acc[e];
      } else {
        float* o = (slot ? lds_tail : lds_head) + first * v.lanes + lane;
#pragma unroll
        for (int e = 0; e < V; ++e) o[e * kRunThreads] = acc[e];
      }
    };
    auto close = [&](bool goes_on) {
      if (from_left) {
        out_head = cur;
        out_open = goes_on;
        hand_on(0);
      } else if (goes_on) {
        out_tail = cur;
        hand_on(1);
      } else {
        write(cur, acc);
      }
      cur = kNone;
    };
    // (what a batch of groups left is read at once: their keys and heads do not wait for each other)
    constexpr int kMerge = 8;
    for (int i0 = 0; i0 < count; i0 += kMerge) {
      u32 heads[kMerge], tails[kMerge];
      bool open[kMerge];
      float head[kMerge][V];
#pragma unroll
      for (int j = 0; j < kMerge; ++j) {
        const int g = first + min(i0 + j, count - 1) * step;
        heads[j] = i0 + j < count ? head_key[g] : kNone;
        tails[j] = i0 + j < count ? tail_key[g] : kNone;
        open[j] = head_open[g];
#pragma unroll
        for (int e = 0; e < V; ++e) head[j][e] = lds_head[e * kRunThreads + g * v.lanes + lane];
      }
#pragma unroll
      for (int j = 0; j < kMerge; ++j) {
        if (heads[j] != kNone) {
          if (cur == kNone) {  // it comes in from the groups before
            cur = heads[j];
            from_left = true;
#pragma unroll
            for (int e = 0; e < V; ++e) acc[e] = 0.0f;
          }
#pragma unroll
          for (int e = 0; e < V; ++e) acc[e] += head[j][e];
          if (!open[j]) close(false);
        }
        if (tails[j] != kNone) {
          cur = tails[j];
          from_left = false;
          const int g = first + (i0 + j) * step;
#pragma unroll
          for (int e = 0; e < V; ++e) acc[e] = lds_tail[e * kRunThreads + g * v.lanes + lane];
        }
      }
    }
    if (cur != kNone) close(true);
    return out_open;
  };
  const int wave_groups = 64 / v.lanes;
  if (wave_groups > 1) {
    if ((threadIdx.x & 63) < v.lanes) {
      const bool open = merge(group, wave_groups, 1, false);
      if (lane == 0) {
        head_key[group] = out_head;
        tail_key[group] = out_tail;
        head_open[group] = open;
      }
      out_head = out_tail = kNone;
    }
    __syncthreads();
  }
  if (group > 0) return;
  merge(0, kRunThreads / 64, wave_groups, true);
  if (lane == 0 && blockIdx.y == 0 && v.next_keys) {
    v.next_keys[2 * (int64_t)blockIdx.x] = out_head;
    v.next_keys[2 * (int64_t)blockIdx.x + 1] = out_tail;
  }
}

// Few positions: no sort.  Workgroup i < n looks for its position's token among
// all of them; if it is the token's first, it lists the others and sums their
// rows, a part of the list for each group of lanes, the parts joined in order.
// The workgroups behind zero the rows of the table that no token names.  One launch
// in place of the sort's eight or so, at n reads of n tokens: 2048 positions take
// 10 to 20 us against 32 to 46 sorted, 4096 take as long as sorted or longer (55
// against 42 at 64 columns of 32000 rows).
constexpr int kFew = 2048;
template <typename T, int V, bool kWhole>
__global__ __launch_bounds__(kThreads) void few_kernel(Tokens tokens, int n, u32 vocab, int64_t padding, int D,
                                                       int lanes, float scale, const T* __restrict__ grad,
                                                       T* __restrict__ out) {
  __shared__ u32 keys[kFew];
  __shared__ int list[kFew];
  __shared__ int counts[kThreads / 64];
  __shared__ float sums[kThreads * V];
  auto key_of = [&](int i) {
    const int64_t t = tokens.at(i);
    return t >= 0 && t < vocab && t != padding ? (u32)t : kNone;
  };
  if ((int)blockIdx.x >= n) {
    if (blockIdx.y > 0) return;
    // 256 rows, a bit each
    u32* named = keys;
    const int64_t first = (int64_t)(blockIdx.x - n) * kThreads;
    if (threadIdx.x < kThreads / 32) named[threadIdx.x] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kThreads) {
      const u32 k = key_of(i);
      if (k != kNone && k >= first && k < first + kThreads) atomicOr(&named[(k - first) >> 5], 1u << (k & 31));
    }
    __syncthreads();
    const int64_t wave_first = first + (threadIdx.x & ~63);
    const bool absent = first + threadIdx.x < vocab && !((named[threadIdx.x >> 5] >> (threadIdx.x & 31)) & 1);
    return zero_rows(__ballot(absent), wave_first, D, out);
  }

  const int me = blockIdx.x;
  const u32 mine = key_of(me);
  if (mine == kNone) return;
  // the positions of my token, in order: each wave lists a part of the positions
  const int wave = threadIdx.x >> 6, lane64 = threadIdx.x & 63;
  const int share = (n + kThreads - 1) / kThreads * 64;  // positions of a wave
  const int from = min(n, wave * share), to = min(n, from + share);
  int found = 0;
  for (int i0 = from; i0 < to; i0 += 64) {
    const int i = i0 + lane64;
    const bool same = i < to && key_of(i) == mine;
    const uint64_t who = __ballot(same);
    if (same) keys[from + found + __builtin_popcountll(who & ((1ull << lane64) - 1))] = (u32)i;
    found += __builtin_popcountll(who);
  }
  if (lane64 == 0) counts[wave] = found;
  __syncthreads();
  int before = 0, all = 0;
  for (int w = 0; w < kThreads / 64; ++w) {
    if (w < wave) before += counts[w];
    all += counts[w];
  }
  for (int i = lane64; i < found; i += 64) list[before + i] = (int)keys[from + i];
  __syncthreads();
  if (list[0] != me) return;  // the token's first position does the work

  const int groups = kThreads / lanes, group = threadIdx.x / lanes, lane = threadIdx.x % lanes;
  const bool in = (int)(blockIdx.y * lanes + lane) * V < D;
  const int col = column_of<V>(blockIdx.y * lanes + lane, D);
  const int part = (all + groups - 1) / groups;
  const int p_begin = min(all, group * part), p_end = min(all, p_begin + part);
  float acc[V];
#pragma unroll
  for (int e = 0; e < V; ++e) acc[e] = 0.0f;
  if (in) {
    constexpr int kBatch = 8;
    for (int p0 = p_begin; p0 < p_end; p0 += kBatch) {
      Vec<T, V> x[kBatch];
#pragma unroll
      for (int j = 0; j < kBatch; ++j)
        if (p0 + j < p_end) x[j] = load_vector<kWhole, T, V>(grad + (int64_t)list[p0 + j] * D + col);
#pragma unroll
      for (int j = 0; j < kBatch; ++j)
        if (p0 + j < p_end)
#pragma unroll
          for (int e = 0; e < V; ++e) acc[e] += (float)x[j].v[e];
    }
  }
  if (all > part) {  // more than one group has a part
#pragma unroll
    for (int e = 0; e < V; ++e) sums[e * kThreads + threadIdx.x] = acc[e];
    __syncthreads();
    if (group > 0) return;
    for (int g = 1; g * part < all; ++g)
#pragma unroll
      for (int e = 0; e < V; ++e) acc[e] += sums[e * kThreads + g * lanes + lane];
  }
  if (group > 0 || !in) return;
  Vec<T, V> x;
#pragma unroll
  for (int e = 0; e < V; ++e) x.v[e] = (T)(acc[e] * scale);
  store_vector<kWhole, T, V>(out + (int64_t)mine * D + col, x);
}

template <typename T>
__global__ __launch_bounds__(kThreads) void zero_kernel(T* __restrict__ out, int64_t n) {
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < n; i += (int64_t)gridDim.x * kThreads)
    out[i] = (T)0.0f;
}

// ------------------------------------------------------------------ host
static int vector_of(int32_t dtype, int64_t D) {
  const int V = dtype == GS_FP32 ? 4 : 8;
  return D < V ? 1 : V;
}

// Calls f with V and kWhole for rows of D elements, ld apart in a and contiguous in b.
template <typename T, class F>
static int with_vectors(int64_t D, int64_t ld, const void* a, const void* b, F f) {
  constexpr int V = 16 / sizeof(T);
  if (D < V) return f(std::integral_constant<int, 1>{}, std::true_type{});
  if (D % V == 0 && ld % V == 0 && (uintptr_t)a % 16 == 0 && (uintptr_t)b % 16 == 0)
    return f(std::integral_constant<int, V>{}, std::true_type{});
  return f(std::integral_constant<int, V>{}, std::false_type{});
}

template <typename T>
static int forward(int64_t n, int32_t vocab, int32_t dim, Tokens tokens, const void* table, int64_t ld, float scale,
                   void* out, hipStream_t s) {
  return with_vectors<T>(dim, ld, table, out, [&](auto V, auto kWhole) {
    const int64_t row_vectors = ceil_div(dim, V);
    // a launch has fewer than 2^32 threads
    const int64_t most = std::max((int64_t)1, kMaxLookup / row_vectors);
    for (int64_t i = 0; i < n; i += most) {
      const int64_t here = std::min(most, n - i);
      lookup_kernel<T, V, kWhole><<<(unsigned)ceil_div(here * row_vectors, kThreads), kThreads, 0, s>>>(
          tokens.from(i), here, (u32)vocab, dim, (u32)row_vectors, (const T*)table, ld, scale, (T*)out + i * dim);
    }
    return gs_status_from_hip(hipGetLastError());
  });
}

// Lanes of a row: a power of two, at most a wave.
static int lanes_of(int D, int V) {
  int lanes = 1;
  while (lanes < 64 && lanes * V < D) lanes *= 2;
  return lanes;
}

// Entries of a group.  On the first level 4 to 64, by how many make 512 chunks, two
// a CU (1M x 16 bf16 into 256 rows, with the lookup: 111 us, and 119 at 1024 chunks;
// 65536 x 1024 into 32768 rows: 125, 131 at 1024, 126 at 256); above, all of them
// where that is 8 at most, else 8 and on,
// so that at most 64 chunks hand on to the next level: few levels, and none that
// leaves many rows to one workgroup (2048 rows of 256 bytes take one 43 us).
static int group_length(int64_t n, int lanes, bool first) {
  const int groups = kRunThreads / lanes, most = std::min(64, kMaxChunk / groups);
  // (above, even: a part begins with a chunk's first entry, so that what is empty
  // between two entries of a run is one at most, and before the part)
  if (!first && n <= groups * std::min(8, most)) return (int)round_up(ceil_div(n, groups), 2);
  int length = first ? 4 : std::min(8, most);
  while (2 * length <= most && n / (length * groups) > (first ? 512 : 64)) length *= 2;
  return std::min(length, most);
}

static int64_t chunks_of(int64_t n, int lanes, bool first) {
  return ceil_div(n, (int64_t)kRunThreads / lanes * group_length(n, lanes, first));
}

struct BackwardPlan {
  u32 *keys, *keys_alt, *next_keys[2];
  int *positions, *positions_alt;
  float* next[2];
  int64_t next_ld;
  char* sort_scratch;
  size_t sort_bytes, bytes;

  // vector: elements of a vector of the rows' type
  BackwardPlan(int64_t n, int32_t dim, int vector, void* ws) {
    char* base = (char*)ws;
    size_t at = 0;
    auto take = [&](int64_t size) {
      char* p = base ? base + at : nullptr;
      at += (size_t)round_up(size, 256);
      return p;
    };
    bytes = 256;
    if (n <= kFew) return;  // few_kernel uses none of it
    next_ld = round_up(dim, 8);
    sort_bytes = gs_sort_scratch_bytes(n);
    keys = (u32*)take(n * 4);
    keys_alt = (u32*)take(n * 4);
    positions = (int*)take(n * 4);
    positions_alt = (int*)take(n * 4);
    sort_scratch = take((int64_t)sort_bytes);
    // the levels' entries, in turn in two places
    const int lanes = lanes_of(dim, vector);
    int64_t entries[2];
    entries[0] = 2 * chunks_of(n, lanes, true);
    entries[1] = 2 * chunks_of(entries[0], lanes, false);
    for (int level = 0; level < 2; ++level) {
      next_keys[level] = (u32*)take(entries[level] * 4);
      next[level] = (float*)take(entries[level] * next_ld * 4);
    }
    bytes = at;
  }
};

template <bool kFirst, typename S, typename T, int V, bool kWhole>
static int64_t runs(Level v, const S* src, T* out, hipStream_t s) {
  v.lanes = lanes_of(v.D, V);
  v.length = group_length(v.n, v.lanes, kFirst);
  v.chunks = (int)chunks_of(v.n, v.lanes, kFirst);
  const int64_t blocks = v.chunks + (kFirst ? ceil_div(v.vocab, kRunThreads) : 0);
  const dim3 grid((unsigned)blocks, (unsigned)ceil_div(v.D, v.lanes * V));
  runs_kernel<S, T, V, kWhole><<<grid, kRunThreads, 0, s>>>(v, src, out);
  return v.chunks;
}

template <typename T, int V, bool kWhole>
static int gradient(int64_t n, int32_t vocab, int32_t dim, Tokens tokens, const T* grad, float scale, int64_t padding,
                    T* out, const BackwardPlan& b, hipStream_t s) {
  if (n <= kFew) {
    const int lanes = lanes_of(dim, V);
    const dim3 grid((unsigned)(n + ceil_div(vocab, kThreads)), (unsigned)ceil_div(dim, lanes * V));
    few_kernel<T, V, kWhole><<<grid, kThreads, 0, s>>>(tokens, (int)n, (u32)vocab, padding, dim, lanes, scale, grad,
                                                       out);
    return gs_status_from_hip(hipGetLastError());
  }
  const int64_t key_blocks = std::min(ceil_div(n, kThreads), (int64_t)8192);
  keys_kernel<<<(unsigned)key_blocks, kThreads, 0, s>>>(tokens, n, (u32)vocab, padding,
                                                        b.keys, b.positions);
  int passes = 0;
  const int status = gs_sort_pairs_u32_any(n, gs_bit_length(vocab), b.keys, b.positions, b.keys_alt, b.positions_alt,
                                           b.sort_scratch, b.sort_bytes, &passes, (void*)s);
  if (status != GS_OK) return status;
  Level v = {};
  v.keys = passes % 2 ? b.keys_alt : b.keys;
  v.positions = passes % 2 ? b.positions_alt : b.positions;
  v.n = n;
  v.vocab = (u32)vocab;
  v.ld = dim;
  v.D = dim;
  v.scale = scale;
  v.next_keys = b.next_keys[0];
  v.next = b.next[0];
  v.next_ld = b.next_ld;
  int64_t chunks = runs<true, T, T, V, kWhole>(v, grad, out, s);
  // a level of one chunk hands nothing on
  for (int level = 1; chunks > 1; ++level) {
    const int from = (level - 1) & 1, to = level & 1;
    v.keys = b.next_keys[from];
    v.positions = nullptr;
    v.n = 2 * chunks;
    v.ld = b.next_ld;
    v.next_keys = b.next_keys[to];
    v.next = b.next[to];
    chunks = runs<false, float, T, V, kWhole>(v, b.next[from], out, s);
  }
  return gs_status_from_hip(hipGetLastError());
}

template <typename T>
static int backward(int64_t n, int32_t vocab, int32_t dim, Tokens tokens, const void* grad, float scale,
                    int64_t padding, void* out, const BackwardPlan& b, hipStream_t s) {
  if (n == 0) {
    const int64_t all = (int64_t)vocab * dim;
    zero_kernel<T><<<(unsigned)std::min(ceil_div(all, kThreads), (int64_t)8192), kThreads, 0, s>>>((T*)out, all);
    return gs_status_from_hip(hipGetLastError());
  }
  return with_vectors<T>(dim, dim, grad, out, [&](auto V, auto kWhole) {
    return gradient<T, V, kWhole>(n, vocab, dim, tokens, (const T*)grad, scale, padding, (T*)out, b, s);
  });
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
  return gs_embed::BackwardPlan(n, dim, gs_embed::vector_of(dtype, dim), nullptr).bytes;
}

extern "C" int gs_embed_bwd(int64_t n, int32_t vocab, int32_t dim, int32_t dtype, const void* tokens,
                            int32_t token_bits, const void* grad_out, float scale, int64_t padding_index,
                            void* grad_table, void* workspace, size_t workspace_bytes, void* stream) {
  const int status = gs_embed::check(n, vocab, dim, dtype, tokens, token_bits, scale);
  if (status != GS_OK) return status;
  if (!grad_table || (n > 0 && !grad_out)) return GS_ERR_INVALID_ARGUMENT;
  const size_t need = gs_embed_bwd_workspace_bytes(n, vocab, dim, dtype);
  if (need > 0 && ((uintptr_t)workspace & 255)) return GS_ERR_MISALIGNED;
  if (need > 0 && (!workspace || workspace_bytes < need)) return GS_ERR_SCRATCH_TOO_SMALL;
  const gs_embed::BackwardPlan b(n, dim, gs_embed::vector_of(dtype, dim), workspace);
  const gs_embed::Tokens t = {tokens, token_bits};
  hipStream_t s = (hipStream_t)stream;
  if (dtype == GS_FP32)
    return gs_embed::backward<float>(n, vocab, dim, t, grad_out, scale, padding_index, grad_table, b, s);
  if (dtype == GS_BF16)
    return gs_embed::backward<__bf16>(n, vocab, dim, t, grad_out, scale, padding_index, grad_table, b, s);
  return gs_embed::backward<_Float16>(n, vocab, dim, t, grad_out, scale, padding_index, grad_table, b, s);
}
