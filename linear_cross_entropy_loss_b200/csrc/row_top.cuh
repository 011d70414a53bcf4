// The k largest logits of a row, found while the row streams past once.
//
// The row is looked at in groups of 32 bytes (8 or 16 logits). The k groups that come first by (largest logit descending,
// place ascending) hold the k first logits, since a group ahead of another has a logit ahead of all of its. So only the groups'
// maxima are kept, and the search works on them:
//
// 1. Stream: each thread loads two groups at a time, the next two on their way; a group's maximum goes to shared memory,
//    and four running maxima of the thread's groups stay in registers. No barrier, nothing that depends on the data.
// 2. Bound: the k-th largest of the block's 1024 running maxima. At least k groups reach it, and of a row of random order
//    about k (1 + k / 2048) do.
// 3. Collect: the groups that reach the bound go to a list. If it runs full (rows in an unlucky order, many equal
//    logits, several segments) it is cut back to its first k and the bound raised behind the last of them: an equal maximum that
//    comes later is behind.
// 4. Rank: the logits of the listed groups are read again and those that reach the bound sorted.
//
// A row with more groups than the shared array takes goes through 1 to 3 in segments. A row may also be split over
// the blocks of a cluster; the first block then takes the others' lists.
#pragma once

#include "ptx.cuh"
#include "vocab_row.cuh"

#include <cooperative_groups.h>
#include <type_traits>

namespace lce {

constexpr int kTopMax = 1024;
constexpr int kTopThreads = 256;
constexpr int kTopUnroll = 2;                              // groups a thread loads at a time
constexpr int kTopBatch = kTopThreads * kTopUnroll;
constexpr int kTopChunk = 4 * kTopThreads;                 // groups looked at between two cuts of the list
constexpr int kTopSegmentBytes = 16384;                    // shared array of the maxima
constexpr int kTopList = 2048;                             // groups in the list
constexpr int kTopFull = kTopList - kTopChunk;             // most of them before a chunk: the chunk fits
constexpr int kTopElements = 2 * kTopMax;                  // logits of the last step: what is kept, and as many more
constexpr int kSearchSteps = 33;  // of bound_for: a step leaves a fifth of the range, or one key less
static_assert(kTopFull >= kTopMax, "the list keeps k groups and takes a chunk");

struct TopShared {
  unsigned long long list[kTopList];         // order_pair(largest logit, group)
  union {
    unsigned long long elements[kTopElements]; // order_pair(logit, index); after the last segment
    uint4 maxima[kTopSegmentBytes / 16];       // the segment's groups: their maxima in the type of the logits
  };
  unsigned int counters[2 * kSearchSteps + 1];
  unsigned int range[2];
  unsigned int count;        // entries of `list`
  unsigned int n_elements;   // entries of `elements`
  unsigned long long bound;  // keys from here on enter (2^32: none)
  float scratch[32];
  float part_ref, part_sum;  // log-sum-exp of this block's part
};

struct Group {
  uint32_t w[8];
};
// Streaming 32-byte load of data that is read once.
__device__ __forceinline__ Group load_stream(const void* p) {
  Group g;
  asm volatile("ld.global.nc.L1::no_allocate.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(g.w[0]), "=r"(g.w[1]), "=r"(g.w[2]), "=r"(g.w[3]), "=r"(g.w[4]), "=r"(g.w[5]), "=r"(g.w[6]),
                 "=r"(g.w[7])
               : "l"(p));
  return g;
}

// Two floats in one 64-bit register: half the instructions for the arithmetic around the exponentials.
__device__ __forceinline__ unsigned long long pack2(float a, float b) {
  unsigned long long r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpack2(unsigned long long v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ unsigned long long fma2(unsigned long long a, unsigned long long b, unsigned long long c) {
  unsigned long long r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ unsigned long long add2(unsigned long long a, unsigned long long b) {
  unsigned long long r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// A row as 32-byte groups on 32-byte boundaries. Group v holds the elements v * kPer - lead + 0 .. kPer - 1; those
// outside the row (before its first or after its last element) read as -inf.
template <typename T>
struct RowGroups {
  static constexpr int kPer = 32 / int(sizeof(T));
  using Bits = std::conditional_t<sizeof(T) == 4, uint32_t, unsigned short>;
  static constexpr uint32_t kNegInf =
      sizeof(T) == 4 ? 0xff800000u : (std::is_same<T, __half>::value ? 0xfc00u : 0xff80u);
  const T* row;
  uint32_t vocab;
  int lead;
  int groups;
  __device__ __forceinline__ RowGroups(const T* row_, uint32_t vocab_) : row(row_), vocab(vocab_) {
    lead = int((reinterpret_cast<uintptr_t>(row_) & 31u) / sizeof(T));
    groups = int((vocab + uint32_t(lead) + kPer - 1) / kPer);
  }
  __device__ __forceinline__ int first_of(int v) const { return v * kPer - lead; }
  // Whether the groups a .. b - 1 lie inside the row, and where group 0 would begin.
  __device__ __forceinline__ bool whole(int a, int b) const {
    return first_of(a) >= 0 && (long long)b * kPer - lead <= (long long)vocab;
  }
  __device__ __forceinline__ const char* base() const { return reinterpret_cast<const char*>(row - lead); }
  __device__ __forceinline__ bool exists(int e) const { return e >= 0 && uint32_t(e) < vocab; }
  __device__ __forceinline__ Group load(int v) const {
    const int e = first_of(v);
    if (e >= 0 && uint32_t(e + kPer) <= vocab) return load_stream(row + e);
    Group g = {};
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const uint32_t b = exists(e + i) ? uint32_t(reinterpret_cast<const Bits*>(row)[e + i]) : kNegInf;
      g.w[i * int(sizeof(T)) / 4] |= b << (8 * (i * int(sizeof(T)) % 4));
    }
    return g;
  }
  static __device__ __forceinline__ Group nothing() {
    Group g;
#pragma unroll
    for (int i = 0; i < 8; ++i) g.w[i] = sizeof(T) == 4 ? kNegInf : kNegInf * 0x10001u;
    return g;
  }
};

__device__ __forceinline__ float max_nan(float a, float b) {  // NaN if either is
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// What a NaN is to the search: larger than everything (listing), or nothing, like -inf (drawing).
enum class Nan { kFirst, kNever };
template <Nan kNan>
__device__ __forceinline__ uint32_t search_key(float f) {
  return kNan == Nan::kNever && f != f ? kKeyNegInf : order_key(f);
}
template <Nan kNan>
__device__ __forceinline__ float larger(float a, float b) {
  return kNan == Nan::kFirst ? max_nan(a, b) : fmaxf(a, b);
}

// The two elements of a 16-bit type in one word.
__device__ __forceinline__ void halves(uint32_t w, float& a, float& b, const __nv_bfloat16*) {
  a = __uint_as_float(w << 16);
  b = __uint_as_float(w & 0xffff0000u);
}
__device__ __forceinline__ void halves(uint32_t w, float& a, float& b, const __half*) {
  const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&w));
  a = t.x;
  b = t.y;
}
// The largest of a group (kFirst: NaN if one is).
template <Nan kNan>
__device__ __forceinline__ float largest(const Group& g, const float*) {
  float m = __uint_as_float(g.w[0]);
#pragma unroll
  for (int i = 1; i < 8; ++i) m = larger<kNan>(m, __uint_as_float(g.w[i]));
  return m;
}
template <Nan kNan, typename T2, typename T>
__device__ __forceinline__ float largest_of_pairs(const Group& g, const T* tag) {
  const T2* h = reinterpret_cast<const T2*>(g.w);
  auto two = [](T2 a, T2 b) { return kNan == Nan::kFirst ? __hmax2_nan(a, b) : __hmax2(a, b); };
  const T2 m = two(two(two(h[0], h[1]), two(h[2], h[3])), two(two(h[4], h[5]), two(h[6], h[7])));
  float a, b;
  halves(*reinterpret_cast<const uint32_t*>(&m), a, b, tag);
  return larger<kNan>(a, b);
}
template <Nan kNan>
__device__ __forceinline__ float largest(const Group& g, const __nv_bfloat16* t) {
  return largest_of_pairs<kNan, __nv_bfloat162>(g, t);
}
template <Nan kNan>
__device__ __forceinline__ float largest(const Group& g, const __half* t) {
  return largest_of_pairs<kNan, __half2>(g, t);
}

// sum_j 2^(l_j * scale + minus) of a group, added to two sums.
template <typename T>
__device__ __forceinline__ unsigned long long add_exponentials(unsigned long long sum2, const Group& g,
                                                               unsigned long long scale2, unsigned long long minus2,
                                                               const T* tag) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float a, b;
    if constexpr (sizeof(T) == 4) {
      if (i & 1) continue;
      a = __uint_as_float(g.w[i]);
      b = __uint_as_float(g.w[i + 1]);
    } else {
      halves(g.w[i], a, b, tag);
    }
    unpack2(fma2(pack2(a, b), scale2, minus2), a, b);
    sum2 = add2(sum2, pack2(fast_exp2(a), fast_exp2(b)));
  }
  return sum2;
}

// A key that at least k of the block's entries reach, and (unless many are equal) at most k + slack. The range of the keys
// is cut into five parts at a time (a step costs a barrier and a trip through shared memory, whatever it counts).
// least / most: over this thread's entries; count_from(key): how many of this thread's entries are >= key. With
// fewer than k entries: 0.
template <typename CountFrom>
__device__ __forceinline__ uint32_t bound_for(TopShared& s, int k, int slack, uint32_t least, uint32_t most,
                                              CountFrom count_from) {
  if (threadIdx.x < 2 * kSearchSteps + 1) s.counters[threadIdx.x] = 0;
  if (threadIdx.x == 0) {
    s.range[0] = 0xffffffffu;
    s.range[1] = 0;
  }
  __syncthreads();
  least = __reduce_min_sync(0xffffffffu, least);
  most = __reduce_max_sync(0xffffffffu, most);
  const unsigned int all = __reduce_add_sync(0xffffffffu, (unsigned int)count_from(0u));
  if ((threadIdx.x & 31) == 0) {
    atomicMin(&s.range[0], least);
    atomicMax(&s.range[1], most);
    atomicAdd(&s.counters[2 * kSearchSteps], all);
  }
  __syncthreads();
  if (int(s.counters[2 * kSearchSteps]) < k) return 0u;
  uint32_t lo = s.range[0];                                      // k or more from here on
  unsigned long long above = (unsigned long long)s.range[1] + 1;  // fewer than k from here on
  for (int step = 0; above - lo > 1; ++step) {
    const unsigned long long width = above - lo;
    uint32_t at[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) at[i] = uint32_t(lo + width * (i + 1) / 5);
    // two counts in a word: none is above 2^16
    unsigned int low = (unsigned int)count_from(at[0]) | (unsigned int)count_from(at[1]) << 16;
    unsigned int high = (unsigned int)count_from(at[2]) | (unsigned int)count_from(at[3]) << 16;
    low = __reduce_add_sync(0xffffffffu, low);
    high = __reduce_add_sync(0xffffffffu, high);
    if ((threadIdx.x & 31) == 0) {
      atomicAdd(&s.counters[2 * step], low);
      if (high != 0) atomicAdd(&s.counters[2 * step + 1], high);
    }
    __syncthreads();
    low = s.counters[2 * step];
    high = s.counters[2 * step + 1];
    const int total[4] = {int(low & 0xffffu), int(low >> 16), int(high & 0xffffu), int(high >> 16)};
    bool near = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (total[i] >= k) {
        if (at[i] > lo) lo = at[i];
        near = total[i] <= k + slack;
      } else if (at[i] < above) {
        above = at[i];
      }
    }
    if (near) break;
  }
  return lo;
}

// Keeps the entries of a list for which stay(entry) holds, in place: chunk by chunk, each read before any place up to
// its end is written.
template <typename Stay>
__device__ __forceinline__ void filter_list(unsigned long long* list, unsigned int& count, int n, Stay stay) {
  __syncthreads();
  if (threadIdx.x == 0) count = 0;
  for (int i0 = 0; i0 < n; i0 += kTopThreads) {
    const int at = i0 + int(threadIdx.x);
    const unsigned long long e = at < n ? list[at] : 0;
    __syncthreads();
    if (at < n && stay(e)) list[atomicAdd(&count, 1u)] = e;
  }
  __syncthreads();
}

// Sorts a list of n entries (room for the next power of two of them) and keeps the first k.
__device__ __forceinline__ void sort_list(unsigned long long* list, unsigned int& count, int n, int k) {
  __syncthreads();
  int padded = 2;
  while (padded < n) padded <<= 1;
  for (int i = n + threadIdx.x; i < padded; i += kTopThreads) list[i] = 0;
  block_sort_descending(list, padded);
  if (threadIdx.x == 0) count = min(n, k);
  __syncthreads();
}

// Leaves at least the k first entries of a list, and at most `most_left` (k <= most_left) of them. Returns a key that
// all of them reach; what comes behind them in the order has a smaller one, or the same.
__device__ __noinline__ uint32_t cut_list(TopShared& s, unsigned long long* list, unsigned int& count, int k, int most_left) {
  __syncthreads();
  const int n = int(count);
  uint32_t least = 0xffffffffu, most = 0;
  for (int i = threadIdx.x; i < n; i += kTopThreads) {
    const uint32_t key = pair_key(list[i]);
    least = min(least, key);
    most = max(most, key);
  }
  const uint32_t from = bound_for(s, k, min(k / 4 + 16, most_left - k), least, most, [&](uint32_t key) {
    int c = 0;
    for (int i = threadIdx.x; i < n; i += kTopThreads) c += pair_key(list[i]) >= key;
    return c;
  });
  filter_list(list, count, n, [&](unsigned long long e) { return pair_key(e) >= from; });
  if (int(count) <= most_left) return from;
  sort_list(list, count, int(count), k);  // too many equal ones to tell apart by their keys
  return pair_key(list[k - 1]);
}

// The bound as a float that a vector's maximum can be held against: !(maximum < it) where an element may enter.
__device__ __forceinline__ float bound_value(unsigned long long bound) {
  if (bound <= kKeyNegInf) return -INFINITY;
  return bound <= 0xffffffffull ? key_to_float(uint32_t(bound)) : __uint_as_float(0x7fc00000u);
}

// Groups [v0, v1) of the row into the list, which then has the k first of them among its entries (all of them if there
// are fewer than k). kSum: the thread's share of sum_j 2^(l_j * log2_scale - ref) goes to (ref, sum).
template <typename T, bool kSum, Nan kNan>
__device__ __forceinline__ void stream_top(TopShared& s, const RowGroups<T>& row, int v0, int v1, int k, float log2_scale,
                                           float& ref, float& sum) {
  constexpr int kSegment = kTopSegmentBytes / int(sizeof(T));  // groups
  static_assert(kSegment % kTopChunk == 0 && kSegment % (2 * kTopBatch) == 0, "segments are whole chunks");
  const T* tag = nullptr;
  const int limit = min(2 * k + 64, kTopFull);
  T* const maxima = reinterpret_cast<T*>(s.maxima);
  __syncthreads();
  if (threadIdx.x == 0) {
    s.count = 0;
    s.bound = 0;
  }
  auto fetch = [&](int vb, Group(&to)[kTopUnroll]) {
    if (row.whole(vb, vb + kTopBatch) && vb + kTopBatch <= v1) {
      const char* at = row.base() + ((long long)vb + int(threadIdx.x)) * 32;
#pragma unroll
      for (int u = 0; u < kTopUnroll; ++u) to[u] = load_stream(at + u * kTopThreads * 32);
    } else {
#pragma unroll
      for (int u = 0; u < kTopUnroll; ++u) {
        const int v = vb + u * kTopThreads + int(threadIdx.x);
        to[u] = v < v1 ? row.load(v) : RowGroups<T>::nothing();
      }
    }
  };
  ref = -INFINITY;
  sum = 0.f;
  Group cur[kTopUnroll], nxt[kTopUnroll];
  fetch(v0, cur);
  for (int seg = v0; seg < v1; seg += kSegment) {
    const int end = min(seg + kSegment, v1);
    float run[2 * kTopUnroll];
#pragma unroll
    for (int i = 0; i < 2 * kTopUnroll; ++i) run[i] = -INFINITY;
    auto take = [&](int vb, const Group(&g)[kTopUnroll], float* most) {
      float top[kTopUnroll];
#pragma unroll
      for (int u = 0; u < kTopUnroll; ++u) {
        top[u] = largest<kNan>(g[u], tag);
        maxima[vb - seg + u * kTopThreads + int(threadIdx.x)] = T(top[u]);
        most[u] = larger<kNan>(most[u], top[u]);
      }
      if (kSum) {
        float m = ref;
#pragma unroll
        for (int u = 0; u < kTopUnroll; ++u) m = fmaxf(m, top[u] * log2_scale);  // passes a NaN over
        if (m > ref) {
          sum *= fast_exp2(ref - m);
          ref = m;
        }
        const float minus = ref > -INFINITY ? -ref : 0.f;
        const unsigned long long scale2 = pack2(log2_scale, log2_scale), minus2 = pack2(minus, minus);
        unsigned long long sum2 = 0;
#pragma unroll
        for (int u = 0; u < kTopUnroll; ++u) sum2 = add_exponentials(sum2, g[u], scale2, minus2, tag);
        float even, odd;
        unpack2(sum2, even, odd);
        sum += even + odd;
      }
    };
    for (int vb = seg; vb < end; vb += 2 * kTopBatch) {
      if (vb + kTopBatch < v1) fetch(vb + kTopBatch, nxt);
      take(vb, cur, run);
      if (vb + 2 * kTopBatch < v1) fetch(vb + 2 * kTopBatch, cur);
      if (vb + kTopBatch < end) take(vb + kTopBatch, nxt, run + kTopUnroll);
    }
    __syncthreads();
    // the first bound; with more wanted than half the running maxima they say too little, and the groups' own are searched
    uint32_t from;
    if (k <= kTopThreads * kTopUnroll) {
      uint32_t key[2 * kTopUnroll], least = 0xffffffffu, most = 0;
#pragma unroll
      for (int i = 0; i < 2 * kTopUnroll; ++i) {
        key[i] = seg + i * kTopThreads + int(threadIdx.x) < end ? search_key<kNan>(run[i]) : 0u;  // 0: no group
        least = min(least, key[i]);
        most = max(most, key[i]);
      }
      from = bound_for(s, k, k / 4 + 4, least, most, [&](uint32_t b) {
        int c = 0;
#pragma unroll
        for (int i = 0; i < 2 * kTopUnroll; ++i) c += key[i] >= b;
        return c;
      });
    } else {
      uint32_t least = 0xffffffffu, most = 0;
      for (int i = threadIdx.x; i < end - seg; i += kTopThreads) {
        const uint32_t key = search_key<kNan>(logit_to_float(maxima[i]));
        least = min(least, key);
        most = max(most, key);
      }
      from = bound_for(s, k, 64, least, most, [&](uint32_t b) {
        int c = 0;
        for (int i = threadIdx.x; i < end - seg; i += kTopThreads) c += search_key<kNan>(logit_to_float(maxima[i])) >= b;
        return c;
      });
    }
    if (threadIdx.x == 0) s.bound = max(s.bound, (unsigned long long)from);
    __syncthreads();
    float bound = bound_value(s.bound);
    for (int c = seg; c < end; c += kTopChunk) {
      bool full = false;
      T four[4];
      const int at = c - seg + 4 * int(threadIdx.x);
      if constexpr (sizeof(T) == 4) *reinterpret_cast<uint4*>(four) = reinterpret_cast<const uint4*>(maxima)[at / 4];
      else *reinterpret_cast<uint2*>(four) = reinterpret_cast<const uint2*>(maxima)[at / 4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float top = logit_to_float(four[i]);
        if (!(top < bound) && seg + at + i < end) {
          const uint32_t key = search_key<kNan>(top);
          if (key >= s.bound) {
            const unsigned int place = atomicAdd(&s.count, 1u);
            s.list[place] = order_pair(key, uint32_t(seg + at + i));
            full |= place >= unsigned(limit);
          }
        }
      }
      if (__syncthreads_or(full)) {
        const uint32_t least = cut_list(s, s.list, s.count, k, limit);
        if (threadIdx.x == 0) s.bound = (unsigned long long)least + 1;
        __syncthreads();
        bound = bound_value(s.bound);
      }
    }
  }
  __syncthreads();
}

// Takes the other blocks' lists (and shares of the sum) into the first block, whose list then has the row's k first groups
// among its entries. k * parts <= kTopList. The other blocks return with their part done.
__device__ __forceinline__ void merge_lists(TopShared& s, int k, int parts) {
  if (parts > 1) {
    if (s.count > unsigned(kTopList / parts)) cut_list(s, s.list, s.count, k, kTopList / parts);
    cooperative_groups::cluster_group cluster = cooperative_groups::this_cluster();
    cluster.sync();
    if (cluster.block_rank() == 0) {
      unsigned int at = s.count;
      for (int part = 1; part < parts; ++part) {
        const TopShared* other = cluster.map_shared_rank(&s, part);
        const unsigned int n = other->count;
        for (unsigned int i = threadIdx.x; i < n; i += kTopThreads) s.list[at + i] = other->list[i];
        at += n;
      }
      __syncthreads();
      if (threadIdx.x == 0) {
        s.count = at;
        float m = s.part_ref;
        for (int part = 1; part < parts; ++part) m = fmaxf(m, cluster.map_shared_rank(&s, part)->part_ref);
        float sum = 0.f;
        for (int part = 0; part < parts; ++part) {
          const TopShared* other = cluster.map_shared_rank(&s, part);
          if (other->part_ref > -INFINITY) sum += other->part_sum * fast_exp2(other->part_ref - m);
        }
        s.part_ref = m;
        s.part_sum = sum;
      }
    }
    cluster.sync();
    if (cluster.block_rank() != 0) return;
  }
  __syncthreads();
  if (s.count > unsigned(k + k / 4 + 32)) cut_list(s, s.list, s.count, k, min(2 * k + 64, kTopFull));
}

// The listed groups' logits again: s.elements then holds the k first logits of the row (all of them if there are fewer),
// sorted, s.n_elements of them.
template <Nan kNan, typename T>
__device__ __forceinline__ void rank_elements(TopShared& s, const RowGroups<T>& row, int k) {
  constexpr int kPer = RowGroups<T>::kPer;
  __syncthreads();
  const int n = int(s.count);
  if (threadIdx.x == 0) {
    s.n_elements = 0;
    s.range[0] = 0xffffffffu;
  }
  __syncthreads();
  uint32_t least = 0xffffffffu;
  for (int i = threadIdx.x; i < n; i += kTopThreads) least = min(least, pair_key(s.list[i]));
  least = __reduce_min_sync(0xffffffffu, least);
  if ((threadIdx.x & 31) == 0) atomicMin(&s.range[0], least);
  __syncthreads();
  uint32_t from = n >= k ? s.range[0] : 0u;  // n logits reach it
  int m = 0;
  for (int i0 = 0; i0 < n * kPer; i0 += kTopMax) {
#pragma unroll
    for (int j = 0; j < kTopMax / kTopThreads; ++j) {
      const int i = i0 + j * kTopThreads + int(threadIdx.x);
      if (i < n * kPer) {
        const int e = row.first_of(int(pair_index(s.list[i / kPer]))) + i % kPer;
        if (row.exists(e)) {
          const uint32_t key = search_key<kNan>(logit_to_float(row.row[e]));
          if (key >= from) s.elements[atomicAdd(&s.n_elements, 1u)] = order_pair(key, uint32_t(e));
        }
      }
    }
    __syncthreads();
    m = int(s.n_elements);
    __syncthreads();
    if (m > kTopMax && i0 + kTopMax < n * kPer) from = cut_list(s, s.elements, s.n_elements, k, kTopMax);
  }
  if (m <= kTopThreads) {
    // few: every entry's place is the number of entries ahead of it
    const unsigned long long mine = int(threadIdx.x) < m ? s.elements[threadIdx.x] : 0;
    int place = 0;
    for (int i = 0; i < m; ++i) place += s.elements[i] > mine;
    __syncthreads();
    if (int(threadIdx.x) < m) s.elements[place] = mine;
    if (threadIdx.x == 0) s.n_elements = min(m, k);
    __syncthreads();
  } else {
    sort_list(s.elements, s.n_elements, m, k);
  }
}

}  // namespace lce
