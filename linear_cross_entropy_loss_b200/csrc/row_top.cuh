// The k largest logits of a row, found while the row streams past once.
//
// The row is looked at in groups of 32 bytes (8 or 16 logits). The k groups that come first by (largest logit
// descending, place ascending) hold the k first logits, since a group ahead of another has a logit ahead of all of
// its. So only the groups' maxima are kept, and the search works on them:
//
// 1. Stream: each thread loads two groups at a time, the next two on their way; a group's maximum goes to shared memory,
//    and four running maxima of the thread's groups stay in registers. No barrier, nothing that depends on the data.
// 2. Bound: the k-th largest of the block's 1024 running maxima. At least k groups reach it, and of a row of random
//    order about k (1 + k / 2048) do.
// 3. Collect: the groups that reach the bound go to a list. If it runs full (rows in an unlucky order, many equal
//    logits, several segments) it is cut back to its first k and the bound raised behind the last of them: an equal
//    maximum that comes later is behind.
// 4. Rank: the logits of the listed groups are read again and those that reach the bound sorted.
//
// What bounds it: for many long rows the stream (4096 x 131072 bf16, k = 64: 229 us, 4.7 TB/s; with the search left
// out 167 us would be the rate of a copy). The log-sum-exp costs an exponential per logit and about a tenth of that
// time; steps 2 to 4 are 17,000 of a block's 44,000 cycles, which the other two blocks of an SM hide in part. Four
// blocks of 64 registers were slower (261 us: they spill), and so was a ring of asynchronous copies (290 us). Few or
// short rows are bound by the chain of barriers: 15 us for one row.
//
// A row with more groups than the shared array takes goes through 1 to 3 in segments. A row may also be split over
// the blocks of a cluster, which share their first bounds and hand their lists to the first block.
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
constexpr int kTopParts = 8;
constexpr int kSearchBins = kTopThreads;
static_assert(kTopSegmentBytes >= kTopList * 8, "rank_list borrows the array of the maxima");
static_assert(kTopFull >= kTopMax, "the list keeps k groups and takes a chunk");

struct TopShared {
  unsigned long long list[kTopList];    // order_pair(largest logit, group); later, of a row in parts, the elements
  unsigned long long other[kTopList];   // the elements, order_pair(logit, index); of a row in parts first all lists
  uint4 maxima[kTopSegmentBytes / 16];  // the segment's groups: their maxima in the type of the logits
  unsigned int bins[kSearchBins];
  unsigned int range[2];
  unsigned int found[3];     // bin, keys above it, keys in it
  unsigned int count;        // entries of `list`
  unsigned int n_other;      // entries of `other`
  unsigned int place;
  unsigned long long bound;  // keys from here on enter (2^32: none)
  float scratch[32];
  // written by all blocks of the cluster, each into its own place
  uint32_t part_bound[kTopParts];
  float part_ref[kTopParts], part_sum[kTopParts];  // log-sum-exp of a part
};

// A block may write into another's shared memory only once that one runs: each block of a cluster says so as it starts
// (cluster_started) and waits for the others where it first writes (cluster_wait_started), by when they long have.
// Whole warps, every thread of the block.
__device__ __forceinline__ void cluster_started() { asm volatile("barrier.cluster.arrive.relaxed.aligned;"); }
__device__ __forceinline__ void cluster_wait_started() { asm volatile("barrier.cluster.wait.aligned;" ::: "memory"); }

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
    return e >= 0 && uint32_t(e + kPer) <= vocab ? load_stream(row + e) : load_edge(e);
  }
  __device__ __noinline__ Group load_edge(int e) const {
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

// A key that at least k of the block's keys reach, and (unless many are equal) at most k + slack. least / most: over
// this thread's keys; each(f): f(key) for this thread's keys, 0 for one that does not exist. 0 when there are fewer
// than k. A histogram of 256 bins over the range of the keys; where the bin in question holds too many, one over that
// bin.
template <typename Each>
__device__ __forceinline__ uint32_t bound_for(TopShared& s, int k, int slack, uint32_t least, uint32_t most, Each each) {
  const int lane = int(threadIdx.x & 31);
  __syncthreads();
  if (threadIdx.x == 0) {
    s.range[0] = 0xffffffffu;
    s.range[1] = 0;
  }
  s.bins[threadIdx.x] = 0;
  __syncthreads();
  least = __reduce_min_sync(0xffffffffu, least);
  most = __reduce_max_sync(0xffffffffu, most);
  if (lane == 0) {
    atomicMin(&s.range[0], least);
    atomicMax(&s.range[1], most);
  }
  __syncthreads();
  uint32_t lo = max(s.range[0], 1u), hi = s.range[1];
  unsigned int above = 0;  // keys above hi
  for (;;) {
    if (hi < lo) return 0u;  // no key at all
    const int shift = max(0, 24 - __clz(hi - lo));  // (hi - lo) >> shift < 256
    each([&](uint32_t key) {
      if (key >= lo && key <= hi) atomicAdd(&s.bins[(key - lo) >> shift], 1u);
    });
    __syncthreads();
    if (threadIdx.x < 32) {
      // lane l has the bins from 255 - 8 l downwards
      unsigned int c[8], mine = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        c[i] = s.bins[kSearchBins - 1 - 8 * lane - i];
        mine += c[i];
      }
      unsigned int inc = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned int before = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += before;
      }
      unsigned int seen = above + inc - mine;
      if (lane == 31 && above + inc < unsigned(k)) s.found[2] = 0xffffffffu;  // fewer than k
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (seen < unsigned(k) && seen + c[i] >= unsigned(k)) {
          s.found[0] = kSearchBins - 1 - 8 * lane - i;
          s.found[1] = seen;
          s.found[2] = c[i];
        }
        seen += c[i];
      }
    }
    __syncthreads();
    const unsigned int in_bin = s.found[2];
    if (in_bin == 0xffffffffu) return 0u;
    above = s.found[1];
    lo += s.found[0] << shift;
    if (above + in_bin <= unsigned(k + slack) || shift == 0) return lo;
    const uint32_t width = (1u << shift) - 1u;
    hi = hi - lo > width ? lo + width : hi;
    s.bins[threadIdx.x] = 0;
    __syncthreads();
  }
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

// Leaves at least the k first entries of a list, and at most `most_left` (k <= most_left) of them. Returns a key that
// all of them reach; what comes behind them in the order has a smaller one, or the same.
__device__ __noinline__ uint32_t cut_list(TopShared& s, unsigned long long* list, unsigned int& count, int k,
                                          int most_left) {
  __syncthreads();
  const int n = int(count);
  uint32_t least = 0xffffffffu, most = 0;
  for (int i = threadIdx.x; i < n; i += kTopThreads) {
    const uint32_t key = pair_key(list[i]);
    least = min(least, key);
    most = max(most, key);
  }
  const uint32_t from = bound_for(s, k, min(k / 4 + 16, most_left - k), least, most, [&](auto f) {
    for (int i = threadIdx.x; i < n; i += kTopThreads) f(pair_key(list[i]));
  });
  filter_list(list, count, n, [&](unsigned long long e) { return pair_key(e) >= from; });
  if (int(count) <= most_left) return from;
  // too many equal ones to tell apart by their keys
  block_sort_descending<kTopThreads>(list, int(count));
  if (threadIdx.x == 0) count = k;
  __syncthreads();
  return pair_key(list[k - 1]);
}

// The bound as a float that a vector's maximum can be held against: !(maximum < it) where an element may enter.
__device__ __forceinline__ float bound_value(unsigned long long bound) {
  if (bound <= kKeyNegInf) return -INFINITY;
  return bound <= 0xffffffffull ? key_to_float(uint32_t(bound)) : __uint_as_float(0x7fc00000u);
}

// bound_for four keys of each thread (0: no key), and for the maxima of a segment.
__device__ __noinline__ uint32_t bound_of_four(TopShared& s, int k, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  static_assert(2 * kTopUnroll == 4, "four running maxima");
  auto or_none = [](uint32_t key) { return key != 0 ? key : 0xffffffffu; };
  return bound_for(s, k, k / 4 + 4, min(min(or_none(a), or_none(b)), min(or_none(c), or_none(d))),
                   max(max(a, b), max(c, d)), [&](auto f) {
                     f(a);
                     f(b);
                     f(c);
                     f(d);
                   });
}
template <typename T, Nan kNan>
__device__ __noinline__ uint32_t bound_of_segment(TopShared& s, int k, int groups) {
  const T* const maxima = reinterpret_cast<const T*>(s.maxima);
  uint32_t least = 0xffffffffu, most = 0;
  for (int i = threadIdx.x; i < groups; i += kTopThreads) {
    const uint32_t key = search_key<kNan>(logit_to_float(maxima[i]));
    least = min(least, key);
    most = max(most, key);
  }
  return bound_for(s, k, 64, least, most, [&](auto f) {
    for (int i = threadIdx.x; i < groups; i += kTopThreads) f(search_key<kNan>(logit_to_float(maxima[i])));
  });
}

// The groups [seg, end) of the segment whose maxima lie in shared memory: those that reach the bound go to the list.
// (A function of its own, like the search: the registers of the stream are free here.)
template <typename T, Nan kNan>
__device__ __noinline__ void collect_segment(TopShared& s, int seg, int end, bool first_segment, int k, int limit) {
  const T* const maxima = reinterpret_cast<const T*>(s.maxima);
  // 16 bytes of maxima at a time: one comparison of their largest with the bound decides for all
  constexpr int kAtOnce = 16 / int(sizeof(T));
  auto collect = [&](int at, int stop) {  // this thread's places `at`, at + kTopThreads * kAtOnce, .. below `stop`
    const unsigned long long bound_key = s.bound;
    const float bound = bound_value(bound_key);
    bool full = false;
    for (; at < stop; at += kTopThreads * kAtOnce) {
      const uint4 raw = s.maxima[at / kAtOnce];
      Group one = RowGroups<T>::nothing();
      one.w[0] = raw.x; one.w[1] = raw.y; one.w[2] = raw.z; one.w[3] = raw.w;
      if (largest<kNan>(one, static_cast<const T*>(nullptr)) < bound) continue;
      float top[kAtOnce];
      if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 4; ++i) top[i] = __uint_as_float(one.w[i]);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) halves(one.w[i], top[2 * i], top[2 * i + 1], static_cast<const T*>(nullptr));
      }
      uint32_t hits = 0;
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i)
        hits |= !(top[i] < bound) && search_key<kNan>(top[i]) >= bound_key && seg + at + i < end ? 1u << i : 0u;
      if (hits == 0) continue;
      unsigned int place = atomicAdd(&s.count, (unsigned int)__popc(hits));
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) {
        if (!(hits & (1u << i))) continue;
        if (place < unsigned(kTopList)) s.list[place] = order_pair(search_key<kNan>(top[i]), uint32_t(seg + at + i));
        full |= place >= unsigned(limit);
        ++place;
      }
    }
    return full;
  };
  auto cut = [&]() {
    const uint32_t least_left = cut_list(s, s.list, s.count, k, limit);
    if (threadIdx.x == 0) s.bound = (unsigned long long)least_left + 1;
    __syncthreads();
  };
  // all at once: with a good bound few groups enter
  const int mine = kAtOnce * int(threadIdx.x);
  if (!__syncthreads_or(collect(mine, end - seg))) return;
  const bool lost = s.count > unsigned(kTopList);
  __syncthreads();
  if (!lost) {
    cut();
    return;
  }
  // again, a chunk at a time, cutting the list whenever it is full
  filter_list(s.list, s.count, kTopList,
              [&](unsigned long long e) { return !first_segment && pair_index(e) < uint32_t(seg); });
  for (int c = 0; c < end - seg; c += kTopChunk) {
    const int from = c + mine, stop = min(c + kTopChunk, end - seg);
    if (__syncthreads_or(collect(from, stop))) cut();
  }
}

// Groups [v0, v1) of the row into the list, which then has the k first of them among its entries (all of them if there
// are fewer than k). kSum: the thread's share of sum_j 2^(l_j * log2_scale - ref) goes to (ref, sum).
template <typename T, bool kSum, Nan kNan>
__device__ __forceinline__ void stream_top(TopShared& s, const RowGroups<T>& row, int v0, int v1, int parts, int k,
                                           float log2_scale, float& ref, float& sum) {
  constexpr int kSegment = kTopSegmentBytes / int(sizeof(T));  // groups
  static_assert(kSegment % kTopChunk == 0 && kSegment % (2 * kTopBatch) == 0, "segments are whole chunks");
  const T* tag = nullptr;
  if (parts > 1) cluster_started();
  const int limit = min(2 * k + 64, kTopFull);
  T* const maxima = reinterpret_cast<T*>(s.maxima);
  __syncthreads();
  if (threadIdx.x == 0) {
    s.count = 0;
    s.n_other = 0;
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
  for (int seg = v0; seg < v1; seg += kSegment) {
    const int end = min(seg + kSegment, v1);
    Group cur[kTopUnroll], nxt[kTopUnroll];
    fetch(seg, cur);
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
      if (vb + kTopBatch < end) fetch(vb + kTopBatch, nxt);
      take(vb, cur, run);
      if (vb + 2 * kTopBatch < end) fetch(vb + 2 * kTopBatch, cur);
      if (vb + kTopBatch < end) take(vb + kTopBatch, nxt, run + kTopUnroll);
    }
    __syncthreads();
    // The first bound. A row in parts needs k groups from all of them: each part finds a share of k among its first
    // segment, and the lowest of the parts' bounds is one that k groups reach. Where one part lies far above the
    // others its list runs full and is cut.
    if (parts == 1 || seg == v0) {
      const int want = (k + parts - 1) / parts;
      uint32_t from;
      if (want <= kTopThreads * kTopUnroll) {
        uint32_t key[2 * kTopUnroll];
#pragma unroll
        for (int i = 0; i < 2 * kTopUnroll; ++i)
          key[i] = seg + i * kTopThreads + int(threadIdx.x) < end ? search_key<kNan>(run[i]) : 0u;  // 0: no group
        from = bound_of_four(s, want, key[0], key[1], key[2], key[3]);
      } else {
        // more than half of the running maxima are wanted: they say too little, and the groups' own are searched
        from = bound_of_segment<T, kNan>(s, want, end - seg);
      }
      if (parts > 1) {  // every part comes here once: it has groups
        cooperative_groups::cluster_group cluster = cooperative_groups::this_cluster();
        cluster_wait_started();
        if (int(threadIdx.x) < parts) cluster.map_shared_rank(&s, threadIdx.x)->part_bound[cluster.block_rank()] = from;
        cluster.sync();
        for (int part = 0; part < parts; ++part) from = min(from, s.part_bound[part]);
      }
      if (threadIdx.x == 0) s.bound = max(s.bound, (unsigned long long)from);
      __syncthreads();
    }
    collect_segment<T, kNan>(s, seg, end, seg == v0, k, limit);
  }
  __syncthreads();
}

// The list that has the row's k first groups among its entries, and their number; of a row in parts in the first
// block, the others return with 0. `free_list`: room for the elements.
struct TopGroups {
  unsigned long long* list;
  unsigned long long* free_list;
  int n;
};
__device__ __forceinline__ TopGroups merge_lists(TopShared& s, int k, int parts) {
  __syncthreads();
  if (parts == 1) {
    if (s.count > unsigned(2 * k + 64)) cut_list(s, s.list, s.count, k, 2 * k + 64);
    return TopGroups{s.list, s.other, int(s.count)};
  }
  // every part hands over what it has, up to its share of the room; behind the barrier nobody looks at the others again
  if (s.count > unsigned(kTopList / parts)) cut_list(s, s.list, s.count, k, kTopList / parts);
  cooperative_groups::cluster_group cluster = cooperative_groups::this_cluster();
  TopShared* first = cluster.map_shared_rank(&s, 0);
  if (threadIdx.x == 0) s.place = atomicAdd(&first->n_other, s.count);
  __syncthreads();
  for (unsigned int i = threadIdx.x; i < s.count; i += kTopThreads) first->other[s.place + i] = s.list[i];
  cluster.sync();
  if (cluster.block_rank() != 0) return TopGroups{nullptr, nullptr, 0};
  if (s.n_other > unsigned(2 * k + 64)) cut_list(s, s.other, s.n_other, k, 2 * k + 64);
  return TopGroups{s.other, s.list, int(s.n_other)};
}

// Sorts a list of m <= kTopList entries, largest first, into its own place. `spare`: room for as many.
__device__ __noinline__ void rank_list(TopShared& s, unsigned long long* list, unsigned long long* spare, int m) {
  constexpr int kEach = kTopList / kTopThreads;
  __syncthreads();
  if (m <= kTopThreads / 2) {
    // few: every entry's place is the number of entries ahead of it
    const unsigned long long mine = int(threadIdx.x) < m ? list[threadIdx.x] : 0;
    int place = 0;
    for (int i = 0; i < m; ++i) place += list[i] > mine;
    __syncthreads();
    if (int(threadIdx.x) < m) list[place] = mine;
    __syncthreads();
    return;
  }
  // Entries go to 256 bins over the range of the keys; an entry's place is the number of those in bins ahead and of
  // those of its own bin ahead of it, of which there are few.
  if (threadIdx.x == 0) {
    s.range[0] = 0xffffffffu;
    s.range[1] = 0;
  }
  s.bins[threadIdx.x] = 0;
  __syncthreads();
  uint32_t least = 0xffffffffu, most = 0;
  for (int i = threadIdx.x; i < m; i += kTopThreads) {
    least = min(least, pair_key(list[i]));
    most = max(most, pair_key(list[i]));
  }
  least = __reduce_min_sync(0xffffffffu, least);
  most = __reduce_max_sync(0xffffffffu, most);
  if ((threadIdx.x & 31) == 0) {
    atomicMin(&s.range[0], least);
    atomicMax(&s.range[1], most);
  }
  __syncthreads();
  const uint32_t hi = s.range[1];
  const int shift = max(0, 24 - __clz(hi - s.range[0]));
  unsigned int at[kEach];
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int j = i * kTopThreads + int(threadIdx.x);
    at[i] = j < m ? atomicAdd(&s.bins[(hi - pair_key(list[j])) >> shift], 1u) : 0u;
  }
  __syncthreads();
  const unsigned int mine = s.bins[threadIdx.x];
  if (__syncthreads_or(mine > 64u)) {  // many equal ones
    block_sort_descending<kTopThreads>(list, m);
    return;
  }
  unsigned int total;
  const unsigned int begin = block_prefix(mine, reinterpret_cast<unsigned int*>(s.scratch), &total);
  s.bins[threadIdx.x] = begin;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int j = i * kTopThreads + int(threadIdx.x);
    if (j < m) spare[s.bins[(hi - pair_key(list[j])) >> shift] + at[i]] = list[j];
  }
  __syncthreads();
  for (int j = threadIdx.x; j < m; j += kTopThreads) {
    const unsigned long long e = spare[j];
    const uint32_t b = (hi - pair_key(e)) >> shift;
    const int first = int(s.bins[b]), end = b + 1 < uint32_t(kSearchBins) ? int(s.bins[b + 1]) : m;
    int place = first;
    for (int i = first; i < end; ++i) place += spare[i] > e;
    list[place] = e;
  }
  __syncthreads();
}

// The listed groups' logits again: the k first logits of the row (all of them if there are fewer), sorted, in
// g.free_list; returns how many.
template <Nan kNan, typename T>
__device__ __forceinline__ int rank_elements(TopShared& s, const RowGroups<T>& row, const TopGroups& g, int k) {
  constexpr int kPer = RowGroups<T>::kPer, kPart = kPer / 4;  // logits of a thread: a quarter of a group
  unsigned long long* const elements = g.free_list;
  unsigned int& count = s.place;
  __syncthreads();
  if (threadIdx.x == 0) {
    count = 0;
    s.range[0] = 0xffffffffu;
  }
  __syncthreads();
  uint32_t least = 0xffffffffu;
  for (int i = threadIdx.x; i < g.n; i += kTopThreads) least = min(least, pair_key(g.list[i]));
  least = __reduce_min_sync(0xffffffffu, least);
  if ((threadIdx.x & 31) == 0) atomicMin(&s.range[0], least);
  __syncthreads();
  uint32_t from = g.n >= k ? s.range[0] : 0u;  // g.n logits reach it
  auto expand = [&](int i0, int i1) {  // groups
    for (int i = 4 * i0 + int(threadIdx.x); i < 4 * i1; i += kTopThreads) {
      const int e = row.first_of(int(pair_index(g.list[i / 4]))) + i % 4 * kPart;
      T l[kPart];
      if (e >= 0 && uint32_t(e + kPart) <= row.vocab) {
        *reinterpret_cast<uint2*>(l) = __ldg(reinterpret_cast<const uint2*>(row.row + e));
      } else {
#pragma unroll
        for (int j = 0; j < kPart; ++j) l[j] = row.exists(e + j) ? row.row[e + j] : T(-INFINITY);
      }
#pragma unroll
      for (int j = 0; j < kPart; ++j) {
        const uint32_t key = search_key<kNan>(logit_to_float(l[j]));
        if (key >= from && row.exists(e + j)) {
          const unsigned int place = atomicAdd(&count, 1u);
          if (place < unsigned(kTopList)) elements[place] = order_pair(key, uint32_t(e + j));
        }
      }
    }
    __syncthreads();
    const int m = int(count);
    __syncthreads();
    return m;
  };
  int m = expand(0, g.n);
  if (m > kTopList) {
    // too many equal ones: again, few groups at a time, keeping the first k
    if (threadIdx.x == 0) count = 0;
    __syncthreads();
    m = 0;
    for (int i = 0; i < g.n; i += kTopMax / kPer) {
      if (m > kTopMax) from = cut_list(s, elements, count, k, kTopMax);
      m = expand(i, min(i + kTopMax / kPer, g.n));
    }
  }
  rank_list(s, elements, reinterpret_cast<unsigned long long*>(s.maxima), m);
  return min(m, k);
}

}  // namespace lce
