// The k largest logits of a row, found while the row streams past once.
//
// The row is looked at in vectors of 16 bytes (4 or 8 logits). A list in shared memory keeps the vectors that come first
// by (largest logit descending, place ascending): the k first of them hold the k first logits, since a vector ahead of
// another has a logit ahead of all of its. So the streaming loop handles one number per vector: one comparison of its
// maximum with the bound of the list, and what enters is one entry, however its logits lie. At the end the k vectors are
// read again and their logits ranked.
//
// * Vectors come in batches of kTopThreads * kTopUnroll, the next batch on its way while one is looked at.
// * The first bound comes from the first batch: the k-th largest of its maxima.
// * A list that holds twice what is wanted is cut back and the bound raised behind its last entry, so of a row of random
//   order about k (1 + ln(batches)) vectors enter. An equal maximum that comes later is behind: after a cut only larger ones enter.
// * Between two batches the list holds at most kTopFull entries, so a batch always fits.
// A row may be split over the blocks of a cluster; the first block then takes the others' lists.
#pragma once

#include "ptx.cuh"
#include "vocab_row.cuh"

#include <type_traits>

namespace lce {

constexpr int kTopMax = 1024;
constexpr int kTopThreads = 256;
constexpr int kTopUnroll = 4;
constexpr int kTopList = 2048;             // vectors in the list
constexpr int kTopFull = kTopList - kTopThreads * kTopUnroll;
constexpr int kTopElements = 2 * kTopMax;  // logits of the last step: what is kept, and as many from the next vectors
static_assert(kTopFull >= kTopMax, "the list keeps k vectors and takes a batch");

struct TopShared {
  unsigned long long list[kTopList];         // order_pair(largest logit, vector)
  unsigned long long elements[kTopElements]; // order_pair(logit, index)
  unsigned int counters[34];
  unsigned int range[2];
  unsigned int count;        // entries of `list`
  unsigned int n_elements;   // entries of `elements`
  unsigned long long bound;  // keys from here on enter (2^32: none)
  float scratch[32];
  float part_ref, part_sum;  // log-sum-exp of this block's part
};

// Streaming 16-byte load of data that is read once.
__device__ __forceinline__ uint4 load_stream(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

// A row as 16-byte vectors on 16-byte boundaries. Vector v holds the elements v * kPer - lead + 0 .. kPer - 1; those
// outside the row (before its first or after its last vector's end) read as -inf.
template <typename T>
struct RowVectors {
  static constexpr int kPer = 16 / int(sizeof(T));
  const T* row;
  uint32_t vocab;
  int lead;
  int vectors;
  __device__ __forceinline__ RowVectors(const T* row_, uint32_t vocab_) : row(row_), vocab(vocab_) {
    lead = int((reinterpret_cast<uintptr_t>(row_) & 15u) / sizeof(T));
    vectors = int((vocab + uint32_t(lead) + kPer - 1) / kPer);
  }
  __device__ __forceinline__ int first_of(int v) const { return v * kPer - lead; }
  __device__ __forceinline__ uint4 load(int v) const {
    const int e = first_of(v);
    if (e >= 0 && uint32_t(e + kPer) <= vocab) return load_stream(row + e);
    using Bits = std::conditional_t<sizeof(T) == 4, uint32_t, unsigned short>;
    uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const bool exists = e + i >= 0 && uint32_t(e + i) < vocab;
      const uint32_t b = exists ? uint32_t(reinterpret_cast<const Bits*>(row)[e + i]) : kNegInf;
      w[i * int(sizeof(T)) / 4] |= b << (8 * (i * int(sizeof(T)) % 4));
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  static constexpr uint32_t kNegInf =
      sizeof(T) == 4 ? 0xff800000u : (std::is_same<T, __half>::value ? 0xfc00u : 0xff80u);
  static __device__ __forceinline__ uint4 nothing() {
    constexpr uint32_t b = sizeof(T) == 4 ? kNegInf : kNegInf * 0x10001u;
    return make_uint4(b, b, b, b);
  }
};

__device__ __forceinline__ float max_nan(float a, float b) {  // NaN if either is
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// The elements of a vector as floats, and the largest of them (NaN if one is).
__device__ __forceinline__ void unpack(const uint4& v, float (&f)[4], const float*) {
  f[0] = __uint_as_float(v.x); f[1] = __uint_as_float(v.y); f[2] = __uint_as_float(v.z); f[3] = __uint_as_float(v.w);
}
__device__ __forceinline__ void unpack(const uint4& v, float (&f)[8], const __nv_bfloat16*) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = __uint_as_float(w[i] << 16);
    f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ void unpack(const uint4& v, float (&f)[8], const __half*) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    f[2 * i] = t.x;
    f[2 * i + 1] = t.y;
  }
}
__device__ __forceinline__ float largest(const uint4& v, const float*) {
  return max_nan(max_nan(__uint_as_float(v.x), __uint_as_float(v.y)), max_nan(__uint_as_float(v.z), __uint_as_float(v.w)));
}
__device__ __forceinline__ float largest(const uint4& v, const __nv_bfloat16*) {
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&v);
  const __nv_bfloat162 m = __hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3]));
  return max_nan(__low2float(m), __high2float(m));
}
__device__ __forceinline__ float largest(const uint4& v, const __half*) {
  const __half2* h = reinterpret_cast<const __half2*>(&v);
  const __half2 m = __hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3]));
  return max_nan(__low2float(m), __high2float(m));
}

// A key that at least k of the block's entries reach, and (unless many are equal) at most k + slack. Bisection of the
// range of the keys; every step is one count over the block. least / most: over this thread's entries; count_from(key):
// how many of this thread's entries are >= key. With fewer than k entries: 0.
template <typename CountFrom>
__device__ __forceinline__ uint32_t bound_for(TopShared& s, int k, int slack, uint32_t least, uint32_t most,
                                              CountFrom count_from) {
  if (threadIdx.x < 34) s.counters[threadIdx.x] = 0;
  if (threadIdx.x == 0) {
    s.range[0] = 0xffffffffu;
    s.range[1] = 0;
  }
  __syncthreads();
  least = __reduce_min_sync(0xffffffffu, least);
  most = __reduce_max_sync(0xffffffffu, most);
  if ((threadIdx.x & 31) == 0) {
    atomicMin(&s.range[0], least);
    atomicMax(&s.range[1], most);
  }
  const unsigned int all = __reduce_add_sync(0xffffffffu, (unsigned int)count_from(0u));
  if ((threadIdx.x & 31) == 0) atomicAdd(&s.counters[33], all);
  __syncthreads();
  if (int(s.counters[33]) < k) return 0u;
  uint32_t lo = s.range[0];                                      // k or more from here on
  unsigned long long above = (unsigned long long)s.range[1] + 1;  // fewer than k from here on
  for (int step = 0; above - lo > 1; ++step) {
    const uint32_t mid = uint32_t(lo + (above - lo) / 2);
    const unsigned int mine = __reduce_add_sync(0xffffffffu, (unsigned int)count_from(mid));
    if ((threadIdx.x & 31) == 0 && mine != 0) atomicAdd(&s.counters[step], mine);
    __syncthreads();
    const int total = int(s.counters[step]);
    if (total >= k) {
      lo = mid;
      if (total <= k + slack) break;
    } else {
      above = mid;
    }
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

// Vectors [v0, v1) of the row into the list, which then has the k first of them among its entries (all of them if there
// are fewer than k). kSum: the thread's share of sum_j 2^(l_j * log2_scale - ref) goes to (ref, sum).
template <typename T, bool kSum>
__device__ void stream_top(TopShared& s, const RowVectors<T>& row, int v0, int v1, int k, float log2_scale, float& ref,
                           float& sum) {
  constexpr int kBatch = kTopThreads * kTopUnroll;
  const T* tag = nullptr;
  const int limit = min(2 * k + 64, kTopFull);
  __syncthreads();
  if (threadIdx.x == 0) {
    s.count = 0;
    s.bound = 0;
  }
  uint4 cur[kTopUnroll], nxt[kTopUnroll];
  auto fetch = [&](int vb, uint4(&to)[kTopUnroll]) {
#pragma unroll
    for (int u = 0; u < kTopUnroll; ++u) {
      const int v = vb + u * kTopThreads + int(threadIdx.x);
      to[u] = v < v1 ? row.load(v) : RowVectors<T>::nothing();
    }
  };
  ref = -INFINITY;
  sum = 0.f;
  fetch(v0, cur);
  __syncthreads();
  float bound = -INFINITY;
  for (int vb = v0; vb < v1; vb += kBatch) {
    if (vb + kBatch < v1) fetch(vb + kBatch, nxt);
    float top[kTopUnroll];
#pragma unroll
    for (int u = 0; u < kTopUnroll; ++u) top[u] = largest(cur[u], tag);
    if (kSum) {
      float m = ref;
#pragma unroll
      for (int u = 0; u < kTopUnroll; ++u) m = fmaxf(m, top[u] * log2_scale);  // passes a NaN over
      if (m > ref) {
        sum *= fast_exp2(ref - m);
        ref = m;
      }
      const float minus = ref > -INFINITY ? -ref : 0.f;
#pragma unroll
      for (int u = 0; u < kTopUnroll; ++u) {
        float f[RowVectors<T>::kPer];
        unpack(cur[u], f, tag);
#pragma unroll
        for (int i = 0; i < RowVectors<T>::kPer; ++i) sum += fast_exp2(fmaf(f[i], log2_scale, minus));
      }
    }
    if (vb == v0 && v1 - v0 > kTopThreads && k <= kTopThreads * kTopUnroll / 2) {
      // the k-th largest of the vectors' maxima (vectors that do not exist count as nothing)
      uint32_t key[kTopUnroll];
#pragma unroll
      for (int u = 0; u < kTopUnroll; ++u)
        key[u] = vb + u * kTopThreads + int(threadIdx.x) < v1 ? order_key(top[u]) : 0u;
      uint32_t least = 0xffffffffu, most = 0;
#pragma unroll
      for (int u = 0; u < kTopUnroll; ++u) {
        least = min(least, key[u]);
        most = max(most, key[u]);
      }
      const uint32_t from = bound_for(s, k, k / 4 + 4, least, most, [&](uint32_t b) {
        int c = 0;
#pragma unroll
        for (int u = 0; u < kTopUnroll; ++u) c += key[u] >= b;
        return c;
      });
      if (threadIdx.x == 0) s.bound = from;
      __syncthreads();
      bound = bound_value(from);
    }
    bool full = false;
#pragma unroll
    for (int u = 0; u < kTopUnroll; ++u) {
      const int v = vb + u * kTopThreads + int(threadIdx.x);
      if (!(top[u] < bound) && v < v1) {
        const uint32_t key = order_key(top[u]);
        if (key >= s.bound) {
          const unsigned int at = atomicAdd(&s.count, 1u);
          s.list[at] = order_pair(key, uint32_t(v));
          full |= at >= unsigned(limit);
        }
      }
    }
    if (__syncthreads_or(full)) {
      const uint32_t from = cut_list(s, s.list, s.count, k, limit);
      if (threadIdx.x == 0) s.bound = (unsigned long long)from + 1;
      __syncthreads();
      bound = bound_value(s.bound);
    }
#pragma unroll
    for (int u = 0; u < kTopUnroll; ++u) cur[u] = nxt[u];
  }
  __syncthreads();
}

// The list's vectors read again: s.elements then holds the k first logits of the row (all of them if there are fewer),
// sorted, s.n_elements of them.
template <typename T>
__device__ __forceinline__ void rank_elements(TopShared& s, const RowVectors<T>& row, int k) {
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
  constexpr int kStep = kTopMax / RowVectors<T>::kPer;  // vectors at a time: their logits fit beside what is kept
  static_assert(kStep <= kTopThreads, "one vector per thread");
  int m = 0;
  for (int i0 = 0; i0 < n; i0 += kStep) {
    const int i = i0 + int(threadIdx.x);
    if (int(threadIdx.x) < kStep && i < n) {
      const int v = int(pair_index(s.list[i]));
      const int e = row.first_of(v);
      float f[RowVectors<T>::kPer];
      unpack(row.load(v), f, static_cast<const T*>(nullptr));
#pragma unroll
      for (int j = 0; j < RowVectors<T>::kPer; ++j) {
        const uint32_t key = order_key(f[j]);
        if (key >= from && e + j >= 0 && uint32_t(e + j) < row.vocab)
          s.elements[atomicAdd(&s.n_elements, 1u)] = order_pair(key, uint32_t(e + j));
      }
    }
    __syncthreads();
    m = int(s.n_elements);
    __syncthreads();
    if (i0 + kStep < n && m > kTopMax) from = cut_list(s, s.elements, s.n_elements, k, kTopMax);
  }
  if (m <= kTopThreads) {
    // few: every entry's place is the number of entries ahead of it
    __syncthreads();
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
