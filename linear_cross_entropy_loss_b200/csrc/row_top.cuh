// The k largest logits of a row, found while the row streams past once: a short list in shared memory collects every
// logit that may still be among the k largest, and its bound rises as the row goes on.
//
// * The row is read in batches of kTopThreads * kTopUnroll vectors of 16 bytes, the next batch on its way while one is
//   looked at. One comparison of a vector's maximum with the bound decides for all its elements, so the elements cost
//   no more than their share of the log-sum-exp (or nothing where that is not wanted).
// * The first bound comes from the first batch: the k-th largest of its vectors' maxima. At least k elements reach it, and of
//   a row of random order about k per batch do.
// * When the list runs full it is cut back to the k first of the order, and from then on only larger logits enter:
//   an equal one that comes later has a higher index. A batch that would overflow the list (rows in rising order, or
//   many equal logits) is taken again vector by vector.
// A row may be split over the blocks of a cluster; the first block then takes the others' lists.
#pragma once

#include "ptx.cuh"
#include "vocab_row.cuh"

#include <type_traits>

namespace lce {

constexpr int kTopMax = 1024;
constexpr int kTopThreads = 256;
constexpr int kTopUnroll = 4;
constexpr int kTopList = 4096;             // entries of the list
constexpr int kTopFull = kTopList / 2;     // cut back above this: one more step of 256 vectors still fits
static_assert(kTopFull >= kTopMax && kTopFull + kTopThreads * 8 <= kTopList, "a step has to fit the list");

struct TopShared {
  unsigned long long list[kTopList];
  unsigned int counters[34];
  unsigned int range[2];
  unsigned int count;
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

// Smallest range [lo, ...] of keys that `count_from` says holds at least k entries, or one close to it: stops where the
// number lies in k .. k + slack. count_from(key): this thread's number of entries >= key.
template <typename CountFrom>
__device__ __forceinline__ uint32_t bound_for(TopShared& s, int k, int slack, uint32_t lo, uint32_t hi,
                                              CountFrom count_from) {
  // entries >= lo: at least k (the caller sees to it); entries > hi: none
  if (threadIdx.x < 34) s.counters[threadIdx.x] = 0;
  __syncthreads();
  unsigned long long above = (unsigned long long)hi + 1;  // fewer than k from here on
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

// Keeps the entries of the list for which stay(entry) holds, in place: chunk by chunk, each read before any place up to
// its end is written.
template <typename Stay>
__device__ __forceinline__ void filter_list(TopShared& s, int n, Stay stay) {
  __syncthreads();
  if (threadIdx.x == 0) s.count = 0;
  for (int i0 = 0; i0 < n; i0 += kTopThreads) {
    const int at = i0 + int(threadIdx.x);
    const unsigned long long e = at < n ? s.list[at] : 0;
    __syncthreads();
    if (at < n && stay(e)) s.list[atomicAdd(&s.count, 1u)] = e;
  }
  __syncthreads();
}

// Leaves at least the k first entries of the order in the list, and few more unless many are equal.
__device__ __forceinline__ void thin_list(TopShared& s, int k) {
  __syncthreads();
  const int n = min(int(s.count), kTopList);
  if (n <= k + k / 4 + 32) return;
  if (threadIdx.x == 0) {
    s.range[0] = 0xffffffffu;
    s.range[1] = 0;
  }
  uint32_t least = 0xffffffffu, most = 0;
  for (int i = threadIdx.x; i < n; i += kTopThreads) {
    const uint32_t key = pair_key(s.list[i]);
    least = min(least, key);
    most = max(most, key);
  }
  __syncthreads();
  least = __reduce_min_sync(0xffffffffu, least);
  most = __reduce_max_sync(0xffffffffu, most);
  if ((threadIdx.x & 31) == 0) {
    atomicMin(&s.range[0], least);
    atomicMax(&s.range[1], most);
  }
  __syncthreads();
  const uint32_t from = bound_for(s, k, k / 4 + 16, s.range[0], s.range[1], [&](uint32_t key) {
    int c = 0;
    for (int i = threadIdx.x; i < n; i += kTopThreads) c += pair_key(s.list[i]) >= key;
    return c;
  });
  filter_list(s, n, [&](unsigned long long e) { return pair_key(e) >= from; });
}

// Sorts the list and cuts it to its first k entries.
__device__ __forceinline__ void sort_list(TopShared& s, int k) {
  __syncthreads();
  const int n = min(int(s.count), kTopList);
  int padded = 2;
  while (padded < n) padded <<= 1;
  for (int i = n + threadIdx.x; i < padded; i += kTopThreads) s.list[i] = 0;
  block_sort_descending(s.list, padded);
  if (threadIdx.x == 0) s.count = min(n, k);
  __syncthreads();
}

// Cuts a full list back to its first k entries and raises the bound above the last of them.
__device__ __noinline__ void cut_list(TopShared& s, int k) {
  thin_list(s, k);
  sort_list(s, k);
  if (threadIdx.x == 0 && int(s.count) == k) s.bound = (unsigned long long)pair_key(s.list[k - 1]) + 1;
  __syncthreads();
}

template <typename T>
__device__ __forceinline__ bool enter_list(TopShared& s, const RowVectors<T>& row, int v, const uint4& raw) {
  float f[RowVectors<T>::kPer];
  unpack(raw, f, static_cast<const T*>(nullptr));
  const unsigned long long bound = s.bound;
  const int e = row.first_of(v);
  bool full = false;
#pragma unroll
  for (int i = 0; i < RowVectors<T>::kPer; ++i) {
    const uint32_t key = order_key(f[i]);
    if (key >= bound && e + i >= 0 && uint32_t(e + i) < row.vocab) {
      const unsigned int at = atomicAdd(&s.count, 1u);
      if (at < unsigned(kTopList)) s.list[at] = order_pair(key, uint32_t(e + i));
      full |= at >= unsigned(kTopFull);
    }
  }
  return full;
}

// The bound as a float that a vector's maximum can be held against: !(maximum < it) where an element may enter.
__device__ __forceinline__ float bound_value(unsigned long long bound) {
  if (bound <= kKeyNegInf) return -INFINITY;
  return bound <= 0xffffffffull ? key_to_float(uint32_t(bound)) : __uint_as_float(0x7fc00000u);
}

// Vectors [v0, v1) of the row into the list, which then holds this part's k largest among its entries (all of
// them if there are fewer than k). kSum: the thread's share of sum_j 2^(l_j * log2_scale - ref) goes to (ref, sum).
template <typename T, bool kSum>
__device__ void stream_top(TopShared& s, const RowVectors<T>& row, int v0, int v1, int k, float log2_scale, float& ref,
                           float& sum) {
  constexpr int kBatch = kTopThreads * kTopUnroll;
  const T* tag = nullptr;
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
      const uint32_t from = bound_for(s, k, k / 4 + 4, 0u, 0xffffffffu, [&](uint32_t b) {
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
      if (!(top[u] < bound) && v < v1) full |= enter_list(s, row, v, cur[u]);
    }
    if (__syncthreads_or(full)) {
      if (s.count <= unsigned(kTopList)) {
        cut_list(s, k);
      } else {
        // more than the list holds: what was there before this batch, then the batch vector by vector
        // (of the entries of earlier batches none was lost: they had their places before this batch began)
        const int before = row.first_of(vb);  // the batch's first element
        filter_list(s, kTopList, [&](unsigned long long e) { return before > 0 && pair_index(e) < uint32_t(before); });
#pragma unroll
        for (int u = 0; u < kTopUnroll; ++u) {
          const int v = vb + u * kTopThreads + int(threadIdx.x);
          if (v < v1) enter_list(s, row, v, cur[u]);
          __syncthreads();
          const bool cut = s.count > unsigned(kTopFull);
          __syncthreads();
          if (cut) cut_list(s, k);
        }
      }
      bound = bound_value(s.bound);
      __syncthreads();
    }
#pragma unroll
    for (int u = 0; u < kTopUnroll; ++u) cur[u] = nxt[u];
  }
  __syncthreads();
}

}  // namespace lce
