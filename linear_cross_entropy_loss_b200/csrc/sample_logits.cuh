// sample_logits: one token of each row, drawn with a given random number after temperature, top-k, top-p and min-p.
//   w_j = exp((l_j - max) / T); order: logit descending, index ascending
//   kept: the first top_k of the order; of those the shortest prefix that holds top_p of their mass; of those w >= min_p
//   token = the first j in index order at which the kept weights, added up, exceed u * (their sum)
//
// Rows with a short list (top_k up to `list_limit`, or greedy) go through the search of top_logits and are drawn from
// the sorted list (sample_list_kernel). All others keep the row in shared memory, spread over a cluster, and sweep
// over it (sample_row_kernel): the largest logit; a histogram over the order for each cut; the kept weights; the
// place of the token.
//
// What bounds it: not the memory. A row's weights are taken in 64 bits (vocab_row.cuh says why), about 35
// instructions each, and the sweeps of a block follow one another with a barrier of the cluster between them. 64 x
// 131072 fp32, top-p 0.95: 70 us, of which the histogram with all weights takes 24,000 of a block's 60,000 cycles,
// finding the place in its bin 13,500, the kept weights 10,500; two blocks of 512 threads fit an SM and 512 of them
// make two waves. 1024 x 32768 fp16, min-p: 51 us; min-p leaves few, so their weights are taken 32 at a time after a
// warp has moved them together. Lists: 256 x 131072 bf16, top-k 50: 24 us.
#pragma once

#include "row_top.cuh"

namespace lce {

struct SampleParams {
  const void* u;             // [rows] float or double in [0, 1)
  int u_is_double;
  const float* temperature;  // [rows], or null: the value for all rows
  const int* top_k;
  const float* top_p;
  const float* min_p;
  double temperature_all;
  double top_p_all;
  double min_p_all;
  long long top_k_all;
  int weight_bits;
  int list_limit;            // rows with 1 <= top_k <= list_limit (greedy ones count as 1) go through the list
};

// One row's settings, with whatever stands outside their range taken as the nearest that means something.
struct RowSettings {
  double temperature;
  double top_p;   // >= 1: no cut
  double lowest;  // least weight_steps of a kept token
  double u;
  long long top_k;  // 0: no cut
  bool greedy;
};
__device__ __forceinline__ RowSettings row_settings(const SampleParams& p, long long r) {
  RowSettings s;
  s.temperature = p.temperature ? double(p.temperature[r]) : p.temperature_all;
  s.top_k = p.top_k ? p.top_k[r] : p.top_k_all;
  s.top_p = p.top_p ? double(p.top_p[r]) : p.top_p_all;
  const double min_p = p.min_p ? double(p.min_p[r]) : p.min_p_all;
  s.lowest = min_p > 0.0 ? kSteps * log2(fmin(min_p, 1.0)) : -INFINITY;
  s.u = p.u_is_double ? reinterpret_cast<const double*>(p.u)[r] : double(reinterpret_cast<const float*>(p.u)[r]);
  s.u = s.u > 0.0 ? fmin(s.u, 1.0) : 0.0;
  s.greedy = !(s.temperature > 0.0);
  if (s.greedy) {
    s.temperature = 1.0;
    s.top_k = 1;
  }
  if (s.top_k < 0) s.top_k = 0;
  if (!(s.top_p < 1.0)) s.top_p = 1.0;
  return s;
}
__device__ __forceinline__ bool by_list(const SampleParams& p, const RowSettings& s) {
  return s.top_k >= 1 && s.top_k <= p.list_limit;
}
__device__ __forceinline__ RowWeights row_weights(const SampleParams& p, const RowSettings& s, float largest,
                                                  const double* table) {
  RowWeights w;
  w.largest = largest;
  w.only_largest = largest == INFINITY;
  w.steps = fmin(1.0 / (kStepLn2 * s.temperature), 1e300);
  w.to_int = __hiloint2double((1023 + 52 - p.weight_bits) << 20, 0);  // 2^(52 - bits)
  w.table = smem_u32(table);
  return w;
}
// Smallest prefix whose mass reaches top_p of the whole.
__device__ __forceinline__ unsigned long long mass_target(double top_p, unsigned long long mass) {
  const double goal = ceil(fmax(top_p, 0.0) * double(mass));
  const unsigned long long target = goal < 1.0 ? 1ull : (unsigned long long)goal;
  return target < mass ? target : mass;
}
__device__ __forceinline__ unsigned long long draw_target(double u, unsigned long long total) {
  const unsigned long long goal = (unsigned long long)(u * double(total));
  return goal < total ? goal : total - 1;
}
__device__ __forceinline__ float log_share(const SampleParams& p, const RowSettings& s, const RowWeights& w, float logit,
                                           unsigned long long weight, unsigned long long total) {
  if (s.greedy) return 0.f;
  if (w.only_largest) return float(log(double(weight) / double(total)));  // all shares alike
  return float(weight_steps(w, logit) * kStepLn2 - log(ldexp(double(total), -p.weight_bits)));
}
__device__ __forceinline__ void draw_nothing(long long r, long long* tokens, float* logprobs) {
  tokens[r] = -1;
  logprobs[r] = -INFINITY;
}

// ---------------------------------------------------------------------------------------------
// rows with a short list
// ---------------------------------------------------------------------------------------------
template <typename T>
__global__ void __launch_bounds__(kTopThreads, 3)
sample_list_kernel(const T* __restrict__ logits, long long ld, uint32_t vocab, int parts, const SampleParams p,
                   long long* __restrict__ tokens, float* __restrict__ logprobs) {
  extern __shared__ __align__(16) unsigned char dynamic[];
  TopShared& s = *reinterpret_cast<TopShared*>(dynamic);
  __shared__ double table[kSteps];
  __shared__ unsigned long long reduce[32];
  const long long r = blockIdx.x / parts;
  const int part = int(blockIdx.x % parts);
  const RowSettings set = row_settings(p, r);
  // (sample_row_kernel, launched behind this one, has other rows and may start)
  asm volatile("griddepcontrol.launch_dependents;");
  if (!by_list(p, set)) return;  // the whole cluster
  const int k = int(min((long long)vocab, set.top_k));
  const RowGroups<T> row(logits + r * ld, vocab);
  const int v0 = int((long long)row.groups * part / parts), v1 = int((long long)row.groups * (part + 1) / parts);
  float ref, sum;
  if (threadIdx.x < kSteps) table[threadIdx.x] = exp2(double(threadIdx.x) / kSteps);
  stream_top<T, false, Nan::kNever>(s, row, v0, v1, parts, k, 1.f, ref, sum);
  const TopGroups g = merge_lists(s, k, parts);
  if (part != 0) return;
  const int n = rank_elements<Nan::kNever>(s, row, g, k);
  const unsigned long long* const elements = g.free_list;
  const uint32_t first = pair_key(elements[0]);
  if (first == kKeyNegInf) {
    if (threadIdx.x == 0) draw_nothing(r, tokens, logprobs);
    return;
  }
  const RowWeights w = row_weights(p, set, key_to_float(first), table);
  // thread t has the ranks 4 t .. 4 t + 3
  constexpr int kEach = kTopMax / kTopThreads;
  unsigned long long mine[kEach], sum4 = 0;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int rank = kEach * int(threadIdx.x) + i;
    mine[i] = rank < n ? row_weight(w, key_to_float(pair_key(elements[rank]))) : 0ull;
    sum4 += mine[i];
  }
  unsigned long long mass;
  unsigned long long before = block_prefix(sum4, reduce, &mass);
  const unsigned long long target = set.top_p < 1.0 ? mass_target(set.top_p, mass) : mass;
  unsigned long long* weights = g.list;            // by rank; 0 where a token is not kept
  unsigned long long* by_index = g.list + kTopMax;
  sum4 = 0;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int rank = kEach * int(threadIdx.x) + i;
    bool keep = before < target;
    if (rank < n && !w.only_largest)
      keep = keep && weight_steps(w, key_to_float(pair_key(elements[rank]))) >= set.lowest;
    before += mine[i];
    if (!keep) mine[i] = 0;
    weights[rank] = mine[i];
    sum4 += mine[i];
  }
  const unsigned long long total = block_sum(sum4, reduce);
  const unsigned long long goal = draw_target(set.u, total);
  // the kept weights are a prefix of the ranks; in index order they are added up
  int kept = 0;
#pragma unroll
  for (int i = 0; i < kEach; ++i) kept += mine[i] != 0;
  kept = int(block_sum((unsigned long long)kept, reduce));
  if (kept <= kTopThreads) {
    const int i = int(threadIdx.x);
    if (i < kept) {
      const uint32_t index = pair_index(elements[i]);
      unsigned long long at = 0;
      for (int j = 0; j < kept; ++j) at += pair_index(elements[j]) < index ? weights[j] : 0ull;
      if (at <= goal && goal < at + weights[i]) {
        tokens[r] = index;
        logprobs[r] = log_share(p, set, w, key_to_float(pair_key(elements[i])), weights[i], total);
      }
    }
  } else {
    for (int i = threadIdx.x; i < kept; i += kTopThreads)
      by_index[i] = order_pair(0xffffffffu - pair_index(elements[i]), uint32_t(i));
    block_sort_descending<kTopThreads>(by_index, kept);
    sum4 = 0;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int at = kEach * int(threadIdx.x) + i;
      mine[i] = at < kept ? weights[pair_index(by_index[at])] : 0ull;
      sum4 += mine[i];
    }
    before = block_prefix(sum4, reduce, &mass);
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      if (mine[i] != 0 && before <= goal && goal < before + mine[i]) {
        const unsigned long long e = elements[pair_index(by_index[kEach * int(threadIdx.x) + i])];
        tokens[r] = pair_index(e);
        logprobs[r] = log_share(p, set, w, key_to_float(pair_key(e)), mine[i], total);
      }
      before += mine[i];
    }
  }
}

// ---------------------------------------------------------------------------------------------
// all other rows
// ---------------------------------------------------------------------------------------------
constexpr int kRowThreads = 512;
constexpr int kRowWarps = kRowThreads / 32;
constexpr int kRowBins = 2048;
constexpr int kRowList = 2048;
constexpr int kRowPieces = 64;  // of a warp's stretch: kept weights are added up for each
constexpr int kRowParts = 8;
constexpr int kRowCoarse = kRowBins / 32;
constexpr int kRowCompact = 2 * kRowList / kRowWarps;

// A stretch of the order that starts at its top: logits above `value`, and equal ones with an index below `end`.
struct RowCut {
  float value;
  uint32_t end;
};
constexpr uint32_t kNoEnd = 0xffffffffu;
__device__ __forceinline__ bool inside(const RowCut& c, float l, uint32_t index) {
  if (!(l >= c.value)) return false;  // also a NaN
  return c.end == kNoEnd || l > c.value || index < c.end;
}

struct RowShared {
  union {
    struct {
      uint32_t low[kRowBins + 32], high[kRowBins + 32];  // a 64-bit sum in two words; 32 more for what is left out
    } bins;
    unsigned long long gathered[kRowList];          // all blocks' lists
    uint32_t together[kRowWarps][kRowCompact];      // indices of what a warp keeps, ascending
  };
  unsigned long long list[kRowList];  // this block's elements of one bin, order_pair(key, index)
  unsigned long long pieces[kRowWarps * kRowPieces];
  unsigned long long reduce[32];
  float reduce_f[32];
  double table[kSteps];
  // written by the blocks of the cluster, each into its own place
  float part_max[kRowParts];
  unsigned long long part_sum[kRowParts];
  uint32_t part_least[kRowParts], part_most[kRowParts], part_listed[kRowParts];
  unsigned long long part_coarse[kRowParts][kRowCoarse];  // sums over 32 bins
  // written by one block into all
  RowCut found_cut;
  // this block's own
  unsigned long long coarse[kRowCoarse];
  unsigned long long found_before, found_total;
  uint32_t found_bin;
  unsigned int listed;
  uint32_t piece;
  unsigned long long piece_before;
};

__device__ __forceinline__ uint4 load_piece(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
__device__ __forceinline__ void copy_async16(void* smem, const void* global) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(smem)), "l"(global) : "memory");
}
__device__ __forceinline__ void copy_async_wait() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// One block's stretch of a row in vectors of 16 bytes, each warp's stretch of it in turn contiguous, so that the order
// of blocks, warps, steps, lanes and elements is the order of the indices.
template <typename T>
struct RowStretch {
  static constexpr int kPer = 16 / int(sizeof(T));
  const T* row;
  uint32_t vocab;
  int lead;        // elements between the 16-byte boundary below the row and its start
  int begin, end;  // this warp's vectors
  int steps;       // of 32 vectors
  int per_piece;   // steps of a piece
  uint4* cache;    // this lane's vector of step 0, or null: the row is read from global memory each time
  const T* flat;   // element e of this block's stretch at flat[e], in the cache or in the row

  __device__ __forceinline__ uint4 load(int v) const {
    const long long e = (long long)v * kPer - lead;
    if (e >= 0 && e + kPer <= (long long)vocab) return load_piece(row + e);
    constexpr uint32_t none = RowGroups<T>::kNegInf;
    uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const bool exists = e + i >= 0 && e + i < (long long)vocab;
      const uint32_t b = exists ? uint32_t(reinterpret_cast<const typename RowGroups<T>::Bits*>(row)[e + i]) : none;
      w[i * int(sizeof(T)) / 4] |= b << (8 * (i * int(sizeof(T)) % 4));
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  static __device__ __forceinline__ void unpack(const uint4& raw, float (&l)[kPer]) {
    if constexpr (sizeof(T) == 4) {
      l[0] = __uint_as_float(raw.x); l[1] = __uint_as_float(raw.y);
      l[2] = __uint_as_float(raw.z); l[3] = __uint_as_float(raw.w);
    } else {
      const T* tag = nullptr;
      halves(raw.x, l[0], l[1], tag);
      halves(raw.y, l[2], l[3], tag);
      halves(raw.z, l[4], l[5], tag);
      halves(raw.w, l[6], l[7], tag);
    }
  }
  // The largest of this lane's elements, -inf where there is none (a NaN is none).
  __device__ __forceinline__ float largest() const {
    constexpr uint32_t none = sizeof(T) == 4 ? RowGroups<T>::kNegInf : RowGroups<T>::kNegInf * 0x10001u;
    uint4 m = make_uint4(none, none, none, none);
    for (int step = 0; step < steps; ++step) {
      const int v = begin + step * 32 + int(threadIdx.x & 31);
      if (v >= end) break;
      const uint4 raw = cache != nullptr ? cache[step * 32] : load(v);
      m.x = larger_of_word(m.x, raw.x);
      m.y = larger_of_word(m.y, raw.y);
      m.z = larger_of_word(m.z, raw.z);
      m.w = larger_of_word(m.w, raw.w);
    }
    float l[kPer];
    unpack(m, l);
    float r = l[0];
#pragma unroll
    for (int i = 1; i < kPer; ++i) r = fmaxf(r, l[i]);
    return r;
  }
  static __device__ __forceinline__ uint32_t larger_of_word(uint32_t a, uint32_t b) {
    if constexpr (sizeof(T) == 4) {
      return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
    } else {
      using T2 = std::conditional_t<std::is_same<T, __half>::value, __half2, __nv_bfloat162>;
      const T2 r = __hmax2(*reinterpret_cast<T2*>(&a), *reinterpret_cast<T2*>(&b));
      return *reinterpret_cast<const uint32_t*>(&r);
    }
  }
  // f(first element's index, the elements) for this lane's vector of a step; elements outside the row are -inf.
  template <typename F>
  __device__ __forceinline__ void at_step(int step, F f) const {
    const int v = begin + step * 32 + int(threadIdx.x & 31);
    if (v >= end) return;
    float l[kPer];
    unpack(cache != nullptr ? cache[step * 32] : load(v), l);
    f(uint32_t(v * kPer - lead), l);
  }
  // f(index, logit) for the elements of a step with test(logit). Few of many: a lane takes its next one while others
  // take theirs, so a step costs as many rounds as one lane has elements, not one for each place.
  template <typename Test, typename F>
  __device__ __forceinline__ void some_at_step(int step, Test test, F f) const {
    at_step(step, [&](uint32_t index, float(&l)[kPer]) {
      uint32_t hits = 0;
#pragma unroll
      for (int i = 0; i < kPer; ++i) hits |= test(l[i]) ? 1u << i : 0u;
      while (hits != 0) {
        const int at = __ffs(hits) - 1;
        hits &= hits - 1;
        float value = l[0];
#pragma unroll
        for (int i = 1; i < kPer; ++i)
          if (at == i) value = l[i];
        f(index + at, value);
      }
    });
  }
};

struct RowCluster {
  cooperative_groups::cluster_group group;
  int rank, parts;
  RowShared& s;
  __device__ __forceinline__ RowShared& of(int part) const { return *group.map_shared_rank(&s, part); }
};

// The smallest float up to `largest` for which holds(float) is true; it is true for `largest` and, once true, for all
// larger ones. All lanes of a warp take part: they try the floats around the estimate, or, where the border is not
// among them, cut the whole range into 32 parts at a time.
template <typename Holds>
__device__ __forceinline__ float border_of(float estimate, float largest, Holds holds) {
  const int lane = int(threadIdx.x & 31);
  uint32_t left = kKeyNegInf + 1, right = order_key(largest);
  {
    const uint32_t mid = min(max(order_key(estimate), left + 16), right);
    const uint32_t at = min(mid - 16 + uint32_t(lane), right);
    const uint32_t yes = __ballot_sync(0xffffffffu, holds(key_to_float(at)));
    if (yes != 0 && (yes & 1u) == 0) return key_to_float(min(mid - 16 + uint32_t(__ffs(yes) - 1), right));
  }
  while (left < right) {
    const uint32_t width = (right - left) / 32 + 1;
    const uint32_t at = left + min(width * uint32_t(lane), right - left);
    const uint32_t yes = __ballot_sync(0xffffffffu, holds(key_to_float(at)));
    const uint32_t none = yes != 0 ? __ffs(yes) - 1 : 32u;  // lanes below the border
    if (none < 32) right = left + min(width * none, right - left);
    if (none > 0) left = min(left + width * (none - 1) + 1, right);
  }
  return key_to_float(right);
}
// The smallest logit whose weight_steps are at least `least` (<= 0): what a comparison of logits has to use for the
// comparison of the steps.
__device__ __forceinline__ float logit_from_steps(const RowWeights& w, double inv_steps, float largest, double least) {
  if (w.only_largest) return largest;
  return border_of(float(w.largest + least * inv_steps), largest,
                   [&](float l) { return weight_steps(w, l) >= least; });
}

struct Crossing {
  uint32_t bin;
  unsigned long long before;  // what lies in the bins ahead of it
  unsigned long long total;
};

// Sums amount(logit) by bin(logit) over the elements of the row that `active` selects and finds the bin in which
// target(total) is reached, bin 0 first. The 64-bit sums are kept in two words, the carry passed on by the one who
// causes it.
template <typename T, typename Amount, typename Bin, typename Active, typename Target>
__device__ __forceinline__ Crossing find_bin(const RowCluster& c, const RowStretch<T>& x, Amount amount, Bin bin,
                                             Active active, Target target) {
  RowShared& s = c.s;
  __syncthreads();
  for (int i = threadIdx.x; i < kRowBins; i += kRowThreads) s.bins.low[i] = s.bins.high[i] = 0;
  __syncthreads();
  const uint32_t spare = uint32_t(kRowBins) + (threadIdx.x & 31);
  for (int step = 0; step < x.steps; ++step)
    x.at_step(step, [&](uint32_t index, float(&l)[RowStretch<T>::kPer]) {
      // Four elements side by side, without branches: what is not active goes, whatever its amount comes out as, to a
      // word of the lane's own. The answer of the first word's addition (a carry) is only looked at when all four are on
      // their way.
#pragma unroll
      for (int i0 = 0; i0 < RowStretch<T>::kPer; i0 += 4) {
        uint32_t at[4], low[4], high[4], was[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const unsigned long long a = amount(l[i0 + i]);
          at[i] = active(index + i0 + i, l[i0 + i]) ? bin(l[i0 + i]) : spare;
          low[i] = uint32_t(a);
          high[i] = uint32_t(a >> 32);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) was[i] = atomicAdd(&s.bins.low[at[i]], low[i]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          high[i] += was[i] + low[i] < was[i] ? 1u : 0u;
          if (high[i] != 0) atomicAdd(&s.bins.high[at[i]], high[i]);
        }
      }
    });
  __syncthreads();
  // Sums over 32 bins go to all blocks; behind the barrier every block finds the 32 bins in question by itself, reads
  // those of all blocks and finds the bin. (Reading and adding up all bins instead, a share per block, took two more
  // barriers and 9,000 cycles against 3,000.)
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
  for (int i = 0; i < kRowCoarse / kRowWarps; ++i) {
    const int g = i * kRowWarps + warp, b = g * 32 + lane;
    unsigned long long v = ((unsigned long long)s.bins.high[b] << 32) + s.bins.low[b];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (lane < c.parts) c.of(lane).part_coarse[c.rank][g] = v;
  }
  c.group.sync();
  if (threadIdx.x < kRowCoarse) {
    unsigned long long v = 0;
    for (int part = 0; part < c.parts; ++part) v += s.part_coarse[part][threadIdx.x];
    s.coarse[threadIdx.x] = v;
  }
  __syncthreads();
  auto prefix = [&](unsigned long long v) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned long long other = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += other;
    }
    return v;
  };
  unsigned long long goal = 0;
  if (warp == 0) {
    static_assert(kRowCoarse == 64, "two per lane");
    const unsigned long long v0 = s.coarse[2 * lane], v1 = s.coarse[2 * lane + 1];
    const unsigned long long end = prefix(v0 + v1);
    const unsigned long long total = __shfl_sync(0xffffffffu, end, 31);
    goal = target(total);
    const unsigned long long before0 = end - v1 - v0, before1 = end - v1;
    if (before0 < goal && goal <= before1) {
      s.found_bin = 2 * lane;
      s.found_before = before0;
    } else if (before1 < goal && goal <= end) {
      s.found_bin = 2 * lane + 1;
      s.found_before = before1;
    }
    if (lane == 0) s.found_total = total;
  }
  __syncthreads();
  Crossing found;
  found.total = s.found_total;
  const uint32_t group = s.found_bin;
  if (warp == 0) {
    unsigned long long v = 0;
#pragma unroll
    for (int part = 0; part < kRowParts; ++part) {
      if (part < c.parts) {
        const RowShared& other = c.of(part);
        v += ((unsigned long long)other.bins.high[group * 32 + lane] << 32) + other.bins.low[group * 32 + lane];
      }
    }
    const unsigned long long end = s.found_before + prefix(v);
    __syncwarp();
    if (end - v < goal && goal <= end) {
      s.found_bin = group * 32 + lane;
      s.found_before = end - v;
    }
  }
  __syncthreads();
  found.bin = s.found_bin;
  found.before = s.found_before;
  return found;
}

// The logits of a bin.
struct RowBin {
  float from, below;  // below: NaN where it goes up to +inf
  __device__ __forceinline__ bool has(float l) const { return l >= from && !(l >= below); }
};

// The place in the order at which the amounts reach `target`, given that this happens among the elements of `bin` inside
// `outer` and that `before` lies ahead of them.
template <typename T, typename Amount>
__device__ __forceinline__ RowCut find_place(const RowCluster& c, const RowStretch<T>& x, unsigned long long before,
                                             unsigned long long target, Amount amount, const RowBin bin,
                                             const RowCut outer) {
  RowShared& s = c.s;
  float from = bin.from, to = INFINITY;  // logits that still matter
  for (;;) {
    __syncthreads();
    if (threadIdx.x == 0) s.listed = 0;
    __syncthreads();
    uint32_t least = 0xffffffffu, most = 0;
    for (int step = 0; step < x.steps; ++step)
      x.some_at_step(
          step, [&](float l) { return l >= from && !(l >= bin.below); },
          [&](uint32_t index, float l) {
            if (l > to || !inside(outer, l, index)) return;
            const uint32_t key = order_key(l);
            least = min(least, key);
            most = max(most, key);
            const unsigned int at = atomicAdd(&s.listed, 1u);
            if (at < unsigned(kRowList)) s.list[at] = order_pair(key, index);
          });
    least = __reduce_min_sync(0xffffffffu, least);
    most = __reduce_max_sync(0xffffffffu, most);
    uint32_t* scratch = reinterpret_cast<uint32_t*>(s.reduce);
    if ((threadIdx.x & 31) == 0) {
      scratch[threadIdx.x >> 5] = least;
      scratch[32 + (threadIdx.x >> 5)] = most;
    }
    __syncthreads();
    if (threadIdx.x < 32) {
      const int i = int(threadIdx.x) < kRowWarps ? int(threadIdx.x) : 0;
      least = __reduce_min_sync(0xffffffffu, scratch[i]);
      most = __reduce_max_sync(0xffffffffu, scratch[32 + i]);
      if (int(threadIdx.x) < c.parts) {
        RowShared& other = c.of(threadIdx.x);
        other.part_least[c.rank] = least;
        other.part_most[c.rank] = most;
        other.part_listed[c.rank] = s.listed;
      }
    }
    c.group.sync();
    unsigned int n = 0;
    least = 0xffffffffu;
    most = 0;
    for (int part = 0; part < c.parts; ++part) {
      n += s.part_listed[part];
      least = min(least, s.part_least[part]);
      most = max(most, s.part_most[part]);
    }
    if (n <= unsigned(kRowList)) {
      // few enough: every block takes them all, in any order, and finds the place by itself
      for (unsigned int i = threadIdx.x; i < n; i += kRowThreads) {
        unsigned int at = i;
        int part = 0;
        while (at >= s.part_listed[part]) at -= s.part_listed[part++];
        s.gathered[i] = c.of(part).list[at];
      }
      auto found = [&](unsigned long long e) {
        s.found_cut = RowCut{key_to_float(pair_key(e)), pair_index(e) + 1};
      };
      constexpr int kShare = 4;  // threads per element
      __syncthreads();
      if (n <= kRowThreads / kShare) {
        // every element's place is the sum of the amounts ahead of it
        if (threadIdx.x < n) s.pieces[threadIdx.x] = amount(key_to_float(pair_key(s.gathered[threadIdx.x])));
        __syncthreads();
        const unsigned int i = threadIdx.x / kShare;
        unsigned long long mine = 0, place = 0;
        if (i < n) {
          mine = s.gathered[i];
          for (unsigned int j = threadIdx.x % kShare; j < n; j += kShare)
            place += s.gathered[j] > mine ? s.pieces[j] : 0ull;
        }
#pragma unroll
        for (int o = 1; o < kShare; o <<= 1) place += __shfl_xor_sync(0xffffffffu, place, o);
        place += before;
        if (i < n && threadIdx.x % kShare == 0 && place < target && target <= place + s.pieces[i]) found(mine);
      } else {
        block_sort_descending<kRowThreads>(s.gathered, int(n));
        unsigned long long seen = before;
        for (int i0 = 0; i0 < int(n); i0 += kRowThreads) {
          const int i = i0 + int(threadIdx.x);
          unsigned long long a = 0;
          if (i < int(n)) a = amount(key_to_float(pair_key(s.gathered[i])));
          unsigned long long sum;
          const unsigned long long place = seen + block_prefix(a, s.reduce, &sum);
          if (a != 0 && place < target && target <= place + a) found(s.gathered[i]);
          seen += sum;
          if (seen >= target) break;
        }
      }
      __syncthreads();
      return s.found_cut;
    }
    if (least == most) {
      // one value: the m-th of its places
      const float value = key_to_float(least);
      const unsigned long long each = amount(value);
      const unsigned long long m = (target - before + each - 1) / each;
      auto is_one = [&](uint32_t index, float l) { return l == value && inside(outer, l, index); };
      unsigned long long mine = 0;
      for (int step = 0; step < x.steps; ++step)
        x.at_step(step, [&](uint32_t index, float(&l)[RowStretch<T>::kPer]) {
#pragma unroll
          for (int i = 0; i < RowStretch<T>::kPer; ++i) mine += is_one(index + i, l[i]);
        });
      // in index order: lanes of a step, steps, warps, blocks
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
      unsigned long long total;
      unsigned long long ahead = block_prefix((threadIdx.x & 31) == 0 ? mine : 0ull, s.reduce, &total);
      ahead = __shfl_sync(0xffffffffu, ahead, 0);
      if (int(threadIdx.x) < c.parts) c.of(threadIdx.x).part_sum[c.rank] = total;
      c.group.sync();
      for (int part = 0; part < c.rank; ++part) ahead += s.part_sum[part];
      if (ahead < m && m <= ahead + mine) {
        for (int step = 0; step < x.steps; ++step) {
          unsigned int here = 0;
          x.at_step(step, [&](uint32_t index, float(&l)[RowStretch<T>::kPer]) {
#pragma unroll
            for (int i = 0; i < RowStretch<T>::kPer; ++i) here += is_one(index + i, l[i]);
          });
          unsigned int inc = here;
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const unsigned int other = __shfl_up_sync(0xffffffffu, inc, o);
            if (int(threadIdx.x & 31) >= o) inc += other;
          }
          unsigned long long at = ahead + inc - here;
          if (at < m && m <= at + here)
            x.some_at_step(step, [&](float l) { return l == value; }, [&](uint32_t index, float l) {
              if (is_one(index, l) && ++at == m)
                for (int part = 0; part < c.parts; ++part) c.of(part).found_cut = RowCut{value, index + 1};
            });
          ahead += __shfl_sync(0xffffffffu, inc, 31);
        }
      }
      c.group.sync();
      return s.found_cut;
    }
    // too many of several values: a finer histogram over their keys
    int shift = 0;
    while (((most - least) >> shift) >= uint32_t(kRowBins)) ++shift;
    const float low = key_to_float(least), high = key_to_float(most);
    const uint32_t top_key = most;
    const Crossing at = find_bin(
        c, x, amount, [&](float l) { return (top_key - order_key(l)) >> shift; },
        [&](uint32_t index, float l) { return l >= low && l <= high && inside(outer, l, index); },
        [&](unsigned long long) { return target - before; });
    before += at.before;
    const uint32_t to_key = most - (at.bin << shift);
    const uint32_t down = (1u << shift) - 1u;
    to = key_to_float(to_key);
    from = key_to_float(to_key - least > down ? to_key - down : least);
  }
}

template <typename T>
__device__ __forceinline__ void sample_row(const T* __restrict__ logits, long long ld, uint32_t vocab, int parts,
                                           int cache_vectors, const SampleParams& p, long long* __restrict__ tokens,
                                           float* __restrict__ logprobs) {
  extern __shared__ __align__(16) unsigned char dynamic[];
  RowShared& s = *reinterpret_cast<RowShared*>(dynamic);
  const long long r = blockIdx.x / parts;
  const RowSettings set = row_settings(p, r);
  if (by_list(p, set)) return;  // the whole cluster
  cluster_started();
  RowCluster c{cooperative_groups::this_cluster(), int(blockIdx.x % parts), parts, s};
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int kPer = RowStretch<T>::kPer;

  RowStretch<T> x;
  x.row = logits + r * ld;
  x.vocab = vocab;
  x.lead = int((reinterpret_cast<uintptr_t>(x.row) & 15u) / sizeof(T));
  const int vectors = int(((long long)vocab + x.lead + kPer - 1) / kPer);
  const int per_block = (vectors + parts - 1) / parts;
  const int per_warp = (per_block + kRowThreads - 1) / kRowThreads * 32;
  const int block_begin = min(c.rank * per_block, vectors), block_end = min(block_begin + per_block, vectors);
  x.begin = min(block_begin + warp * per_warp, block_end);
  x.end = min(x.begin + per_warp, block_end);
  x.steps = (x.end - x.begin + 31) / 32;
  x.per_piece = (per_warp / 32 + kRowPieces - 1) / kRowPieces;
  x.cache = nullptr;
  x.flat = x.row;
  if (cache_vectors > 0) {
    uint4* const block_cache = reinterpret_cast<uint4*>(dynamic + (sizeof(RowShared) + 15) / 16 * 16);
    uint4* const cache = block_cache + (x.begin - block_begin) + lane;
    x.flat = reinterpret_cast<const T*>(block_cache) + (x.lead - (long long)block_begin * kPer);
    for (int step = 0; step < x.steps; ++step) {
      const int v = x.begin + step * 32 + lane;
      if (v >= x.end) break;
      const long long e = (long long)v * kPer - x.lead;
      if (e >= 0 && e + kPer <= (long long)vocab) copy_async16(cache + step * 32, x.row + e);
      else cache[step * 32] = x.load(v);
    }
    copy_async_wait();  // a lane reads back what it has copied itself
    x.cache = cache;
  }
  if (threadIdx.x < kSteps) s.table[threadIdx.x] = exp2(double(threadIdx.x) / kSteps);

  // ---- the largest logit
  float top = x.largest();  // passes NaN over
  top = block_max(top, s.reduce_f);
  cluster_wait_started();
  if (int(threadIdx.x) < parts) c.of(threadIdx.x).part_max[c.rank] = top;
  c.group.sync();
  for (int part = 0; part < parts; ++part) top = fmaxf(top, s.part_max[part]);
  if (!(top > -INFINITY)) {
    if (c.rank == 0 && threadIdx.x == 0) draw_nothing(r, tokens, logprobs);
    return;  // the whole cluster; nothing of it is read any more
  }
  RowWeights w = row_weights(p, set, top, s.table);
  // Of a row with +inf only those are kept: for their weights they are the largest finite number, as is the row's
  // largest logit then, and all weights come out alike.
  constexpr float kLargestFinite = 3.4028234663852886e38f;
  if (w.only_largest) w.largest = kLargestFinite;
  auto weight = [&](float l) { return weight_of_steps(w, (double(fminf(l, kLargestFinite)) - w.largest) * w.steps); };

  // ---- the cuts, among the logits that have any weight. First bins: equal steps of the logit below the largest.
  const double inv_steps = set.temperature * kStepLn2;
  const float weighty = logit_from_steps(w, inv_steps, top, kNoWeight);
  RowCut cut{weighty, kNoEnd};
  // (The last bins lie below `weighty`, so no logit with weight falls behind them. Halves: the difference of two floats may
  // be more than a float holds. +inf next to +inf is NaN, which becomes bin 0.)
  const float per_bin = fminf(float(2.0 * kRowBins / ((kWeightBits + 2.5) * kLn2 * set.temperature)), 1e30f);
  auto place = [&](float l) { return (0.5f * top - 0.5f * l) * per_bin; };
  auto bin = [&](float l) { return uint32_t(min(__float2int_rz(place(l)), kRowBins - 1)); };
  // a bin goes from the smallest logit that lies ahead of the next bin up to, and without, its own border
  auto logits_of = [&](uint32_t b) {
    if (w.only_largest) return RowBin{top, __uint_as_float(0x7fc00000u)};
    auto border = [&](uint32_t first) {
      return border_of(top - 2.f * float(first) / per_bin, top, [&](float l) { return place(l) < float(first); });
    };
    return RowBin{border(b + 1), b > 0 ? border(b) : __uint_as_float(0x7fc00000u)};
  };
  if (set.top_k > 0 && set.top_k < (long long)vocab) {
    const unsigned long long k = (unsigned long long)set.top_k;
    auto one = [](float) { return 1ull; };
    auto all = [&](uint32_t, float l) { return l >= weighty; };
    const Crossing at = find_bin(c, x, one, bin, all, [&](unsigned long long total) { return total < k ? total : k; });
    if (at.total > k) cut = find_place(c, x, at.before, k, one, logits_of(at.bin), cut);
    else c.group.sync();  // the others may still read the bins, which the next cut overwrites
  }
  if (set.top_p < 1.0) {
    const RowCut outer = cut;
    const Crossing at = find_bin(
        c, x, weight, bin, [&](uint32_t index, float l) { return inside(outer, l, index); },
        [&](unsigned long long total) { return mass_target(set.top_p, total); });
    cut = find_place(c, x, at.before, mass_target(set.top_p, at.total), weight, logits_of(at.bin), outer);
  }
  const bool few = cut.value > weighty || set.lowest > -INFINITY;
  if (set.lowest > -INFINITY) {
    const float lowest = logit_from_steps(w, inv_steps, top, set.lowest);
    if (lowest > cut.value) cut = RowCut{lowest, kNoEnd};
  }

  // ---- the kept weights, piece by piece in index order. Where a cut leaves few, a warp first moves them together
  // (up to kCompact of them), so that a piece is 32 kept elements, one per lane.
  auto kept = [&](uint32_t index, float l) { return inside(cut, l, index); };
  auto kept_at_step = [&](int step) {
    unsigned long long sum = 0;
    x.at_step(step, [&](uint32_t index, float(&l)[kPer]) {
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        bool is = l[i] >= cut.value;
        if (cut.end != kNoEnd) is = kept(index + i, l[i]);
        const unsigned long long a = weight(is ? l[i] : top);
        sum += is ? a : 0ull;
      }
    });
    return sum;
  };
  constexpr int kCompact = kRowCompact;
  uint32_t* const together = s.together[warp];
  int n_kept = few ? 0 : kCompact + 1;
  __syncthreads();
  for (int i = threadIdx.x; i < kRowWarps * kRowPieces; i += kRowThreads) s.pieces[i] = 0;
  __syncthreads();
  for (int step = 0; step < x.steps && n_kept <= kCompact; ++step) {
    uint32_t hits = 0, first = 0;
    x.at_step(step, [&](uint32_t index, float(&l)[kPer]) {
      first = index;
#pragma unroll
      for (int i = 0; i < kPer; ++i) hits |= l[i] >= cut.value ? 1u << i : 0u;
      if (cut.end != kNoEnd) {
#pragma unroll
        for (int i = 0; i < kPer; ++i)
          if (l[i] == cut.value && index + i >= cut.end) hits &= ~(1u << i);
      }
    });
    if (!__any_sync(0xffffffffu, hits != 0)) continue;
    int inc = __popc(hits);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int other = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += other;
    }
    int at = n_kept + inc - __popc(hits);
    n_kept += __shfl_sync(0xffffffffu, inc, 31);
    if (n_kept > kCompact) break;
    while (hits != 0) {
      together[at++] = first + uint32_t(__ffs(hits) - 1);
      hits &= hits - 1;
    }
  }
  const bool compact = n_kept <= kCompact;
  __syncwarp();
  auto weight_together = [&](int i, float* l) {
    const bool is = i < n_kept;
    *l = is ? logit_to_float(x.flat[together[i]]) : top;
    const unsigned long long a = weight(*l);
    return is ? a : 0ull;
  };
  float logit;
  const int pieces = compact ? (n_kept + 31) / 32 : (x.steps + x.per_piece - 1) / x.per_piece;
  for (int piece = 0; piece < pieces; ++piece) {
    unsigned long long mine = 0;
    if (compact)
      mine = weight_together(piece * 32 + lane, &logit);
    else
      for (int step = piece * x.per_piece; step < min((piece + 1) * x.per_piece, x.steps); ++step)
        mine += kept_at_step(step);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
    if (lane == 0) s.pieces[warp * kRowPieces + piece] = mine;
  }
  __syncthreads();
  constexpr int kEach = kRowWarps * kRowPieces / kRowThreads;
  unsigned long long mine = 0, block_total;
#pragma unroll
  for (int i = 0; i < kEach; ++i) mine += s.pieces[kEach * threadIdx.x + i];
  unsigned long long before = block_prefix(mine, s.reduce, &block_total);
  if (int(threadIdx.x) < parts) c.of(threadIdx.x).part_sum[c.rank] = block_total;
  c.group.sync();
  // ---- the token: no block touches another's memory from here on
  unsigned long long total = 0, block_before = 0;
  for (int part = 0; part < parts; ++part) {
    if (part < c.rank) block_before += s.part_sum[part];
    total += s.part_sum[part];
  }
  const unsigned long long goal = draw_target(set.u, total);
  if (goal < block_before || goal >= block_before + block_total) return;
  before += block_before;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const unsigned long long a = s.pieces[kEach * threadIdx.x + i];
    if (a != 0 && before <= goal && goal < before + a) {
      s.piece = kEach * threadIdx.x + i;
      s.piece_before = before;
    }
    before += a;
  }
  __syncthreads();
  if (warp != int(s.piece) / kRowPieces) return;
  const int piece = int(s.piece) % kRowPieces;
  before = s.piece_before;
  auto drawn = [&](uint32_t index, float l, unsigned long long a) {
    tokens[r] = index;
    logprobs[r] = log_share(p, set, w, l, a, total);
  };
  auto lanes_before = [&](unsigned long long here, unsigned long long* all) {
    unsigned long long inc = here;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned long long other = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += other;
    }
    *all = __shfl_sync(0xffffffffu, inc, 31);
    return inc - here;
  };
  unsigned long long all;
  if (compact) {
    const unsigned long long a = weight_together(piece * 32 + lane, &logit);
    const unsigned long long at = before + lanes_before(a, &all);
    if (a != 0 && at <= goal && goal < at + a) drawn(together[piece * 32 + lane], logit, a);
    return;
  }
  for (int step = piece * x.per_piece; step < min((piece + 1) * x.per_piece, x.steps); ++step) {
    const unsigned long long here = kept_at_step(step);
    unsigned long long at = before + lanes_before(here, &all);
    if (at <= goal && goal < at + here)
      x.some_at_step(step, [&](float l) { return l >= cut.value; }, [&](uint32_t index, float l) {
        if (!kept(index, l)) return;
        const unsigned long long a = weight(l);
        if (at <= goal && goal < at + a) drawn(index, l, a);
        at += a;
      });
    before += all;
  }
}

// It may run beside sample_list_kernel: the two read the same inputs and write different rows (256 x 131072 bf16, a
// quarter of the rows here: 68.7 us against 72.5 one after the other; their registers leave little room for both). Its
// end is the end of both, since its first block waits for the other kernel (and for nothing where that was not launched).
template <typename T>
__global__ void __launch_bounds__(kRowThreads, 2)
sample_row_kernel(const T* __restrict__ logits, long long ld, uint32_t vocab, int parts, int cache_vectors,
                  const SampleParams p, long long* __restrict__ tokens, float* __restrict__ logprobs) {
  sample_row(logits, ld, vocab, parts, cache_vectors, p, tokens, logprobs);
  if (blockIdx.x == 0) asm volatile("griddepcontrol.wait;" ::: "memory");
}

}  // namespace lce
