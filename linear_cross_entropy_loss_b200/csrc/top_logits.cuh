// top_logits: the k largest logits of each row with their indices, and the row's log-sum-exp. The row is read once
// (row_top.cuh); `parts` blocks of a cluster share a row when there are too few rows to fill the GPU.
#pragma once

#include "row_top.cuh"

namespace lce {

constexpr float kLog2e = 1.4426950408889634f;

template <typename T>
__global__ void __launch_bounds__(kTopThreads, 3)
top_logits_kernel(const T* __restrict__ logits, long long ld, uint32_t vocab, int k, int parts, float inv_temperature,
                  T* __restrict__ values, long long* __restrict__ indices, float* __restrict__ lse) {
  extern __shared__ __align__(16) unsigned char dynamic[];
  TopShared& s = *reinterpret_cast<TopShared*>(dynamic);
  const long long r = blockIdx.x / parts;
  const int part = int(blockIdx.x % parts);
  const RowGroups<T> row(logits + r * ld, vocab);
  const int v0 = int((long long)row.groups * part / parts), v1 = int((long long)row.groups * (part + 1) / parts);
  const float log2_scale = inv_temperature * kLog2e;
  float ref, sum;
  stream_top<T, true, Nan::kFirst>(s, row, v0, v1, parts, k, log2_scale, ref, sum);
  const float m = block_max(ref, s.scratch);
  sum = block_sum(ref > -INFINITY ? sum * fast_exp2(ref - m) : 0.f, s.scratch);
  if (threadIdx.x == 0) {
    TopShared* first = parts > 1 ? cooperative_groups::this_cluster().map_shared_rank(&s, 0) : &s;
    first->part_ref[part] = m;
    first->part_sum[part] = sum;
  }
  const TopGroups g = merge_lists(s, k, parts);
  if (part != 0) return;
  const int n = rank_elements<Nan::kFirst>(s, row, g, k);
  for (int i = threadIdx.x; i < n; i += kTopThreads) {
    const unsigned long long e = g.free_list[i];
    values[r * k + i] = T(key_to_float(pair_key(e)));
    indices[r * k + i] = pair_index(e);
  }
  if (threadIdx.x == 0) {
    float top = s.part_ref[0], total = 0.f;
    for (int i = 1; i < parts; ++i) top = fmaxf(top, s.part_ref[i]);
    for (int i = 0; i < parts; ++i)
      if (s.part_ref[i] > -INFINITY) total += s.part_sum[i] * fast_exp2(s.part_ref[i] - top);
    // The sum is over 2^(l * log2_scale), whose exponents are right to the rounding of log2_scale; at the largest
    // logit, which carries the sum, that rounding is put back.
    const uint32_t first = pair_key(g.free_list[0]);
    const double largest = double(key_to_float(first));
    const double put_back = largest * (double(inv_temperature) - double(log2_scale) * kLn2);
    float v = float((double(top) + double(log2f(total))) * kLn2 + put_back);
    if (first >= kKeyPosInf || first == kKeyNegInf) v = key_to_float(first);  // +inf, NaN; nothing but -inf
    // From 2^30 on a float's steps are 64 and more, and the others (at most 2^30, log 21) do not move it. The sum is of no
    // use there: its terms are off by the rounding of the reference, which is an exponent of 2^6 and more.
    else if (fabs(largest * double(inv_temperature)) >= 1073741824.0) v = float(largest * double(inv_temperature));
    lse[r] = v;
  }
}

}  // namespace lce
