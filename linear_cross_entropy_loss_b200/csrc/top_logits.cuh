// top_logits: the k largest logits of each row with their indices, and the row's log-sum-exp. The row is read once
// (row_top.cuh); `parts` blocks of a cluster share a row when there are too few rows to fill the GPU.
#pragma once

#include "row_top.cuh"

namespace lce {

template <typename T>
__global__ void __launch_bounds__(kTopThreads, 4)
top_logits_kernel(const T* __restrict__ logits, long long ld, uint32_t vocab, int k, int parts, float inv_temperature,
                  T* __restrict__ values, long long* __restrict__ indices, float* __restrict__ lse) {
  __shared__ TopShared s;
  const long long r = blockIdx.x / parts;
  const int part = int(blockIdx.x % parts);
  const RowGroups<T> row(logits + r * ld, vocab);
  const int share = (row.groups + parts - 1) / parts;
  const int v0 = min(part * share, row.groups), v1 = min(v0 + share, row.groups);
  const float log2_scale = inv_temperature * 1.4426950408889634f;
  float ref, sum;
  stream_top<T, true, Nan::kFirst>(s, row, v0, v1, k, log2_scale, ref, sum);
  const float m = block_max(ref, s.scratch);
  sum = block_sum(ref > -INFINITY ? sum * fast_exp2(ref - m) : 0.f, s.scratch);
  if (threadIdx.x == 0) {
    s.part_ref = m;
    s.part_sum = sum;
  }
  merge_lists(s, k, parts);
  if (part != 0) return;
  rank_elements<Nan::kFirst>(s, row, k);
  for (int i = threadIdx.x; i < k; i += kTopThreads) {
    const unsigned long long e = s.elements[i];
    values[r * k + i] = T(key_to_float(pair_key(e)));
    indices[r * k + i] = pair_index(e);
  }
  if (threadIdx.x == 0) {
    // The sum is over 2^(l * log2_scale), whose exponents are right to the rounding of log2_scale; at the largest
    // logit, which carries the sum, that rounding is put back.
    const uint32_t first = pair_key(s.elements[0]);
    const double largest = double(key_to_float(first));
    const double put_back = largest * (double(inv_temperature) - double(log2_scale) * 0.69314718055994531);
    float v = float((double(s.part_ref) + double(log2f(s.part_sum))) * 0.69314718055994531 + put_back);
    if (first >= kKeyPosInf || first == kKeyNegInf) v = key_to_float(first);  // +inf, NaN; nothing but -inf
    lse[r] = v;
  }
}

}  // namespace lce
