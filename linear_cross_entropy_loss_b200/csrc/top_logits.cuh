// top_logits: the k largest logits of each row with their indices, and the row's log-sum-exp.
#pragma once

#include "row_select.cuh"

namespace lce {

constexpr int kTopMax = 1024;
constexpr int kTopThreads = 512;

// One block per row. k <= min(vocab, kTopMax); `padded`: k rounded up to a power of two.
template <typename T>
__global__ void __launch_bounds__(kTopThreads)
top_logits_kernel(const T* __restrict__ logits, long long ld, uint32_t vocab, int k, int padded, float inv_temperature,
                  T* __restrict__ values, long long* __restrict__ indices, float* __restrict__ lse) {
  __shared__ SelectScratch s;
  __shared__ float scratch[32];
  __shared__ unsigned long long list[kTopMax];
  __shared__ int listed;
  const long long r = blockIdx.x;
  const T* row = logits + r * ld;
  const RowCut cut = find_cut(row, vocab, (unsigned long long)k, s, [](float, uint32_t, uint32_t) { return 1ull; });
  if (threadIdx.x == 0) listed = 0;
  for (int i = threadIdx.x; i < padded; i += blockDim.x) list[i] = 0;
  __syncthreads();
  float m = -INFINITY;
  bool nan = false;
  for (uint32_t j = threadIdx.x; j < vocab; j += blockDim.x) {
    const float l = logit_to_float(row[j]);
    const uint32_t key = order_key(l);
    m = fmaxf(m, l);
    nan |= l != l;
    if (inside(cut, key, j)) list[atomicAdd(&listed, 1)] = order_pair(key, j);
  }
  m = block_max(m, scratch);
  nan = block_max(nan ? 1.f : 0.f, scratch) > 0.f;
  float sum = 0.f;
  if (m > -INFINITY && m < INFINITY)
    for (uint32_t j = threadIdx.x; j < vocab; j += blockDim.x)
      sum += __expf((logit_to_float(row[j]) - m) * inv_temperature);
  sum = block_sum(sum, scratch);
  if (threadIdx.x == 0)
    lse[r] = nan ? __uint_as_float(0x7fc00000u) : ((m > -INFINITY && m < INFINITY) ? m * inv_temperature + logf(sum) : m);
  block_sort_descending(list, padded);
  for (int i = threadIdx.x; i < k; i += blockDim.x) {
    const uint32_t j = pair_index(list[i]);
    values[r * k + i] = row[j];
    indices[r * k + i] = j;
  }
}

}  // namespace lce
