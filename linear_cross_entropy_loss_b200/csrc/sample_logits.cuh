// sample_logits: one token of each row, drawn with a given random number after temperature, top-k, top-p and min-p.
//   w_j = exp((l_j - max) / T); order: logit descending, index ascending
//   kept: the first top_k of the order; of those the shortest prefix that holds top_p of their mass; of those w >= min_p
//   token = the first j in index order at which the kept weights, added up, exceed u * (their sum)
#pragma once

#include "row_select.cuh"

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
};

constexpr int kSampleThreads = 512;

template <typename T>
__global__ void __launch_bounds__(kSampleThreads)
sample_logits_kernel(const T* __restrict__ logits, long long ld, uint32_t vocab, int weight_bits, const SampleParams p,
                     long long* __restrict__ tokens, float* __restrict__ logprobs) {
  __shared__ SelectScratch s;
  __shared__ float scratch[32];
  __shared__ double table[32];
  const long long r = blockIdx.x;
  const T* row = logits + r * ld;
  if (threadIdx.x < 32) table[threadIdx.x] = exp2(threadIdx.x / 32.0);
  float m = -INFINITY;
  unsigned long long allowed = 0;
  for (uint32_t j = threadIdx.x; j < vocab; j += blockDim.x) {
    const float l = logit_to_float(row[j]);
    m = fmaxf(m, l);  // a NaN is passed over
    allowed += l > -INFINITY;
  }
  m = block_max(m, scratch);
  allowed = block_sum(allowed, s.reduce);
  if (!(m > -INFINITY)) {  // nothing may be drawn
    if (threadIdx.x == 0) {
      tokens[r] = -1;
      logprobs[r] = -INFINITY;
    }
    return;
  }
  double T_row = p.temperature ? double(p.temperature[r]) : p.temperature_all;
  long long k = p.top_k ? p.top_k[r] : p.top_k_all;
  const double top_p = p.top_p ? double(p.top_p[r]) : p.top_p_all;
  const double min_p = p.min_p ? double(p.min_p[r]) : p.min_p_all;
  double u = p.u_is_double ? reinterpret_cast<const double*>(p.u)[r] : double(reinterpret_cast<const float*>(p.u)[r]);
  u = u > 0.0 ? u : 0.0;
  if (!(T_row > 0.0)) {  // greedy
    T_row = 1.0;
    k = 1;
  }
  RowWeights w;
  w.largest = m;
  w.only_largest = m == INFINITY;
  w.steps = fmin(46.166241308446828 / T_row, 1e300);  // 32 log2(e) / T
  w.to_int = exp2(double(52 - weight_bits));
  w.table = table;

  auto weight = [&](float l) { return l > -INFINITY ? row_weight(w, l) : 0ull; };
  RowCut cut = {0u, kNoIndexLimit};
  if (k > 0 && (unsigned long long)k < allowed)
    cut = find_cut(row, vocab, (unsigned long long)k, s,
                   [](float l, uint32_t, uint32_t) { return l > -INFINITY ? 1ull : 0ull; });
  if (top_p < 1.0) {
    unsigned long long mass = 0;
    for (uint32_t j = threadIdx.x; j < vocab; j += blockDim.x) {
      const float l = logit_to_float(row[j]);
      if (inside(cut, order_key(l), j)) mass += weight(l);
    }
    mass = block_sum(mass, s.reduce);
    const double goal = ceil(fmax(top_p, 0.0) * double(mass));
    unsigned long long target = goal < 1.0 ? 1ull : (unsigned long long)goal;
    if (target > mass) target = mass;
    const RowCut outer = cut;
    cut = find_cut(row, vocab, target, s,
                   [&](float l, uint32_t key, uint32_t j) { return inside(outer, key, j) ? weight(l) : 0ull; });
  }
  // (l - max) / T >= log(min_p), in the steps of the weights
  const double lowest = min_p > 0.0 ? 32.0 * log2(fmin(min_p, 1.0)) : -INFINITY;
  auto kept = [&](float l, uint32_t j) {
    if (!(l > -INFINITY) || !inside(cut, order_key(l), j)) return 0ull;
    if (!w.only_largest && !(weight_steps(w, l) >= lowest)) return 0ull;
    return weight(l);
  };
  unsigned long long total = 0;
  for (uint32_t j = threadIdx.x; j < vocab; j += blockDim.x) total += kept(logit_to_float(row[j]), j);
  total = block_sum(total, s.reduce);
  unsigned long long goal = (unsigned long long)(fmin(u, 1.0) * double(total));
  if (goal >= total) goal = total - 1;
  unsigned long long seen = 0;
  for (uint32_t j0 = 0; j0 < vocab; j0 += blockDim.x) {
    const uint32_t j = j0 + threadIdx.x;
    float l = -INFINITY;
    unsigned long long a = 0;
    if (j < vocab) {
      l = logit_to_float(row[j]);
      a = kept(l, j);
    }
    unsigned long long sum;
    const unsigned long long at = seen + block_prefix(a, s.reduce, &sum);
    if (a != 0 && at <= goal && goal < at + a) {
      tokens[r] = j;
      const double log_share = w.only_largest ? log(double(a) / double(total))
                                              : weight_steps(w, l) * kStepLn2 - log(ldexp(double(total), -weight_bits));
      logprobs[r] = float(log_share);
    }
    seen += sum;
    if (seen > goal) break;
  }
}

}  // namespace lce
