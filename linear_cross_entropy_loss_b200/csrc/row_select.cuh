// Exact selection in one row of logits: the place in the order (logit descending, index ascending) at which a count or
// a mass is reached. One block per row; radix search over the 32-bit keys, eight bits at a time from the top, with one
// sweep over the row per level, then one sweep that finds the index among equal keys.
#pragma once

#include "vocab_row.cuh"

namespace lce {

// Everything up to and including (key, index) in the order is inside: key > cut.key, or key == cut.key and
// index <= cut.index.
struct RowCut {
  uint32_t key;
  uint32_t index;
};
constexpr uint32_t kNoIndexLimit = 0xffffffffu;
__device__ __forceinline__ bool inside(const RowCut& c, uint32_t key, uint32_t index) {
  return key > c.key || (key == c.key && index <= c.index);
}

struct SelectScratch {
  unsigned long long bins[256];
  unsigned long long reduce[32];
  unsigned long long found[2];  // digit, amount before it
};

// amount(key, index): what one element contributes (1 to count, its weight for a mass). Finds the smallest prefix of
// the order whose amounts add up to at least `target` (1 <= target <= the sum over the row).
template <typename T, typename Amount>
__device__ RowCut find_cut(const T* row, uint32_t vocab, unsigned long long target, SelectScratch& s, Amount amount) {
  uint32_t prefix = 0, mask = 0;
  unsigned long long before = 0;
  for (int shift = 24; shift >= 0; shift -= 8) {
    __syncthreads();
    for (int b = threadIdx.x; b < 256; b += blockDim.x) s.bins[b] = 0;
    __syncthreads();
    for (uint32_t j = threadIdx.x; j < vocab; j += blockDim.x) {
      const float l = logit_to_float(row[j]);
      const uint32_t key = order_key(l);
      if ((key & mask) == prefix) {
        const unsigned long long a = amount(l, key, j);
        if (a != 0) atomicAdd(&s.bins[(key >> shift) & 255u], a);
      }
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      int d = 255;
      while (d > 0 && before + s.bins[d] < target) before += s.bins[d--];
      s.found[0] = (unsigned long long)d;
      s.found[1] = before;
    }
    __syncthreads();
    prefix |= uint32_t(s.found[0]) << shift;
    mask |= 255u << shift;
    before = s.found[1];
  }
  // among the elements with this key, in index order: the one at which the target is reached
  unsigned long long seen = before;
  uint32_t index = kNoIndexLimit;
  for (uint32_t j0 = 0; j0 < vocab; j0 += blockDim.x) {
    const uint32_t j = j0 + threadIdx.x;
    unsigned long long a = 0;
    if (j < vocab) {
      const float l = logit_to_float(row[j]);
      const uint32_t key = order_key(l);
      if (key == prefix) a = amount(l, key, j);
    }
    unsigned long long total;
    const unsigned long long at = seen + block_prefix(a, s.reduce, &total);
    if (a != 0 && at < target && at + a >= target) s.found[0] = j;
    if (seen + total >= target) {
      __syncthreads();
      index = uint32_t(s.found[0]);
      break;
    }
    seen += total;
  }
  return RowCut{prefix, index};
}

}  // namespace lce
