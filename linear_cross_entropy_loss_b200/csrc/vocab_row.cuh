// Pieces shared by the kernels that work on one row of logits (top_logits.cuh, sample_logits.cuh): the order of the
// logits, the exact weights of the sampler, block-wide reductions and sorting.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <cstdint>

namespace lce {

__device__ __forceinline__ float logit_to_float(float v) { return v; }
__device__ __forceinline__ float logit_to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float logit_to_float(__nv_bfloat16 v) { return __bfloat162float(v); }

// Logits as unsigned keys in the same order: -inf = kKeyNegInf < finite < +inf < NaN (all NaN alike); -0 equals +0.
constexpr uint32_t kKeyNegInf = 0x007fffffu;
constexpr uint32_t kKeyPosInf = 0xff800000u;
constexpr uint32_t kKeyNaN = 0xffffffffu;
__device__ __forceinline__ uint32_t order_key(float f) {
  const uint32_t b = __float_as_uint(f + 0.0f);
  const uint32_t key = b ^ (uint32_t(int32_t(b) >> 31) | 0x80000000u);
  return f != f ? kKeyNaN : key;
}
__device__ __forceinline__ float key_to_float(uint32_t key) {
  if (key == kKeyNaN) return __uint_as_float(0x7fc00000u);
  return __uint_as_float((key & 0x80000000u) ? (key ^ 0x80000000u) : ~key);
}

// A logit and its place as one number: larger = larger logit, then lower index.
__device__ __forceinline__ unsigned long long order_pair(uint32_t key, uint32_t index) {
  return ((unsigned long long)key << 32) | (0xffffffffu - index);
}
__device__ __forceinline__ uint32_t pair_key(unsigned long long pair) { return uint32_t(pair >> 32); }
__device__ __forceinline__ uint32_t pair_index(unsigned long long pair) { return 0xffffffffu - uint32_t(pair); }

// ---------------------------------------------------------------------------------------------
// block-wide steps; every thread of the block takes part, blockDim.x is a multiple of 32
// ---------------------------------------------------------------------------------------------
template <typename T, typename Op>
__device__ __forceinline__ T block_reduce(T v, T* scratch /*[32]*/, Op op) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  __syncthreads();  // scratch may still be read from an earlier call
  if (lane == 0) scratch[warp] = v;
  __syncthreads();
  v = scratch[lane < warps ? lane : 0];
  T r = v;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const T other = __shfl_xor_sync(0xffffffffu, r, o);
    r = op(r, other);
  }
  return r;  // warps beyond the block repeat scratch[0]: fine for max / min; block_sum masks them itself
}
template <typename T>
__device__ __forceinline__ T block_max(T v, T* scratch) {
  return block_reduce(v, scratch, [](T a, T b) { return a > b ? a : b; });
}
template <typename T>
__device__ __forceinline__ T block_sum(T v, T* scratch /*[32]*/) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  __syncthreads();
  if (lane == 0) scratch[warp] = v;
  __syncthreads();
  T r = lane < warps ? scratch[lane] : T(0);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) r += __shfl_xor_sync(0xffffffffu, r, o);
  return r;
}
// Sum of v over the threads before this one; the sum over all of them in *total.
template <typename T>
__device__ __forceinline__ T block_prefix(T v, T* scratch /*[32]*/, T* total) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  T inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const T other = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += other;
  }
  __syncthreads();
  if (lane == 31) scratch[warp] = inc;
  __syncthreads();
  T w = lane < warps ? scratch[lane] : T(0);
  T winc = w;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const T other = __shfl_up_sync(0xffffffffu, winc, o);
    if (lane >= o) winc += other;
  }
  *total = __shfl_sync(0xffffffffu, winc, 31);
  const T before = __shfl_sync(0xffffffffu, winc - w, warp);
  return before + inc - v;
}

// Sorts kThreads * kEach numbers in shared memory, largest first (a bitonic network). Thread t holds the places t *
// kEach ..: strides below kEach stay in its registers, strides below 32 * kEach go through shuffles, and only the few
// longer ones through shared memory. (All 55 steps of 1024 numbers through shared memory took 21,000 cycles.)
template <int kThreads, int kEach>
__device__ __forceinline__ void block_sort_each(unsigned long long* a) {
  unsigned long long v[kEach];
  const int first = int(threadIdx.x) * kEach;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kEach; ++i) v[i] = a[first + i];
  for (int size = 2; size <= kThreads * kEach; size <<= 1) {
    for (int stride = size >> 1; stride > 0; stride >>= 1) {
      if (stride >= 32 * kEach) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kEach; ++i) a[first + i] = v[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
          const int at = first + i;
          const unsigned long long other = a[at ^ stride];
          const bool larger = ((at & size) == 0) == ((at & stride) == 0);  // this place gets the larger of the two
          v[i] = (other > v[i]) == larger ? other : v[i];
        }
      } else if (stride >= kEach) {
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
          const int at = first + i;
          const unsigned long long other = __shfl_xor_sync(0xffffffffu, v[i], stride / kEach);
          const bool larger = ((at & size) == 0) == ((at & stride) == 0);
          v[i] = (other > v[i]) == larger ? other : v[i];
        }
      } else {
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
#pragma unroll
          for (int j = 1; j < kEach; j <<= 1) {
            if (j == stride && (i & j) == 0) {
              const unsigned long long x = v[i], y = v[i | j];
              const bool down = ((first + i) & size) == 0;
              v[i] = (x < y) == down ? y : x;
              v[i | j] = (x < y) == down ? x : y;
            }
          }
        }
      }
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kEach; ++i) a[first + i] = v[i];
  __syncthreads();
}
// Sorts the first n numbers of an array that has room for kThreads times a power of two of them (up to 2048 in all),
// largest first.
template <int kThreads>
__device__ __noinline__ void block_sort_descending(unsigned long long* a, int n) {
  __syncthreads();
  int each = 1;
  while (each * kThreads < n) each <<= 1;
  for (int i = n + int(threadIdx.x); i < each * kThreads; i += kThreads) a[i] = 0;
  switch (each) {
    case 1: block_sort_each<kThreads, 1>(a); break;
    case 2: block_sort_each<kThreads, 2>(a); break;
    case 4: block_sort_each<kThreads, 4>(a); break;
    default: block_sort_each<kThreads, 2048 / kThreads>(a);
  }
}

// ---------------------------------------------------------------------------------------------
// weights of the sampler
// ---------------------------------------------------------------------------------------------
// w = exp((l - max) / T) as an integer: w * 2^bits rounded to the nearest. Integers add up to the same sum in any
// order, so the sums of a row do not depend on how it is split over threads and blocks, and a token's border is where
// 64-bit arithmetic puts it: the rounding of one weight is 2^-(bits + 1) of the largest one (bits = 44 for up to
// 2^18 columns), the exponential is off by at most 2.3e-12 of itself. A sum of 32-bit floats would be off by 1e-7 of the
// total, which is as wide as the share of a token in the tail of a vocabulary.
//   exp(d / T) = 2^(n / 128) (1 + x + x^2 / 2 + x^3 / 6),  n = round(128 d log2(e) / T),  |x| <= ln(2) / 256
struct RowWeights {
  double largest;        // the row's largest logit
  double steps;          // kSteps log2(e) / T: logit difference -> n
  double to_int;         // 2^(52 - bits): adding it leaves w * 2^bits in the low bits of the sum
  uint32_t table;        // shared-memory address of 2^(j / kSteps), j = 0 .. kSteps - 1
  bool only_largest;     // the largest logit is +inf: it alone has weight
};
constexpr int kWeightBits = 44;
constexpr int kSteps = 128;  // a power of two
constexpr double kLn2 = 0.69314718055994531, kStepLn2 = kLn2 / kSteps;

__device__ __forceinline__ double weight_steps(const RowWeights& w, float logit) {
  return (double(logit) - w.largest) * w.steps;
}
// Steps below which a weight rounds to nothing.
constexpr double kNoWeight = -double(kSteps) * (kWeightBits + 2);
// The weight of `steps` in [kNoWeight, 0].
__device__ __forceinline__ unsigned long long weight_of_steps(const RowWeights& w, double steps) {
  const double shifted = steps + 6755399441055744.0;  // 1.5 * 2^52: the integer part ends up in the low word
  const int n = __double2loint(shifted);
  const double y = steps - (shifted - 6755399441055744.0);  // |y| <= 1/2; the series is in y ln(2) / kSteps
  constexpr double c = kStepLn2;
  double p = fma(y, c * c * c / 6.0, c * c / 2.0);
  p = fma(y, p, c);
  p = fma(y, p, 1.0);
  double step;
  asm("ld.shared.f64 %0, [%1];" : "=d"(step) : "r"(w.table + (uint32_t(n) & (kSteps - 1)) * 8u));
  p *= step;
  constexpr int kShift = 20 - 7;  // n / kSteps into the exponent
  static_assert(kSteps == 1 << 7, "kShift goes with it");
  p = __hiloint2double(__double2hiint(p) + ((n & ~(kSteps - 1)) << kShift), __double2loint(p));
  return (unsigned long long)(__double_as_longlong(p + w.to_int) - __double_as_longlong(w.to_int));
}
__device__ __forceinline__ unsigned long long row_weight(const RowWeights& w, float logit) {
  if (w.only_largest) return double(logit) == w.largest ? 1ull << 32 : 0ull;
  const double steps = weight_steps(w, logit);
  return steps >= kNoWeight ? weight_of_steps(w, steps) : 0ull;  // also 0 for -inf and NaN
}

}  // namespace lce
