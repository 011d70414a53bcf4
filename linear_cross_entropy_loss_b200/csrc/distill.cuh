// Distillation from a teacher's top logits on the contraction engine of the cross-entropy loss.
//
//   q_k  = softmax of the listed teacher logits / T (or exp(t_k / T - lse) when the teacher's log-sum-exp is given)
//   loss = T^2 / n sum_i sum_k q_ik (log q_ik - z_ik / T + logsumexp_j(z_ij / T))
//   dZ_i = T / n (Q_i softmax(z_i / T) - sum_k q_ik [idx_ik = j]),   Q_i = sum_k q_ik
//
// The same shape as cross-entropy, with a row factor Q_i and a short sorted list in the place of the one label:
//   teacher_prepare_kernel  q, Q, sum q log q; each row's list sorted by index, equal indices merged, with the place in the list
//                           at which every 256-column tile of the vocabulary begins
//   forward contraction     its epilogue also copies the logits at the listed columns (gather_listed in gemm_sm100.cuh)
//   row statistics          sum_k q z - sum_k q log q in the place of the label's logit
//   distill_finish_kernel / distill_dz_kernel   dZ from the slab, with the listed entries written from their fp32 logits
// then the dx and dW contractions as they are.
#pragma once

#include "aux_kernels.cuh"

namespace lce {

constexpr int kTeacherMax = 1024;         // entries per row
constexpr int kPrepareThreads = 256;
constexpr int kPrepareEntries = 2048;     // entries a block holds: rows of a block x their length rounded up to 2^n

struct TeacherInput {
  const void* logits;
  const void* indices;
  const float* lse;  // may be null
  long long logits_ld;
  long long indices_ld;
  int k;
  int logits_dtype;   // LCE_DTYPE_*
  int indices_64;     // 1: int64, 0: int32
  float inv_temperature;
};

__device__ __forceinline__ float teacher_logit(const TeacherInput& t, long long row, int k) {
  const long long at = row * t.logits_ld + k;
  if (t.logits_dtype == 0) return __half2float(reinterpret_cast<const __half*>(t.logits)[at]);
  if (t.logits_dtype == 1) return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(t.logits)[at]);
  return reinterpret_cast<const float*>(t.logits)[at];
}
// The column of an entry; 0xffffffff for an entry that is not there (index outside the vocabulary).
__device__ __forceinline__ uint32_t teacher_column(const TeacherInput& t, long long row, int k, long long vocab) {
  const long long at = row * t.indices_ld + k;
  const long long i = t.indices_64 ? reinterpret_cast<const long long*>(t.indices)[at]
                                   : (long long)reinterpret_cast<const int*>(t.indices)[at];
  return i >= 0 && i < vocab ? uint32_t(i) : 0xffffffffu;
}

// Row r of the launch is row row0 + r of the problem. kLists: false writes labels / mass / plogp only (every row of the
// problem, so that the valid rows can be counted before the first chunk), true the lists of one chunk too.
//   labels[r] = -1 where the row counts (Q != 0), else ignored
// One block holds `rows_per_block` rows of `padded` (a power of two) entries each.
template <bool kLists>
__global__ void __launch_bounds__(kPrepareThreads)
teacher_prepare_kernel(const TeacherInput t, long long row0, int rows, long long vocab, int rows_per_block, int padded,
                       long long ignored, long long* __restrict__ labels, float* __restrict__ mass,
                       float* __restrict__ plogp, int* __restrict__ list_idx, float* __restrict__ list_q,
                       unsigned short* __restrict__ start, long long start_ld, int n_tiles) {
  __shared__ unsigned long long list[kPrepareEntries];  // column << 32 | bits of q
  __shared__ int lengths[32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int first = blockIdx.x * rows_per_block;
  for (int b = warp; b < rows_per_block; b += kPrepareThreads / 32) {
    const int r = first + b;
    unsigned long long* mine = list + b * padded;
    const bool exists = r < rows;
    float top = -INFINITY;
    bool bad = false;  // NaN or +inf among the entries that are there
    for (int k = lane; k < padded; k += 32) {
      uint32_t col = 0xffffffffu;
      float l = -INFINITY;
      if (exists && k < t.k) {
        col = teacher_column(t, row0 + r, k, vocab);
        if (col != 0xffffffffu) l = teacher_logit(t, row0 + r, k) * t.inv_temperature;
        if (!(l > -INFINITY) && l == l) col = 0xffffffffu;  // -inf: no weight
      }
      bad |= l != l || l == INFINITY;
      top = fmaxf(top, l);
      mine[k] = ((unsigned long long)col << 32) | __float_as_uint(l);
    }
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    bad = __any_sync(0xffffffffu, bad);
    float base = top;  // q = exp(l - base) / total
    float total = 1.f;
    __syncwarp();
    if (t.lse != nullptr) {
      base = exists ? t.lse[row0 + r] : 0.f;
    } else {
      float s = 0.f;
      for (int k = lane; k < padded; k += 32)
        if (uint32_t(mine[k] >> 32) != 0xffffffffu) s += expf(__uint_as_float(uint32_t(mine[k])) - base);
      for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      total = s;
    }
    const float log_total = logf(total);
    float sum = 0.f, ent = 0.f;
    for (int k = lane; k < padded; k += 32) {
      uint32_t col = uint32_t(mine[k] >> 32);
      float q = 0.f;
      if (col != 0xffffffffu) {
        const float log_q = __uint_as_float(uint32_t(mine[k])) - base - log_total;
        q = bad ? __uint_as_float(0x7fc00000u) : expf(log_q);
        if (q == 0.f) col = 0xffffffffu;
        else ent += q * log_q;
        sum += q;
      }
      mine[k] = ((unsigned long long)col << 32) | __float_as_uint(q);
    }
    for (int o = 16; o > 0; o >>= 1) {
      sum += __shfl_xor_sync(0xffffffffu, sum, o);
      ent += __shfl_xor_sync(0xffffffffu, ent, o);
    }
    if (lane == 0 && exists) {
      labels[r] = sum == 0.f ? ignored : -1;  // a NaN counts: it has to reach the loss
      mass[r] = sum;
      plogp[r] = ent;
    }
  }
  if (!kLists) return;

  // every row by column, ascending (the columns that are not there come last)
  for (int size = 2; size <= padded; size <<= 1) {
    for (int stride = size >> 1; stride > 0; stride >>= 1) {
      __syncthreads();
      for (int i = threadIdx.x; i < rows_per_block * padded / 2; i += kPrepareThreads) {
        const int lo = ((i & ~(stride - 1)) << 1) | (i & (stride - 1));
        const int hi = lo | stride;
        const unsigned long long x = list[lo], y = list[hi];
        const bool ascending = (lo & (padded - 1) & size) == 0 || size == padded;
        if ((x > y) == ascending) {
          list[lo] = y;
          list[hi] = x;
        }
      }
    }
  }
  __syncthreads();
  // equal columns become one entry with the sum of their q (in ascending order of q)
  for (int b = warp; b < rows_per_block; b += kPrepareThreads / 32) {
    unsigned long long* mine = list + b * padded;
    int length = 0;
    for (int k0 = 0; k0 < padded; k0 += 32) {
      const int k = k0 + lane;
      const uint32_t col = k < padded ? uint32_t(mine[k] >> 32) : 0xffffffffu;
      const uint32_t before = k > 0 && k < padded ? uint32_t(mine[k - 1] >> 32) : 0xffffffffu;
      const bool head = col != 0xffffffffu && (k == 0 || col != before);
      float q = 0.f;
      if (head)
        for (int m = k; m < padded && uint32_t(mine[m] >> 32) == col; ++m) q += __uint_as_float(uint32_t(mine[m]));
      const uint32_t heads = __ballot_sync(0xffffffffu, head);
      const int at = length + __popc(heads & ((1u << lane) - 1u));
      if (head && first + b < rows) {
        list_idx[(long long)(first + b) * t.k + at] = int(col);
        list_q[(long long)(first + b) * t.k + at] = q;
      }
      length += __popc(heads);
    }
    if (lane == 0) lengths[b] = length;
  }
  __syncthreads();
  // start[tile][r]: entries of row r with a column before tile * 256
  for (int i = threadIdx.x; i < (n_tiles + 1) * rows_per_block; i += kPrepareThreads) {
    const int tile = i / rows_per_block, b = i - tile * rows_per_block, r = first + b;
    if (r >= rows) continue;
    const int* idx = list_idx + (long long)r * t.k;
    int lo = 0, hi = lengths[b];
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (idx[mid] < tile * 256) lo = mid + 1;
      else hi = mid;
    }
    start[(long long)tile * start_ld + r] = (unsigned short)lo;
  }
}

// dZ / T * n of one listed entry.
__device__ __forceinline__ float listed_dz(float z, float lse, float mass, float q) { return expf(z - lse) * mass - q; }

// Row-reference mode (see row_finish_kernel): one block per row,
//   C = Q exp(ref - lse);  xs = C x;  slab[listed] = (Q softmax - q) / C, from the fp32 logit and rounded once.
template <typename T>
__global__ void __launch_bounds__(256)
distill_finish_kernel(const T* __restrict__ x, long long x_ld, T* __restrict__ xs, long long xs_ld, int hidden,
                      T* __restrict__ slab, long long slab_ld, const float* __restrict__ ref,
                      const float* __restrict__ lse, const float* __restrict__ mass, const TeacherRows t,
                      int rows_valid, float* __restrict__ row_coef) {
  const int r = blockIdx.x;
  const bool exists = r < rows_valid;
  const float l = exists ? lse[r] : 0.f;
  const float Q = exists ? mass[r] : 0.f;
  float C = Q != 0.f ? Q * __expf(ref[r] - l) : 0.f;
  if (Q != 0.f && fabsf(C) < 1e-30f) C = 1e-30f;  // keeps the entries finite
  if (threadIdx.x == 0) row_coef[r] = C;
  if (Q != 0.f) {
    const int n = t.start[(long long)t.n_tiles * t.start_ld + r];
    for (int k = threadIdx.x; k < n; k += blockDim.x) {
      const long long at = (long long)r * t.k + k;
      slab[(long long)r * slab_ld + t.idx[at]] = cast_from_float<T>(listed_dz(t.z[at], l, Q, t.q[at]) / C);
    }
  }
  const T* src = x + (long long)r * x_ld;
  T* dst = xs + (long long)r * xs_ld;
  for (int c = threadIdx.x * 8; c < hidden; c += blockDim.x * 8) {  // hidden % 8 == 0
    Vec8<T> v;
    float f[8];
    if (exists) {
      v.load(src + c);
      v.to_float(f);
#pragma unroll
      for (int k = 0; k < 8; ++k) f[k] *= C;
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) f[k] = 0.f;
    }
    v.from_float(f);
    v.store(dst + c);
  }
}

// Per-tile mode (see dz_transform_kernel): slab = boost * (Q softmax - q), in place. boost: a power of two that the
// contractions divide by again. |dZ| <= 1 before it is scaled, so fp16 has room for 2^14, without which a softmax entry of 1 / V is
// a subnormal number.
template <typename T>
__global__ void __launch_bounds__(256)
distill_dz_kernel(T* __restrict__ slab, long long slab_ld, const float* __restrict__ tile_max,
                  const float* __restrict__ lse, const float* __restrict__ mass, const TeacherRows t, int rows,
                  int rows_valid, int n_tiles, long long stat_ld, float boost) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long items = (long long)(rows / 8) * n_tiles;
  for (long long item = blockIdx.x; item < items; item += gridDim.x) {
    const int tile = (int)(item % n_tiles);
    const int r = (int)(item / n_tiles) * 8 + warp;
    const bool exists = r < rows_valid;
    const float Q = exists ? mass[r] : 0.f;
    const float l = exists ? lse[r] : 0.f;
    const float coef = Q != 0.f ? Q * __expf(tile_max[(long long)tile * stat_ld + r] - l) * boost : 0.f;
    T* ptr = slab + (long long)r * slab_ld + (long long)tile * 256 + lane * 8;
    Vec8<T> v;
    v.load(ptr);
    float f[8];
    v.to_float(f);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] *= coef;
    if (Q != 0.f) {
      const int end = t.start[(long long)(tile + 1) * t.start_ld + r];
      for (int k = t.start[(long long)tile * t.start_ld + r]; k < end; ++k) {
        const long long at = (long long)r * t.k + k;
        const int c = t.idx[at] - tile * 256;
        if ((c >> 3) == lane) {
          const float dz = listed_dz(t.z[at], l, Q, t.q[at]) * boost;
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (i == (c & 7)) f[i] = dz;
        }
      }
    }
    v.from_float(f);
    v.store(ptr);
  }
}

__global__ void distill_finalize_kernel(const PassScalars* sc, float temperature, float* __restrict__ loss) {
  if (threadIdx.x != 0 || blockIdx.x != 0) return;
  double v = sc->sum_nll / (double)sc->n_valid * ((double)temperature * (double)temperature);  // no valid row: NaN
  if (sc->status != 0) v = NAN;
  *loss = (float)v;
}

}  // namespace lce
