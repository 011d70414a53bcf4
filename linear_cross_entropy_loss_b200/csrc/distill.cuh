// Distillation from a teacher's top logits on the contraction engine of the cross-entropy loss.
//
//   q_k  = softmax of the listed teacher logits / T (or exp(t_k / T - lse) when the teacher's log-sum-exp is given)
//   loss = T^2 / n sum_i sum_k q_ik (log q_ik - z_ik / T + logsumexp_j(z_ij / T))
//   dZ_i = T / n (Q_i softmax(z_i / T) - sum_k q_ik [idx_ik = j]),   Q_i = sum_k q_ik
//
// The same shape as cross-entropy, with a row factor Q_i and a short sorted list in the place of the one label:
//   teacher_prepare_kernel  q, Q, sum q log q; each row's list sorted by index, equal indices merged, with the place in
//                           the list at which every 256-column tile of the vocabulary begins
//   forward contraction     its epilogue also copies the logits at the listed columns (gather_listed in gemm_sm100.cuh)
//   row statistics          sum_k q z - sum_k q log q in the place of the label's logit
//   distill_finish_kernel / distill_dz_kernel   dZ from the slab, with the listed entries written from their fp32 logits
// then the dx and dW contractions as they are.
//
// What bounds it: the three contractions, 6 N H V operations. At N=4096 H=2048 V=32768 K=32 (bf16) they take 1,060 of
// the 1,164 us of a step's kernels (one after the other, cold), preparing the lists 14, the listed entries of dZ and the
// scaled rows of x 17; at N=8192 H=2048 V=131072 K=64 a step takes 10.5 to 11.1 ms, 1,190 to 1,260 TFLOP/s.
//
// Roundings to the element type. dZ is an operand of the tensor cores, so the slab has the type of x: one rounding of
// each entry (listed entries once, from fp32). One base per row (bf16, fp32 slabs): the row's factor C goes into the
// fp32 epilogue of dx, but for dW, where rows are summed over, into a copy C x of the rows of x, a second rounding;
// with the result's own the error of dW is sqrt(3) times one rounding (2.9e-3 of its norm for bf16 against 1.7e-3).
// Powers of two in the place of C would be exact, but C is known only after the exponentials are stored. Per-tile
// slabs round each entry twice and x not at all.
#pragma once

#include "aux_kernels.cuh"

namespace lce {

constexpr int kTeacherMax = 1024;         // entries per row
constexpr int kPrepareThreads = 256;
constexpr int kPrepareEntries = 4096;     // entries a block holds: its rows x their length rounded up to 2^n

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
// One warp has a row, of `padded` (a power of two) entries; a block has rows_per_block <= 8 of them, as many as its
// shared memory holds. The work is short chains of shuffles and shared-memory steps, so what counts is that many
// warps run at once: 4096 rows of 32 entries take 14 us, against 27 us with 32 rows in a block.
template <bool kLists>
__global__ void __launch_bounds__(kPrepareThreads)
teacher_prepare_kernel(const TeacherInput t, long long row0, int rows, long long vocab, int rows_per_block, int padded,
                       long long ignored, long long* __restrict__ labels, float* __restrict__ mass,
                       float* __restrict__ plogp, int* __restrict__ list_idx, float* __restrict__ list_q,
                       unsigned short* __restrict__ start, long long start_ld, int n_tiles) {
  __shared__ unsigned long long list[kPrepareEntries];  // column << 32 | bits of q
  __shared__ int lengths[kPrepareThreads / 32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int first = blockIdx.x * rows_per_block;
  const int r = first + warp;
  unsigned long long* mine = list + warp * padded;
  if (warp < rows_per_block && r < rows) {
    float top = -INFINITY;
    bool bad = false;  // NaN or +inf among the entries that are there
    for (int k = lane; k < padded; k += 32) {
      uint32_t col = 0xffffffffu;
      float l = -INFINITY;
      if (k < t.k) {
        col = teacher_column(t, row0 + r, k, vocab);
        if (col != 0xffffffffu) l = teacher_logit(t, row0 + r, k);
        if (!(l > -INFINITY) && l == l) col = 0xffffffffu;  // -inf: no weight
      }
      bad |= l != l || l == INFINITY;
      top = fmaxf(top, l);
      mine[k] = ((unsigned long long)col << 32) | __float_as_uint(l);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    bad = __any_sync(0xffffffffu, bad);
    // q = exp(log_share) / total. Without a given log-sum-exp the largest logit comes off before the division by T:
    // finite logits over a low T may be more than a float holds, their distances are what counts.
    const bool given = t.lse != nullptr;
    const float base = given ? t.lse[row0 + r] : 0.f;
    auto log_share = [&](float l) {
      if (!given) return (l - top) * t.inv_temperature;
      const float scaled = l * t.inv_temperature;
      return scaled > -INFINITY ? scaled - base : -INFINITY;
    };
    float total = 1.f;
    if (!given) {
      total = 0.f;
      for (int k = lane; k < padded; k += 32)
        if (uint32_t(mine[k] >> 32) != 0xffffffffu) total += expf(log_share(__uint_as_float(uint32_t(mine[k]))));
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    }
    const float log_total = logf(total);
    float sum = 0.f, ent = 0.f;
    for (int k = lane; k < padded; k += 32) {
      uint32_t col = uint32_t(mine[k] >> 32);
      float q = 0.f;
      if (col != 0xffffffffu) {
        const float log_q = log_share(__uint_as_float(uint32_t(mine[k]))) - log_total;
        q = bad ? __uint_as_float(0x7fc00000u) : expf(log_q);
        if (q == 0.f) col = 0xffffffffu;
        else ent += q * log_q;
        sum += q;
      }
      mine[k] = ((unsigned long long)col << 32) | __float_as_uint(q);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      sum += __shfl_xor_sync(0xffffffffu, sum, o);
      ent += __shfl_xor_sync(0xffffffffu, ent, o);
    }
    if (lane == 0) {
      labels[r] = sum == 0.f ? ignored : -1;  // a NaN counts: it has to reach the loss
      mass[r] = sum;
      plogp[r] = ent;
    }
    if (kLists) {
      // by column, ascending (what is not there comes last)
      for (int size = 2; size <= padded; size <<= 1) {
        for (int stride = size >> 1; stride > 0; stride >>= 1) {
          __syncwarp();
          for (int i = lane; i < padded / 2; i += 32) {
            const int lo = ((i & ~(stride - 1)) << 1) | (i & (stride - 1));
            const int hi = lo | stride;
            const unsigned long long x = mine[lo], y = mine[hi];
            if ((x > y) == ((lo & size) == 0)) {
              mine[lo] = y;
              mine[hi] = x;
            }
          }
        }
      }
      __syncwarp();
      // equal columns become one entry with the sum of their q (in ascending order of q); the list moves together in
      // place
      int length = 0;
      for (int k0 = 0; k0 < padded; k0 += 32) {
        const int k = k0 + lane;
        const uint32_t col = k < padded ? uint32_t(mine[k] >> 32) : 0xffffffffu;
        // (a place before k0 may have been written already, with an entry of no higher column)
        const uint32_t before = k > k0 && k < padded ? uint32_t(mine[k - 1] >> 32) : 0xffffffffu;
        const bool head = col != 0xffffffffu &&
                          (k == k0 ? length == 0 || uint32_t(mine[length - 1] >> 32) != col : col != before);
        float q = 0.f;
        if (head)
          for (int m = k; m < padded && uint32_t(mine[m] >> 32) == col; ++m) q += __uint_as_float(uint32_t(mine[m]));
        const uint32_t heads = __ballot_sync(0xffffffffu, head);
        __syncwarp();  // all have read what the places below are about to hold
        const int at = length + __popc(heads & ((1u << lane) - 1u));
        if (head) {
          mine[at] = ((unsigned long long)col << 32) | __float_as_uint(q);
          list_idx[(long long)r * t.k + at] = int(col);
          list_q[(long long)r * t.k + at] = q;
        }
        length += __popc(heads);
        __syncwarp();
      }
      if (lane == 0) lengths[warp] = length;
    }
  }
  if (!kLists) return;
  __syncthreads();
  // start[tile][r]: entries of row r with a column before tile * 256
  for (int i = threadIdx.x; i < (n_tiles + 1) * rows_per_block; i += kPrepareThreads) {
    const int tile = i / rows_per_block, b = i - tile * rows_per_block;
    if (first + b >= rows) continue;
    const unsigned long long* row = list + b * padded;
    const unsigned long long from = (unsigned long long)tile << 40;  // column tile * 256
    int lo = 0, hi = lengths[b];
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (row[mid] < from) lo = mid + 1;
      else hi = mid;
    }
    start[(long long)tile * start_ld + first + b] = (unsigned short)lo;
  }
}

// dZ / T * n of one listed entry.
__device__ __forceinline__ float listed_dz(float z, float lse, float mass, float q) { return expf(z - lse) * mass - q; }

// The chunk's conditional re-run is behind: its flags are counted and cleared for the next chunk. One block.
__device__ __forceinline__ void close_rescue(PassScalars* sc, int* rescue_groups, int n_groups, int rows) {
  int flagged = 0;
  for (int g0 = 0; g0 < n_groups; g0 += blockDim.x) {
    const int g = g0 + int(threadIdx.x);
    flagged += __syncthreads_count(g + 1 < n_groups && rescue_groups[g] != 0);
    if (g < n_groups) rescue_groups[g] = 0;
  }
  if (threadIdx.x == 0) {
    sc->rerun_groups += flagged;
    sc->seen_groups += (rows + 255) >> 8;
  }
}
__global__ void close_rescue_kernel(PassScalars* sc, int* rescue_groups, int n_groups, int rows) {
  close_rescue(sc, rescue_groups, n_groups, rows);
}

// Row-reference mode (see row_finish_kernel): one block per row,
//   C = Q exp(ref - lse);  xs = C x;  slab[listed] = (Q softmax - q) / C, from the fp32 logit and rounded once.
// Where C is too small for that (row_factor) the slab takes the powers of two that are missing.
template <typename T>
__global__ void __launch_bounds__(256)
distill_finish_kernel(const T* __restrict__ x, long long x_ld, T* __restrict__ xs, long long xs_ld, int hidden,
                      T* __restrict__ slab, long long slab_ld, const float* __restrict__ ref,
                      const float* __restrict__ lse, const float* __restrict__ mass, const TeacherRows t,
                      int rows_valid, float* __restrict__ row_coef, PassScalars* sc, int* rescue_groups, int n_groups) {
  const int r = blockIdx.x;
  const bool exists = r < rows_valid;
  const float l = exists ? lse[r] : 0.f;
  const float Q = exists ? mass[r] : 0.f;
  float C = Q != 0.f ? Q * __expf(ref[r] - l) : 0.f;
  if (Q != 0.f && C < kLeastFactor) {  // (the whole block)
    const RowFactor f = row_factor(ref[r] - l, Q);
    shift_row(slab + (long long)r * slab_ld, slab_ld, f.shift);
    C = f.C;
  }
  if (threadIdx.x == 0) row_coef[r] = C;
  if (r == 0) close_rescue(sc, rescue_groups, n_groups, rows_valid);
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
// contractions divide by again. |dZ| <= 1 before it is scaled, so fp16 has room for 2^14, without which a softmax entry
// of 1 / V is a subnormal number. It reads and writes the slab once: 1000 x 50257 in fp16 31 us, 6.6 TB/s.
// grid: x over groups of kDzTiles tiles, y over groups of 8 rows. A warp takes the tiles of a row, all their loads on the
// way before the first is used. (One tile at a time, its place from 64-bit divisions: 58 us.)
constexpr int kDzTiles = 4;
template <typename T>
__global__ void __launch_bounds__(256)
distill_dz_kernel(T* __restrict__ slab, long long slab_ld, const float* __restrict__ tile_max,
                  const float* __restrict__ lse, const float* __restrict__ mass, const TeacherRows t, int rows,
                  int rows_valid, int n_tiles, long long stat_ld, float boost) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tile0 = blockIdx.x * kDzTiles;
  for (int r = blockIdx.y * 8 + warp; r < rows; r += gridDim.y * 8) {
    const bool exists = r < rows_valid;
    T* const ptr = slab + (long long)r * slab_ld + (long long)tile0 * 256 + lane * 8;
    Vec8<T> v[kDzTiles];
    float most[kDzTiles];
    int start[kDzTiles + 1];
#pragma unroll
    for (int i = 0; i < kDzTiles; ++i)
      if (tile0 + i < n_tiles) v[i].load(ptr + i * 256);
    const float Q = exists ? mass[r] : 0.f;
    const float l = exists ? lse[r] : 0.f;
#pragma unroll
    for (int i = 0; i < kDzTiles; ++i)
      most[i] = exists && tile0 + i < n_tiles ? tile_max[(long long)(tile0 + i) * stat_ld + r] : 0.f;
#pragma unroll
    for (int i = 0; i <= kDzTiles; ++i)
      start[i] = exists ? t.start[(long long)min(tile0 + i, n_tiles) * t.start_ld + r] : 0;
#pragma unroll
    for (int i = 0; i < kDzTiles; ++i) {
      if (tile0 + i >= n_tiles) break;
      const float coef = Q != 0.f ? Q * __expf(most[i] - l) * boost : 0.f;
      float f[8];
      v[i].to_float(f);
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] *= coef;
      if (Q != 0.f) {
        for (int k = start[i]; k < start[i + 1]; ++k) {
          const long long at = (long long)r * t.k + k;
          const int c = t.idx[at] - (tile0 + i) * 256;
          if ((c >> 3) == lane) {
            const float dz = listed_dz(t.z[at], l, Q, t.q[at]) * boost;
#pragma unroll
            for (int j = 0; j < 8; ++j)
              if (j == (c & 7)) f[j] = dz;
          }
        }
      }
      v[i].from_float(f);
      v[i].store(ptr + i * 256);
    }
  }
}

// One block: loss = T^2 / n * the sum of the rows' losses, always added up in the same order.
__global__ void __launch_bounds__(1024)
distill_finalize_kernel(const PassScalars* sc, const double* __restrict__ row_loss, long long rows, float temperature,
                        float* __restrict__ loss) {
  __shared__ double scratch[32];
  double v = 0.0;
  for (long long r = threadIdx.x; r < rows; r += blockDim.x) v += row_loss[r];
  v = block_sum_double(v, scratch);
  if (threadIdx.x != 0) return;
  v = v / (double)sc->n_valid * ((double)temperature * (double)temperature);  // no valid row: NaN
  if (sc->status != 0) v = NAN;
  *loss = (float)v;
}

// dst[r, c] = src[r, c] for rows that start anywhere: dst rows lie on 16-byte boundaries (dst_ld elements apart,
// whole vectors of them are written). A vector of dst is cut out of the two aligned vectors of src that hold it, so
// both sides move 16 bytes at a time (1000 x 50257 in fp16: 34 us, 5.9 TB/s; element by element 108 us). T: the bits
// of an element.
template <typename T>
__global__ void __launch_bounds__(256)
align_rows_kernel(const T* __restrict__ src, long long src_ld, T* __restrict__ dst, long long dst_ld, long long rows,
                  long long cols) {
  constexpr int kPer = 16 / int(sizeof(T));
  const long long per_row = (cols + kPer - 1) / kPer;
  const uintptr_t begin = reinterpret_cast<uintptr_t>(src);
  const uintptr_t end = reinterpret_cast<uintptr_t>(src + (rows - 1) * src_ld + cols);
  for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < rows * per_row;
       i += (long long)gridDim.x * blockDim.x) {
    const long long r = i / per_row, c = (i - r * per_row) * kPer;
    const T* from = src + r * src_ld + c;
    const uintptr_t at = reinterpret_cast<uintptr_t>(from);
    const uintptr_t low = at & ~uintptr_t(15);
    uint32_t w[8];
    if (low >= begin && low + 32 <= end) {
      const uint4 a = __ldg(reinterpret_cast<const uint4*>(low)), b = __ldg(reinterpret_cast<const uint4*>(low) + 1);
      w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w;
      w[4] = b.x; w[5] = b.y; w[6] = b.z; w[7] = b.w;
      const int bytes = int(at - low);
      if (bytes & 8) {
#pragma unroll
        for (int k = 0; k < 6; ++k) w[k] = w[k + 2];
      }
      if (bytes & 4) {
#pragma unroll
        for (int k = 0; k < 5; ++k) w[k] = w[k + 1];
      }
      if (bytes & 2) {
#pragma unroll
        for (int k = 0; k < 4; ++k) w[k] = __funnelshift_r(w[k], w[k + 1], 16);
      }
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) w[k] = 0;
#pragma unroll
      for (int k = 0; k < kPer; ++k)
        if (c + k < cols) w[k * int(sizeof(T)) / 4] |= uint32_t(from[k]) << (8 * (k * int(sizeof(T)) % 4));
    }
    *reinterpret_cast<uint4*>(dst + r * dst_ld + c) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// Two matrices times *factor, in place; untouched where the factor is exactly 1. Blocks below `split` have the first.
template <typename T>
__global__ void __launch_bounds__(256)
scale_pair_kernel(T* a, long long a_ld, long long a_rows, long long a_cols, T* b, long long b_ld, long long b_rows,
                  long long b_cols, int split, const float* __restrict__ factor) {
  const float f = *factor;
  if (f == 1.0f) return;
  const bool second = int(blockIdx.x) >= split;
  T* m = second ? b : a;
  const long long ld = second ? b_ld : a_ld, per_row = (second ? b_cols : a_cols) / 8;
  const long long n = (second ? b_rows : a_rows) * per_row;
  const long long block = second ? blockIdx.x - split : blockIdx.x, blocks = second ? gridDim.x - split : split;
  for (long long i = block * blockDim.x + threadIdx.x; i < n; i += blocks * blockDim.x) {
    const long long r = i / per_row, c = (i - r * per_row) * 8;
    Vec8<T> v;
    v.load(m + r * ld + c);
    float e[8];
    v.to_float(e);
#pragma unroll
    for (int k = 0; k < 8; ++k) e[k] *= f;
    v.from_float(e);
    v.store(m + r * ld + c);
  }
}

}  // namespace lce
