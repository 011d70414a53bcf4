// C ABI of the operators on given logits (include/lce_b200.h): argument checks and launches.
#include "launch.h"
#include "sample_logits.cuh"
#include "top_logits.cuh"

#include <algorithm>
#include <cmath>

namespace {

using namespace lce;

static_assert(LCE_TOP_MAX == kTopMax, "the header's limit");

int check_rows(int dtype, const void* logits, long long ld, long long rows, long long vocab) {
  if (dtype != LCE_DTYPE_F16 && dtype != LCE_DTYPE_BF16 && dtype != LCE_DTYPE_F32) return LCE_ERR_INVALID_ARGUMENT;
  if (rows < 0 || vocab <= 0 || ld < 0 || (rows > 0 && logits == nullptr)) return LCE_ERR_INVALID_ARGUMENT;
  if (rows > (1ll << 27) || vocab > (1ll << 30)) return LCE_ERR_TOO_LARGE;
  if ((reinterpret_cast<uintptr_t>(logits) & (dtype == LCE_DTYPE_F32 ? 3u : 1u)) != 0) return LCE_ERR_MISALIGNED;
  return LCE_OK;
}

// SMs of the current device (148 where that cannot be asked), read once per device.
int sm_count() {
  static std::atomic<int> known[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  int n = known[dev].load(std::memory_order_relaxed);
  if (n == 0) {
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) return 148;
    known[dev].store(n, std::memory_order_relaxed);
  }
  return n;
}

// Dynamic shared memory above 48 KiB has to be allowed for each kernel, once per device.
template <auto kKernel>
int allow_smem(size_t bytes) {
  static std::atomic<uint64_t> done{0};  // one bit per device
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return LCE_ERR_CUDA;
  if (dev < 0 || dev >= 64) return LCE_ERR_UNSUPPORTED_DEVICE;
  if ((done.load(std::memory_order_relaxed) >> dev) & 1u) return LCE_OK;
  if (cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) != cudaSuccess) {
    cudaGetLastError();
    return LCE_ERR_CUDA;
  }
  done.fetch_or(1ull << dev, std::memory_order_relaxed);
  return LCE_OK;
}

// One launch of `blocks` blocks in clusters of `parts`. `beside`: it may start once all blocks of the launch before it
// have started.
template <typename... Args, typename... Given>
int launch_clusters(void (*kernel)(Args...), long long blocks, int threads, size_t smem, int parts, bool beside,
                    cudaStream_t st, Given... given) {
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3((unsigned)blocks);
  config.blockDim = dim3((unsigned)threads);
  config.dynamicSmemBytes = smem;
  config.stream = st;
  cudaLaunchAttribute attrs[2];
  config.attrs = attrs;
  if (parts > 1) {
    cudaLaunchAttribute& attr = attrs[config.numAttrs++];
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = (unsigned)parts;
    attr.val.clusterDim.y = 1;
    attr.val.clusterDim.z = 1;
  }
  if (beside) {
    cudaLaunchAttribute& attr = attrs[config.numAttrs++];
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
  }
  if (cudaLaunchKernelEx(&config, kernel, Args(given)...) != cudaSuccess) {
    cudaGetLastError();
    return LCE_ERR_CUDA;
  }
  return check_launch();
}

// Blocks that share a row: doubled while the blocks of all rows fit the GPU at once (three of kTopThreads on an SM),
// a part keeps a whole batch, and the lists of all parts fit one.
template <typename T>
int top_parts(int64_t rows, int64_t vocab, int k) {
  const int64_t batch = (int64_t)kTopBatch * (32 / (int)sizeof(T));
  int parts = 1;
  while (parts < kTopParts && rows * parts * 2 <= 3ll * sm_count() && vocab >= batch * parts && k * parts * 2 <= kTopList)
    parts *= 2;
  return parts;
}

template <typename T>
int launch_top(const void* logits, int64_t ld, int64_t rows, int64_t vocab, int k, float inv_t, void* values,
               int64_t* indices, float* lse, cudaStream_t st) {
  const int parts = top_parts<T>(rows, vocab, k);
  const int v = allow_smem<&top_logits_kernel<T>>(sizeof(TopShared));
  if (v != LCE_OK) return v;
  return launch_clusters(top_logits_kernel<T>, rows * parts, kTopThreads, sizeof(TopShared), parts, false, st,
                         reinterpret_cast<const T*>(logits), (long long)ld, (uint32_t)vocab, k, parts, inv_t,
                         reinterpret_cast<T*>(values), reinterpret_cast<long long*>(indices), lse);
}

// Blocks that share a row of sample_row_kernel, and the vectors of 16 bytes that each keeps in shared memory (0: too
// long a row, it is read again for each sweep). A block keeps up to 65 KiB, so that two are on an SM; few rows are
// split further, down to 8 KiB; up to 176 KiB where eight blocks are not enough.
constexpr int64_t kRowCacheMax = 176 << 10;
static_assert((sizeof(RowShared) + 15) / 16 * 16 + kRowCacheMax <= 232448, "dynamic shared memory limit of sm_100");
void row_layout(int64_t rows, int64_t vocab, int es, int* parts, int* cache_vectors) {
  const int64_t bytes = vocab * es + 32;
  int n = 1;
  while (n < kRowParts && bytes > n * (65ll << 10)) n *= 2;
  while (n < kRowParts && rows * n * 2 <= 2ll * sm_count() && bytes > n * (16ll << 10)) n *= 2;
  const int64_t vectors = (bytes + 15) / 16;
  const int64_t each = (vectors + n - 1) / n;
  *parts = n;
  *cache_vectors = each * 16 <= kRowCacheMax ? (int)each : 0;
}

template <typename T>
int launch_sample(const void* logits_, int64_t ld, int64_t rows, int64_t vocab, SampleParams p, int64_t* tokens_,
                  float* logprobs, cudaStream_t st) {
  const T* logits = reinterpret_cast<const T*>(logits_);
  long long* tokens = reinterpret_cast<long long*>(tokens_);
  p.weight_bits = kWeightBits;  // the sum over the row stays below 2^62
  while (vocab > (1ll << (62 - p.weight_bits))) --p.weight_bits;
  // top_k for all rows: one of the two kernels has them all, but for greedy rows, which the list has. A top_k for
  // each row: both run, side by side, and a cluster whose row is the other's ends at once.
  const bool each = p.top_k != nullptr;
  const int want = each ? 256 : (int)std::min<long long>(std::max<long long>(p.top_k_all, 1), kTopMax);
  const int list_parts = top_parts<T>(rows, vocab, want);
  p.list_limit = std::min(kTopMax, kTopList / list_parts);
  const bool greedy = p.temperature != nullptr || !(p.temperature_all > 0.0);
  const bool lists = each || greedy || (p.top_k_all >= 1 && p.top_k_all <= p.list_limit);
  const bool others = each || ((p.temperature != nullptr || p.temperature_all > 0.0) &&
                               !(p.top_k_all >= 1 && p.top_k_all <= p.list_limit));
  int v;
  if (lists) {
    if ((v = allow_smem<&sample_list_kernel<T>>(sizeof(TopShared))) != LCE_OK) return v;
    if ((v = launch_clusters(sample_list_kernel<T>, rows * list_parts, kTopThreads, sizeof(TopShared), list_parts, false,
                             st, logits, (long long)ld, (uint32_t)vocab, list_parts, p, tokens, logprobs)) != LCE_OK)
      return v;
  }
  if (!others) return LCE_OK;
  int parts = 1, cache = 0;
  row_layout(rows, vocab, (int)sizeof(T), &parts, &cache);
  const size_t fixed = (sizeof(RowShared) + 15) / 16 * 16;
  if ((v = allow_smem<&sample_row_kernel<T>>(fixed + kRowCacheMax)) != LCE_OK) return v;
  return launch_clusters(sample_row_kernel<T>, rows * parts, kRowThreads, fixed + (size_t)cache * 16, parts, lists, st,
                         logits, (long long)ld, (uint32_t)vocab, parts, cache, p, tokens, logprobs);
}

}  // namespace

extern "C" {

int lce_top_logits(int32_t dtype, const void* logits, int64_t ld, int64_t rows, int64_t vocab, int32_t k,
                   float temperature, void* values, int64_t* indices, float* lse, void* stream) {
  const int v = check_rows(dtype, logits, ld, rows, vocab);
  if (v != LCE_OK) return v;
  // (a temperature whose log2(e) / T, the scale of the exponents, is a number too)
  if (k < 1 || !(temperature > 0.f) || !(temperature < INFINITY) || !(1.f / temperature * kLog2e < INFINITY))
    return LCE_ERR_INVALID_ARGUMENT;
  if (k > vocab || k > LCE_TOP_MAX) return LCE_ERR_TOO_LARGE;
  if (rows == 0) return LCE_OK;
  if (!values || !indices || !lse) return LCE_ERR_INVALID_ARGUMENT;
  cudaStream_t st = (cudaStream_t)stream;
  const float inv_t = 1.f / temperature;
  switch (dtype) {
    case LCE_DTYPE_F16: return launch_top<__half>(logits, ld, rows, vocab, k, inv_t, values, indices, lse, st);
    case LCE_DTYPE_BF16: return launch_top<__nv_bfloat16>(logits, ld, rows, vocab, k, inv_t, values, indices, lse, st);
  }
  return launch_top<float>(logits, ld, rows, vocab, k, inv_t, values, indices, lse, st);
}

int lce_sample_logits(int32_t dtype, const void* logits, int64_t ld, int64_t rows, int64_t vocab,
                      const lce_sampling* s, int64_t* tokens, float* logprobs, void* stream) {
  const int v = check_rows(dtype, logits, ld, rows, vocab);
  if (v != LCE_OK) return v;
  if (s == nullptr || (s->u_dtype != LCE_DTYPE_F32 && s->u_dtype != LCE_SAMPLING_U_F64)) return LCE_ERR_INVALID_ARGUMENT;
  if (!s->temperature && !(s->temperature_all >= 0.0)) return LCE_ERR_INVALID_ARGUMENT;
  if (!s->top_k && s->top_k_all < 0) return LCE_ERR_INVALID_ARGUMENT;
  if (!s->top_p && !(s->top_p_all > 0.0 && s->top_p_all <= 1.0)) return LCE_ERR_INVALID_ARGUMENT;
  if (!s->min_p && !(s->min_p_all >= 0.0 && s->min_p_all <= 1.0)) return LCE_ERR_INVALID_ARGUMENT;
  if (rows == 0) return LCE_OK;
  if (!s->u || !tokens || !logprobs) return LCE_ERR_INVALID_ARGUMENT;
  SampleParams p = {};
  p.u = s->u;
  p.u_is_double = s->u_dtype == LCE_SAMPLING_U_F64;
  p.temperature = s->temperature;
  p.top_k = s->top_k;
  p.top_p = s->top_p;
  p.min_p = s->min_p;
  p.temperature_all = s->temperature_all;
  p.top_k_all = s->top_k_all;
  p.top_p_all = s->top_p_all;
  p.min_p_all = s->min_p_all;
  cudaStream_t st = (cudaStream_t)stream;
  switch (dtype) {
    case LCE_DTYPE_F16: return launch_sample<__half>(logits, ld, rows, vocab, p, tokens, logprobs, st);
    case LCE_DTYPE_BF16: return launch_sample<__nv_bfloat16>(logits, ld, rows, vocab, p, tokens, logprobs, st);
  }
  return launch_sample<float>(logits, ld, rows, vocab, p, tokens, logprobs, st);
}

}  // extern "C"
