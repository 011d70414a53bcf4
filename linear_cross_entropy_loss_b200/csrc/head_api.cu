// C ABI of the operators on given logits (include/lce_b200.h): argument checks and launches.
#include "launch.h"
#include "sample_logits.cuh"
#include "top_logits.cuh"

namespace {

using namespace lce;

int check_rows(int dtype, const void* logits, long long ld, long long rows, long long vocab) {
  if (dtype != LCE_DTYPE_F16 && dtype != LCE_DTYPE_BF16 && dtype != LCE_DTYPE_F32) return LCE_ERR_INVALID_ARGUMENT;
  if (rows < 0 || vocab <= 0 || ld < 0 || (rows > 0 && logits == nullptr)) return LCE_ERR_INVALID_ARGUMENT;
  if (rows > (1ll << 30) || vocab > (1ll << 30)) return LCE_ERR_TOO_LARGE;
  if ((reinterpret_cast<uintptr_t>(logits) & (dtype == LCE_DTYPE_F32 ? 3u : 1u)) != 0) return LCE_ERR_MISALIGNED;
  return LCE_OK;
}

int power_of_two_from(long long n) {
  int p = 1;
  while (p < n) p <<= 1;
  return p;
}

template <typename T>
int launch_top(const void* logits, int64_t ld, int64_t rows, int64_t vocab, int k, float inv_t, void* values,
               int64_t* indices, float* lse, cudaStream_t st) {
  top_logits_kernel<T><<<(int)rows, kTopThreads, 0, st>>>(
      reinterpret_cast<const T*>(logits), ld, (uint32_t)vocab, k, power_of_two_from(k), inv_t,
      reinterpret_cast<T*>(values), reinterpret_cast<long long*>(indices), lse);
  return check_launch();
}

template <typename T>
int launch_sample(const void* logits, int64_t ld, int64_t rows, int64_t vocab, const SampleParams& p, int64_t* tokens,
                  float* logprobs, cudaStream_t st) {
  int bits = kWeightBits;  // the sum over the row stays below 2^62
  while (bits > 0 && (vocab << bits) > (1ll << 62)) --bits;
  sample_logits_kernel<T><<<(int)rows, kSampleThreads, 0, st>>>(reinterpret_cast<const T*>(logits), ld, (uint32_t)vocab,
                                                                bits, p, reinterpret_cast<long long*>(tokens), logprobs);
  return check_launch();
}

}  // namespace

extern "C" {

int lce_top_logits(int32_t dtype, const void* logits, int64_t ld, int64_t rows, int64_t vocab, int32_t k,
                   float temperature, void* values, int64_t* indices, float* lse, void* stream) {
  const int v = check_rows(dtype, logits, ld, rows, vocab);
  if (v != LCE_OK) return v;
  if (k < 1 || !(temperature > 0.f)) return LCE_ERR_INVALID_ARGUMENT;
  if (k > vocab || k > kTopMax) return LCE_ERR_TOO_LARGE;
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
  SampleParams p;
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
