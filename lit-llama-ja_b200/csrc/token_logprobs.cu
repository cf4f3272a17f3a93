// Log-probabilities of given tokens: l_t / T - m - log(sum exp(l / T - m)), a row of logits a token.
#include "common.cuh"

namespace llb {
namespace {

constexpr int LP_THREADS = 512;

// A block a row: the largest logit, then the sum in 64 bits.
template <typename T>
__global__ void __launch_bounds__(LP_THREADS) token_logprobs_kernel(const T* __restrict__ logits, int V, long long row, const int64_t* __restrict__ tokens,
                                                                   const float* __restrict__ temperature, float temperature_all, float* __restrict__ out) {
  __shared__ float s_max[LP_THREADS / 32];
  __shared__ double s_sum[LP_THREADS / 32];
  const int r = blockIdx.x, t = threadIdx.x, lane = t & 31, warp = t >> 5;
  const T* l = logits + r * row;
  const double inv = 1.0 / (double)(temperature ? temperature[r] : temperature_all);
  const int64_t token = tokens[r];
  float m = -INFINITY;
  bool none = false;
  for (int i = t; i < V; i += LP_THREADS) {
    const float x = dt<T>::ld(l, i);
    none |= isnan(x);
    m = fmaxf(m, x);
  }
  m = warp_max(m);
  if (lane == 0) s_max[warp] = m;
  none = __syncthreads_or(none);
  for (int w = 0; w < LP_THREADS / 32; ++w) m = fmaxf(m, s_max[w]);
  double sum = 0.0;
  for (int i = t; i < V; i += LP_THREADS) {
    const float x = dt<T>::ld(l, i);
    sum += x == m ? 1.0 : exp(((double)x - (double)m) * inv);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) s_sum[warp] = sum;
  __syncthreads();
  if (t == 0) {
    sum = 0.0;
    for (int w = 0; w < LP_THREADS / 32; ++w) sum += s_sum[w];
    const bool there = token >= 0 && token < V && inv > 0.0 && inv < INFINITY && !none && m > -INFINITY;
    const float x = there ? dt<T>::ld(l, token) : 0.f;
    out[r] = there ? (float)((x == m ? 0.0 : ((double)x - (double)m) * inv) - log(sum)) : NAN;
  }
}

}  // namespace
}  // namespace llb

using namespace llb;

extern "C" {

int ll_token_logprobs(const void* logits, int dtype, int R, int V, long long row, const int64_t* tokens, const float* temperature, float temperature_all, float* out,
                      ll_stream stream) {
  LL_CHECK_ARG(logits && tokens && out && R > 0 && V > 0 && V <= 1 << 18, "token_logprobs: %d rows of %d logits (1 to %d)", R, V, 1 << 18);
  LL_CHECK_ARG(dtype == LL_F32 || dtype == LL_BF16 || dtype == LL_F16, "token_logprobs: type %d", dtype);
  cudaStream_t st = (cudaStream_t)stream;
#define LP(TT) token_logprobs_kernel<TT><<<R, LP_THREADS, 0, st>>>((const TT*)logits, V, row, tokens, temperature, temperature_all, out);
  if (dtype == LL_F32) { LP(float) }
  else if (dtype == LL_BF16) { LP(__nv_bfloat16) }
  else { LP(__half) }
#undef LP
  LL_LAUNCH_OK("token_logprobs_kernel");
  return LL_OK;
}

}  // extern "C"
