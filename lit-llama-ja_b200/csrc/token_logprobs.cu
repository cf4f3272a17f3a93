// Log-probabilities of given tokens: (l_t - m) / T - log(sum exp((l - m) / T)), a row of logits a token.
//
// One pass over the row, bound by memory: a thread keeps the largest logit that it has met, how many equal it, and the others' sum under it; both meet at the end.
// What equals the largest is counted, not summed: where one token has all but 2^-24, its score is the logarithm of the others' sum, which 1 + sum in 32 bits has lost.
#include "row_values.cuh"

namespace llb {
namespace {

__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// exp((l - m) / T) over some logits: the largest one, how many equal it, the others' sum.
struct RowSum {
  float m, ones, sum;
  __device__ __forceinline__ void under(float top, float c) {      // top >= m
    if (top == m) return;
    const float f = exp2_fast((m - top) * c);
    sum = (sum + ones) * f;
    ones = 0.f;
    m = top;
  }
  __device__ __forceinline__ void join(RowSum o, float c) {
    const float top = fmaxf(m, o.m);
    under(top, c);
    o.under(top, c);
    ones += o.ones;
    sum += o.sum;
  }
};

struct LogprobArgs {
  const void* logits;
  long long row;
  int R, V;
  const int64_t* tokens;
  const float* temperature;
  float temperature_all;
  float* out;
};

// `THREADS` threads a row; a warp has a row of its own where there are 32 (eight rows a block).
constexpr int LP_WIDE = 512, LP_NARROW = 32, LP_BATCH = 4;      // LP_BATCH: vectors that a thread asks for at once
template <typename T, int THREADS>
__global__ void __launch_bounds__(THREADS == LP_NARROW ? 256 : THREADS) token_logprobs_kernel(const LogprobArgs a) {
  constexpr int N = row_vec<T>::n, ROWS = THREADS == LP_NARROW ? 8 : 1;
  const int r = blockIdx.x * ROWS + (ROWS > 1 ? threadIdx.x >> 5 : 0), t = ROWS > 1 ? threadIdx.x & 31 : threadIdx.x, V = a.V;
  if (r >= a.R) return;
  const T* l = (const T*)a.logits + r * a.row;
  const float temperature = a.temperature ? a.temperature[r] : a.temperature_all;
  const float c = (float)(1.4426950408889634 / (double)temperature);
  const int64_t token = a.tokens[r];
  const bool there = token >= 0 && token < V;
  const float mine = there ? dt<T>::ld(l, token) : 0.f;
  RowSum s{-INFINITY, 0.f, 0.f};
#pragma unroll 1
  for (int i0 = t * N - row_offset(l); i0 < V; i0 += LP_BATCH * THREADS * N) {
    float x[LP_BATCH][N];
#pragma unroll
    for (int b = 0; b < LP_BATCH; ++b) load_values(l, i0 + b * THREADS * N, V, x[b]);
    float top = s.m;
#pragma unroll
    for (int b = 0; b < LP_BATCH; ++b)
#pragma unroll
      for (int e = 0; e < N; ++e) top = fmaxf(top, x[b][e]);
    s.under(top, c);
#pragma unroll
    for (int b = 0; b < LP_BATCH; ++b) {
      float part = 0.f;
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const bool one = x[b][e] == s.m;
        part += one ? 0.f : exp2_fast((x[b][e] - s.m) * c);
        s.ones += one ? 1.f : 0.f;
      }
      s.sum += part;
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s.join(RowSum{__shfl_xor_sync(0xffffffffu, s.m, o), __shfl_xor_sync(0xffffffffu, s.ones, o), __shfl_xor_sync(0xffffffffu, s.sum, o)}, c);
  if constexpr (ROWS == 1) {
    __shared__ float s_part[3][THREADS / 32];
    if ((t & 31) == 0) s_part[0][t >> 5] = s.m, s_part[1][t >> 5] = s.ones, s_part[2][t >> 5] = s.sum;
    __syncthreads();
    if (t >= 32) return;
    s = t < THREADS / 32 ? RowSum{s_part[0][t], s_part[1][t], s_part[2][t]} : RowSum{-INFINITY, 0.f, 0.f};
#pragma unroll
    for (int o = THREADS / 64; o > 0; o >>= 1) s.join(RowSum{__shfl_xor_sync(0xffffffffu, s.m, o), __shfl_xor_sync(0xffffffffu, s.ones, o), __shfl_xor_sync(0xffffffffu, s.sum, o)}, c);
  }
  if (t == 0) {
    const bool ok = there && temperature > 0.f && temperature < INFINITY && s.m > -INFINITY;
    const double d = mine == s.m ? 0.0 : ((double)mine - (double)s.m) / (double)temperature;
    a.out[r] = ok ? (float)(d - log((double)s.ones + (double)s.sum)) : NAN;
  }
}

template <typename T>
void launch_logprobs(const LogprobArgs& a, cudaStream_t st) {
  if (a.V <= 1024) token_logprobs_kernel<T, LP_NARROW><<<(a.R + 7) / 8, 256, 0, st>>>(a);
  else token_logprobs_kernel<T, LP_WIDE><<<a.R, LP_WIDE, 0, st>>>(a);
}

}  // namespace
}  // namespace llb

using namespace llb;

extern "C" {

int ll_token_logprobs(const void* logits, int dtype, int R, int V, long long row, const int64_t* tokens, const float* temperature, float temperature_all, float* out,
                      ll_stream stream) {
  LL_CHECK_ARG(logits && tokens && out && R > 0 && V > 0 && V <= 1 << 18, "token_logprobs: %d rows of %d logits (1 to %d)", R, V, 1 << 18);
  LL_CHECK_ARG(dtype == LL_F32 || dtype == LL_BF16 || dtype == LL_F16, "token_logprobs: type %d", dtype);
  LL_CHECK_ARG((uintptr_t)logits % (dtype == LL_F32 ? 4 : 2) == 0, "token_logprobs: logits at %p", logits);
  const LogprobArgs a{logits, row, R, V, tokens, temperature, temperature_all, out};
  if (dtype == LL_F32) launch_logprobs<float>(a, (cudaStream_t)stream);
  else if (dtype == LL_BF16) launch_logprobs<__nv_bfloat16>(a, (cudaStream_t)stream);
  else launch_logprobs<__half>(a, (cudaStream_t)stream);
  LL_LAUNCH_OK("token_logprobs_kernel");
  return LL_OK;
}

}  // extern "C"
