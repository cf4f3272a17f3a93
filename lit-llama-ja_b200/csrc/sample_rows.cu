// A token a row of logits from a given random number: temperature, top-k, top-p and min-p (the definition: include/llb200.h).
//
// Weights are whole numbers, w = rint(2^44 exp((l - m) / T)): V of them have a sum of 62 bits, exactly, so that neither a border of top-p nor a draw depends on
// the order of sums.  Both borders are values: top-k's the largest x with k logits at or above it, top-p's the largest x with top_p of the kept weight there.
#include "common.cuh"

namespace llb {
namespace {

constexpr int SR_THREADS = 1024;
constexpr double SR_ONE = 17592186044416.0;      // 2^44

// Numbers in the order of their values, as whole numbers; 0 and -0 are one.
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

struct SampleArgs {
  const void* logits;
  long long row;
  int V;
  const float *u, *temperature, *top_p, *min_p;
  const int32_t* top_k;
  float temperature_all, top_p_all, min_p_all;
  int top_k_all;
  int64_t* tokens;
};

template <typename V>
__device__ __forceinline__ V block_sum(V v, V* s) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  V all = s[threadIdx.x & 31];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
  return all;
}

// A block a row; borders by bisection over the numbers' keys.
template <typename T>
__global__ void __launch_bounds__(SR_THREADS) sample_rows_kernel(const SampleArgs a) {
  __shared__ long long s_sum[32];
  __shared__ uint32_t s_key[32];
  __shared__ long long s_before[32];
  const int r = blockIdx.x, t = threadIdx.x, lane = t & 31, warp = t >> 5, V = a.V;
  const T* l = (const T*)a.logits + r * a.row;
  const float u = a.u[r], T_ = a.temperature ? a.temperature[r] : a.temperature_all, p = a.top_p ? a.top_p[r] : a.top_p_all, mp = a.min_p ? a.min_p[r] : a.min_p_all;
  const int k = a.top_k ? a.top_k[r] : a.top_k_all;
  uint32_t top = 0;
  int bad = !(u >= 0.f && u <= 1.f) || !(T_ >= 0.f && T_ < INFINITY) || isnan(p) || isnan(mp);
  for (int i = t; i < V; i += SR_THREADS) {
    const float x = dt<T>::ld(l, i);
    bad |= isnan(x);
    top = max(top, order_key(x));
  }
  top = __reduce_max_sync(0xffffffffu, top);
  if (lane == 0) s_key[warp] = top;
  bad = __syncthreads_or(bad);
  top = __reduce_max_sync(0xffffffffu, s_key[lane]);
  if (bad || top <= order_key(-INFINITY)) {
    if (t == 0) a.tokens[r] = -1;
    return;
  }
  const float m = __uint_as_float(top & 0x80000000u ? top & 0x7fffffffu : ~top);
  const double inv = 1.0 / (double)T_;
  auto weight = [&](float x) -> long long {
    if (x == m) return (long long)SR_ONE;
    return T_ == 0.f ? 0 : (long long)rint(exp(((double)x - (double)m) * inv) * SR_ONE);
  };
  uint32_t border = 0;
  // the largest key at or above which `measure` reaches `target`
  auto select = [&](auto measure, auto reached) {
    uint32_t lo = border, hi = top;
    while (lo < hi) {
      const uint32_t mid = lo + (hi - lo + 1) / 2;
      long long n = 0;
      for (int i = t; i < V; i += SR_THREADS) {
        const float x = dt<T>::ld(l, i);
        if (order_key(x) >= mid) n += measure(x);
      }
      if (reached(block_sum(n, s_sum))) lo = mid;
      else hi = mid - 1;
    }
    border = lo;
  };
  auto kept_sum = [&]() {
    long long n = 0;
    for (int i = t; i < V; i += SR_THREADS) {
      const float x = dt<T>::ld(l, i);
      if (order_key(x) >= border) n += weight(x);
    }
    return block_sum(n, s_sum);
  };
  if (k >= 1 && k < V) select([&](float) -> long long { return 1; }, [&](long long n) { return n >= k; });
  if (p < 1.f) {
    const double want = (double)p * (double)kept_sum();
    select(weight, [&](long long n) { return (double)n >= want && n > 0; });
  }
  const double least = fmin((double)mp, 1.0) * SR_ONE;
  auto kept = [&](float x) -> long long {
    if (order_key(x) < border) return 0;
    const long long w = weight(x);
    return (double)w >= least ? w : 0;
  };
  // warps have runs of the row, one after the other
  const int run = (V + 31) / 32, i0 = warp * run, i1 = min(V, i0 + run);
  long long n = 0;
  for (int i = i0 + lane; i < i1; i += 32) n += kept(dt<T>::ld(l, i));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
  __syncthreads();
  if (lane == 0) s_before[warp] = n;
  __syncthreads();
  long long total = 0, before = 0;
  for (int w = 0; w < 32; ++w) {
    if (w == warp) before = total;
    total += s_before[w];
  }
  const long long target = T_ == 0.f ? 0 : min((long long)floor((double)u * (double)total), total - 1);
  if (target < before || target >= before + n) return;
  for (int i = i0; i < i1; i += 32) {
    const long long w = i + lane < i1 ? kept(dt<T>::ld(l, i + lane)) : 0;
    long long incl = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    const uint32_t past = __ballot_sync(0xffffffffu, before + incl > target);
    if (past != 0u) {
      if (lane == 0) a.tokens[r] = i + __ffs(past) - 1;
      return;
    }
    before += __shfl_sync(0xffffffffu, incl, 31);
  }
}

}  // namespace
}  // namespace llb

using namespace llb;

extern "C" {

int ll_sample_rows(const void* logits, int dtype, int R, int V, long long row, const float* u, const float* temperature, float temperature_all, const int32_t* top_k,
                   int top_k_all, const float* top_p, float top_p_all, const float* min_p, float min_p_all, int64_t* tokens, ll_stream stream) {
  LL_CHECK_ARG(logits && u && tokens && R > 0 && V > 0 && V <= 1 << 18, "sample_rows: %d rows of %d logits (1 to %d)", R, V, 1 << 18);
  LL_CHECK_ARG(dtype == LL_F32 || dtype == LL_BF16 || dtype == LL_F16, "sample_rows: type %d", dtype);
  const SampleArgs a{logits, row, V, u, temperature, top_p, min_p, top_k, temperature_all, top_p_all, min_p_all, top_k_all, tokens};
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == LL_F32) sample_rows_kernel<float><<<R, SR_THREADS, 0, st>>>(a);
  else if (dtype == LL_BF16) sample_rows_kernel<__nv_bfloat16><<<R, SR_THREADS, 0, st>>>(a);
  else sample_rows_kernel<__half><<<R, SR_THREADS, 0, st>>>(a);
  LL_LAUNCH_OK("sample_rows_kernel");
  return LL_OK;
}

}  // extern "C"
