// Log-probabilities of given tokens: (l_t - m) / T - log(sum exp((l - m) / T)), a row of logits a token.
//
// One pass over the row, by warps, a batch at a time in registers: a warp finds its largest logit first, so that few vectors have one that equals it, and the others'
// exponentials are added under it without a look at each: four instructions a number.  Bound by memory: 777 rows of 100 003 (fp32) 51
// us, 92 % of the copy rate; 2048 of 32 000 (bf16) 31 us, 65 %, of which the exponentials alone take 15 (a largest logit a thread, looked for in every number: 40; a
// block's largest, behind a barrier a batch: 61 and 39).
// What equals the largest is counted, not summed: where one token has all but 2^-24, its score is the logarithm of the others' sum, which 1 + sum in 32 bits has lost.
#include <cooperative_groups.h>

#include "row_values.cuh"

namespace llb {
namespace {

namespace cg = cooperative_groups;

__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

__device__ __forceinline__ void add2(float2& a, float2 b) {
  asm("{\n\t.reg .b64 p, q;\n\tmov.b64 p, {%0, %1};\n\tmov.b64 q, {%2, %3};\n\tadd.rn.f32x2 p, p, q;\n\tmov.b64 {%0, %1}, p;\n\t}" : "+f"(a.x), "+f"(a.y) : "f"(b.x), "f"(b.y));
}
// (a - b) / (T ln 2).  FAR, for temperatures above 1e36: as (a / 4 - b / 4) (4 / (T ln 2)), since differences may be more than a number of 32 bits holds (their quarters are exact, and rounded
// once; the factor stays a normal number).  Under lower temperatures such differences come to less than -100, of which no exponential is left.
constexpr float LP_FAR = 1e36f;
template <bool FAR>
__device__ __forceinline__ float scaled(float a, float b, float c) { return (FAR ? fmaf(a, 0.25f, b * -0.25f) : a - b) * c; }
// exp((l - m) / T) over some logits: the largest one, how many equal it, the others' sum.
// Sum: of 64 bits for 32-bit numbers of a block's rows, of which a thread has up to 65 batches; of 32 for the others (17 of 16-bit numbers, 6 where a warp has a row).  With 32 for
// all, a slowly rising row, whose every batch has a new largest logit, took the error of a factor and some additions a batch (2^18 numbers that rise by up to 30: 2.6e-6 off, now 0.8e-6);
// with 64 for all, 2048 rows of 32 000 (bf16) took 31.8 us instead of 30.8.
template <typename Sum>
struct RowSum {
  float m, ones;
  Sum sum;
  template <bool FAR>
  __device__ __forceinline__ void under(float top, float c) {      // top >= m
    if (top == m) return;
    const float y = scaled<FAR>(m, top, c);
    sum += (Sum)ones;
    if (sizeof(Sum) == 8 && y > -1.f) {          // by the factor's difference from 1: many small steps are off by as much as one large one
      float p = 1.0178086e-7f;                   // (2^y - 1) / y: ln 2^k / k! from k = 9 down; the next term is under 2^-26
      p = fmaf(p, y, 1.3215487e-6f);
      p = fmaf(p, y, 1.5252734e-5f);
      p = fmaf(p, y, 1.5403530e-4f);
      p = fmaf(p, y, 1.3333558e-3f);
      p = fmaf(p, y, 9.6181291e-3f);
      p = fmaf(p, y, 5.5504109e-2f);
      p = fmaf(p, y, 2.4022651e-1f);
      p = fmaf(p, y, 6.9314718e-1f);
      sum = fma(sum, (Sum)(p * y), sum);
    } else {
      sum *= (Sum)exp2_fast(y);
    }
    ones = 0.f;
    m = top;
  }
  __device__ __forceinline__ void add_lanes() {      // of one largest logit
    ones = warp_sum(ones);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  }
};

struct LogprobArgs {
  const void* logits;
  long long row;
  int R, V, split;                               // split: blocks of a row, one cluster
  const int64_t* tokens;
  const float* temperature;
  float temperature_all;
  float* out;
};

// `THREADS` threads a row; a warp has a row of its own where there are 32 (eight rows a block).
constexpr int LP_WIDE = 256, LP_NARROW = 32, LP_MOST = 8;      // LP_MOST: blocks of a row
// Vectors that a thread asks for at once, and blocks of an SM: the exponentials of 16-bit numbers need fewer warps, 32-bit ones' bytes more (777 rows of 100 003 with eight and
// four 63 us, 2048 of 32 000 with four and six 30.5).
template <typename T> constexpr int lp_batch = sizeof(T) == 4 ? 4 : 8;
template <typename T> constexpr int lp_blocks = sizeof(T) == 4 ? 6 : 4;
template <typename T, int THREADS> using lp_sum = RowSum<typename std::conditional<sizeof(T) == 4 && THREADS == LP_WIDE, double, float>::type>;
// a - b and a * b of pairs, one instruction each
__device__ __forceinline__ float2 sub_mul2(float2 x, float m, float c) {
  float2 r;
  asm("{\n\t.reg .b64 p, q, s;\n\tmov.b64 p, {%2, %3};\n\tmov.b64 q, {%4, %4};\n\tmov.b64 s, {%5, %5};\n\tadd.rn.f32x2 p, p, q;\n\tmul.rn.f32x2 p, p, s;\n\tmov.b64 {%0, %1}, p;\n\t}"
      : "=f"(r.x), "=f"(r.y) : "f"(x.x), "f"(x.y), "f"(-m), "f"(c));
  return r;
}
// The row's largest logit, how many equal it and the others' sum, of the thread's numbers (a warp has one largest).
template <typename T, int THREADS, bool FAR>
__device__ __forceinline__ lp_sum<T, THREADS> row_sum(const T* l, int V, int t, int rank, int C, float c) {
  constexpr int LP_BATCH = lp_batch<T>, N = row_vec<T>::n;
  lp_sum<T, THREADS> s{-INFINITY, 0.f, 0};
#pragma unroll 1
  for (int at = rank * LP_BATCH * THREADS * N - row_offset(l); at < V; at += C * LP_BATCH * THREADS * N) {      // (all lanes go as often)
    const int i0 = at + t * N;
    uint4 raw[LP_BATCH];
#pragma unroll
    for (int b = 0; b < LP_BATCH; ++b)
      raw[b] = i0 + b * THREADS * N < V ? load_vector(l, i0 + b * THREADS * N, V) : none_vector<T>();
    float top = s.m;
#pragma unroll
    for (int b = 0; b < LP_BATCH; ++b) top = fmaxf(top, vec_max<T>(raw[b]));
    s.template under<FAR>(warp_max(top), c);
    float sum = 0.f;
#pragma unroll
    for (int b = 0; b < LP_BATCH; ++b) {
      float x[N];
      vec_values<T>(raw[b], x);
      float2 w[N / 2];
      if (FAR || __any_sync(0xffffffffu, vec_max<T>(raw[b]) == s.m)) {
        auto one = [&](float v) {
          if (v != s.m) return exp2_fast(scaled<FAR>(v, s.m, c));
          s.ones += 1.f;
          return 0.f;
        };
#pragma unroll
        for (int e = 0; e < N; e += 2) w[e / 2] = make_float2(one(x[e]), one(x[e + 1]));
      } else {
#pragma unroll
        for (int e = 0; e < N; e += 2) {
          const float2 d = sub_mul2(make_float2(x[e], x[e + 1]), s.m, c);
          w[e / 2] = make_float2(exp2_fast(d.x), exp2_fast(d.y));
        }
      }
#pragma unroll
      for (int n = N / 4; n > 0; n /= 2)         // (by halves: three additions a number at most)
#pragma unroll
        for (int e = 0; e < n; ++e) add2(w[e], w[e + n]);
      sum += w[0].x + w[0].y;
    }
    s.sum += sum;
  }
  return s;
}
template <typename T, int THREADS>
__global__ void __launch_bounds__(256, lp_blocks<T>) token_logprobs_kernel(const LogprobArgs a) {
  constexpr int ROWS = THREADS == LP_NARROW ? 8 : 1;
  const int C = ROWS > 1 ? 1 : a.split, rank = ROWS > 1 ? 0 : (int)blockIdx.x % C;
  const int r = (int)blockIdx.x / C * ROWS + (ROWS > 1 ? threadIdx.x >> 5 : 0), t = ROWS > 1 ? threadIdx.x & 31 : threadIdx.x, V = a.V;
  if (r >= a.R) return;
  const T* l = (const T*)a.logits + r * a.row;
  const float temperature = a.temperature ? a.temperature[r] : a.temperature_all;
  const bool far = temperature > LP_FAR;
  const float c = (float)(1.4426950408889634 / (double)temperature * (far ? 4.0 : 1.0));
  const int64_t token = a.tokens[r];
  const bool there = token >= 0 && token < V;
  const float mine = there ? dt<T>::ld(l, token) : 0.f;
  lp_sum<T, THREADS> s = far ? row_sum<T, THREADS, true>(l, V, t, rank, C, c) : row_sum<T, THREADS, false>(l, V, t, rank, C, c);
  s.add_lanes();
  if constexpr (ROWS == 1) {
    __shared__ lp_sum<T, THREADS> s_part[THREADS / 32];
    if ((t & 31) == 0) s_part[t >> 5] = s;
    __syncthreads();
    auto join = [&](const lp_sum<T, THREADS>* part, int n) {      // by one warp
      s = t < n ? part[t] : lp_sum<T, THREADS>{-INFINITY, 0.f, 0};
      const float top = warp_max(s.m);
      if (far) s.template under<true>(top, c);
      else s.template under<false>(top, c);
      s.add_lanes();
    };
    if (t < 32) join(s_part, THREADS / 32);
    if (C > 1) {
      __shared__ lp_sum<T, THREADS> s_all[LP_MOST];
      cg::cluster_group cluster = cg::this_cluster();
      cluster.sync();                            // (the first block has begun)
      if (t == 0) cluster.map_shared_rank(s_all, 0)[rank] = s;
      cluster.sync();
      if (rank > 0) return;
      if (t < 32) join(s_all, C);
    }
  }
  if (t == 0) {
    const bool ok = there && temperature > 0.f && temperature < INFINITY && s.m > -INFINITY;
    const double d = mine == s.m ? 0.0 : ((double)mine - (double)s.m) / (double)temperature;
    a.out[r] = ok ? (float)(d - log((double)s.ones + (double)s.sum)) : NAN;
  }
}

// A warp a row where a lane has up to eight vectors, or 20 while there are four rows an SM; else a block, and several while their blocks fit the SMs.  us, a warp / a
// block: bf16, 4000 rows of 1500 6.1 / 27, 300 of 1500 3.8 / 5.0, 2000 of 5000 8.2 / 14.9, 100 of 5000 6.4 / 3.7, 2000 of 16 000 18.1 / 16.0; fp32, 4000 of 1500 6.6 / 13.2, 1000 of
// 5000 10.1 / 7.8.  One row of 200 000 (fp32) by one block 32.8, by eight 7.7.
template <typename T>
int launch_logprobs(LogprobArgs a, cudaStream_t st) {
  const int sms = sm_count() > 0 ? sm_count() : 148;
  constexpr int N = row_vec<T>::n;
  if (a.V <= 32 * 8 * N || (a.V <= 32 * 20 * N && a.R >= 4 * sms)) {
    token_logprobs_kernel<T, LP_NARROW><<<(a.R + 7) / 8, 256, 0, st>>>(a);
  } else {
    a.split = 1;
    while (a.split < LP_MOST && (long long)2 * a.split * a.R <= lp_blocks<T> * sms && a.V > a.split * LP_WIDE * lp_batch<T> * N) a.split *= 2;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)a.R * a.split);
    cfg.blockDim = dim3(LP_WIDE);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = a.split;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = a.split > 1 ? 1 : 0;
    LL_CUDA(cudaLaunchKernelEx(&cfg, token_logprobs_kernel<T, LP_WIDE>, a));
  }
  LL_LAUNCH_OK("token_logprobs_kernel");
  return LL_OK;
}

}  // namespace
}  // namespace llb

using namespace llb;

extern "C" {

int ll_token_logprobs(const void* logits, int dtype, int R, int V, long long row, const int64_t* tokens, const float* temperature, float temperature_all, float* out,
                      ll_stream stream) {
  LL_CHECK_ARG(logits && tokens && out && R > 0 && R <= 1 << 27 && V > 0 && V <= 1 << 18, "token_logprobs: %d rows of %d logits (1 to %d)", R, V, 1 << 18);
  LL_CHECK_ARG(dtype == LL_F32 || dtype == LL_BF16 || dtype == LL_F16, "token_logprobs: type %d", dtype);
  LL_CHECK_ARG((uintptr_t)logits % (dtype == LL_F32 ? 4 : 2) == 0, "token_logprobs: logits at %p", logits);
  const LogprobArgs a{logits, row, R, V, 1, tokens, temperature, temperature_all, out};
  if (dtype == LL_F32) return launch_logprobs<float>(a, (cudaStream_t)stream);
  if (dtype == LL_BF16) return launch_logprobs<__nv_bfloat16>(a, (cudaStream_t)stream);
  return launch_logprobs<__half>(a, (cudaStream_t)stream);
}

}  // extern "C"
