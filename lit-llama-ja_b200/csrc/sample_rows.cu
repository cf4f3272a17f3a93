// A token a row of logits from a given random number: temperature, top-k, top-p and min-p (the definition: include/llb200.h).
//
// Weights are whole numbers, w = rint(2^44 exp((l - m) / T)): V of them have a sum of 62 bits, exactly, so that neither a border of top-p nor a draw depends on
// the order of sums, and blocks may add in any order.  Both borders are values: top-k's the largest x with k logits at or above it, top-p's the largest x with
// top_p of the kept weight there.  A border is found by counts (or weights) in 1024 equal steps below m down to where weights are 0, then by those of
// the numbers' keys within the step that it falls into: once for 16-bit logits, up to three times for 32.
//
// A cluster of blocks has a row in its shared memory, read once.
#include <cooperative_groups.h>

#include "row_values.cuh"

namespace llb {
namespace {

namespace cg = cooperative_groups;

constexpr double SR_ONE = 17592186044416.0;      // 2^44
constexpr float SR_REACH = 31.25f;               // weights are 0 from 45 ln 2 = 31.19 temperatures below m on
constexpr int SR_BINS = 1024;
constexpr int SR_WIDE = 512, SR_NARROW = 128, SR_MOST = 8, SR_TURNS = 17;      // threads; blocks a row and vectors a thread, at most
typedef unsigned long long u64;

// Numbers in the order of their values, as whole numbers one after the other in their type; 0 and -0 are one.
__device__ __forceinline__ uint32_t order_bits(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
template <typename T> struct key_shift { static constexpr int n = 0; };
template <> struct key_shift<__nv_bfloat16> { static constexpr int n = 16; };
template <> struct key_shift<__half> { static constexpr int n = 13; };
template <typename T> __device__ __forceinline__ uint32_t order_key(float x) { return order_bits(x) >> key_shift<T>::n; }
template <typename T> __device__ __forceinline__ float key_value(uint32_t k) {
  k <<= key_shift<T>::n;
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~(k | ((1u << key_shift<T>::n) - 1u)));
}

struct SampleArgs {
  const void* logits;
  long long row;
  int V, turns;                                  // turns: vectors of a thread
  const float *u, *temperature, *top_p, *min_p;
  const int32_t* top_k;
  float temperature_all, top_p_all, min_p_all;
  int top_k_all;
  int64_t* tokens;
};

template <int THREADS>
struct SampleShared {
  uint32_t hist[2][2][SR_BINS];                  // two in turn: low and high halves of sums
  u64 scan[THREADS / 32], found_base, totals[SR_MOST], segment[SR_TURNS][THREADS / 32];
  uint32_t key[SR_MOST], warp_key[THREADS / 32], range[2];
  int found;
};

// Sum over the threads before this one.  Every thread of the block calls.
template <int THREADS>
__device__ __forceinline__ u64 threads_before(u64 v, u64* s) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  u64 incl = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 n = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += n;
  }
  if (lane == 31) s[warp] = incl;
  __syncthreads();
  u64 before = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) before += w < warp ? s[w] : 0;
  return before + incl - v;
}

template <typename T, int THREADS>
__global__ void __launch_bounds__(THREADS) sample_rows_kernel(const SampleArgs a) {
  constexpr int N = row_vec<T>::n, WARPS = THREADS / 32, BINS = SR_BINS / THREADS;
  __shared__ SampleShared<THREADS> sh;
  cg::cluster_group cluster = cg::this_cluster();
  cluster.barrier_arrive();                      // (other blocks' memory is touched when all of them have begun)
  const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int r = blockIdx.x / C, t = threadIdx.x, lane = t & 31, warp = t >> 5, V = a.V;
  const T* l = (const T*)a.logits + r * a.row;
  const float u = a.u[r], temperature = a.temperature ? a.temperature[r] : a.temperature_all, top_p = a.top_p ? a.top_p[r] : a.top_p_all,
              min_p = a.min_p ? a.min_p[r] : a.min_p_all;
  const int top_k = a.top_k ? a.top_k[r] : a.top_k_all;
  const int i0 = rank * a.turns * THREADS * N - row_offset(l);      // the block's first number

  // ---- the row, and its largest logit
  extern __shared__ uint4 s_row[];               // [turns][THREADS]: a thread's own vectors
  float top = -INFINITY;
  bool bad = !(u >= 0.f && u <= 1.f) || !(temperature >= 0.f && temperature < INFINITY) || isnan(top_p) || isnan(min_p);
#pragma unroll 4
  for (int j = 0; j < a.turns; ++j) {
    const uint4 raw = load_vector(l, i0 + (j * THREADS + t) * N, V);
    s_row[j * THREADS + t] = raw;
    float x[N];
    vec_values<T>(raw, x);
#pragma unroll
    for (int e = 0; e < N; ++e) {
      bad |= isnan(x[e]);
      top = fmaxf(top, x[e]);
    }
  }
  for (int b = t; b < 2 * 2 * SR_BINS; b += THREADS) (&sh.hist[0][0][0])[b] = 0;
  {
    const uint32_t k = __reduce_max_sync(0xffffffffu, order_bits(top));
    const bool any = __any_sync(0xffffffffu, bad);
    if (lane == 0) sh.warp_key[warp] = any ? 0xffffffffu : k;      // (the key of a number that is none: above all others)
    __syncthreads();
    cluster.barrier_wait();
    if (warp == 0) {
      const uint32_t all = __reduce_max_sync(0xffffffffu, lane < WARPS ? sh.warp_key[lane] : 0u);
      if (lane < C) cluster.map_shared_rank(sh.key, lane)[rank] = all;
    }
    cluster.sync();
  }
  uint32_t top_bits = 0;
  for (int c = 0; c < C; ++c) top_bits = max(top_bits, sh.key[c]);
  if (top_bits == 0xffffffffu || top_bits <= order_bits(-INFINITY)) {      // (the same in all blocks)
    if (rank == 0 && t == 0) a.tokens[r] = -1;
    return;
  }
  const float m = __uint_as_float(top_bits & 0x80000000u ? top_bits & 0x7fffffffu : ~top_bits);
  const uint32_t top_key = top_bits >> key_shift<T>::n;

  // ---- weights, and steps below m
  const double inv = 1.0 / (double)temperature;
  const float per_step = temperature > 0.f ? (float)SR_BINS / (SR_REACH * temperature) : INFINITY;
  // how many steps below m; SR_BINS and more: a weight of 0.  (A temperature so large that a step has no size: one step for all.)
  auto below = [&](float v) -> float { return v == m ? 0.f : v == -INFINITY ? (float)SR_BINS : per_step == 0.f ? 0.f : (m - v) * per_step; };
  auto weight = [&](float v) -> u64 { return v == m ? (u64)SR_ONE : (u64)(long long)rint(exp(((double)v - (double)m) * inv) * SR_ONE); };
  uint32_t border = 0;                           // kept are keys from here on

  // ---- the largest key at or above which counts or weights reach what they have to
  int turn = 0;
  auto select = [&](auto weigh, auto reached) {
    constexpr bool WEIGHTS = decltype(weigh)::value;
    uint32_t lo = 0, hi = 0;
    int shift = -1;                              // -1: steps below m; else steps of 2^shift keys below hi
    u64 base = 0;
    while (true) {
      uint32_t(*hist)[SR_BINS] = sh.hist[turn];
#pragma unroll 1
      for (int j = 0; j < a.turns; ++j) {
        float x[N];
        vec_values<T>(s_row[j * THREADS + t], x);
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const float v = x[e];
          const uint32_t key = order_key<T>(v);
          int bin;
          if (shift < 0) {
            const float s = below(v);
            bin = s < (float)SR_BINS ? (int)s : SR_BINS;
          } else {
            bin = key >= lo && key <= hi ? (int)((hi - key) >> shift) : SR_BINS;
          }
          if (bin < SR_BINS && key >= border) {
            if (WEIGHTS) {
              const u64 w = weight(v);
              const uint32_t part = (uint32_t)w, old = atomicAdd(&hist[0][bin], part), up = (uint32_t)(w >> 32) + (old + part < old ? 1u : 0u);
              if (up != 0u) atomicAdd(&hist[1][bin], up);
            } else {
              atomicAdd(&hist[0][bin], 1u);
            }
          }
        }
      }
      cluster.sync();
      // every block adds up all blocks' and finds the step
      u64 n[BINS], mine = 0;
#pragma unroll
      for (int b = 0; b < BINS; ++b) n[b] = 0;
      for (int c = 0; c < C; ++c) {
        const uint32_t* h = cluster.map_shared_rank(&hist[0][0], c);
#pragma unroll
        for (int b = 0; b < BINS; ++b) n[b] += (WEIGHTS ? (u64)h[SR_BINS + BINS * t + b] << 32 : 0) + h[BINS * t + b];
      }
#pragma unroll
      for (int b = 0; b < BINS; ++b) mine += n[b];
      if (t == 0) sh.found = -1;
      const u64 before = threads_before<THREADS>(mine, sh.scan);
      u64 all = 0;
#pragma unroll
      for (int w = 0; w < WARPS; ++w) all += sh.scan[w];
      u64 at = base + before;
#pragma unroll
      for (int b = 0; b < BINS; ++b) {
        if (!reached(at, all, shift) && reached(at + n[b], all, shift)) sh.found = BINS * t + b, sh.found_base = at;
        at += n[b];
      }
      // (the sums of the turn before have been read by every block: behind a barrier of the cluster that comes after)
      for (int b = t; b < 2 * SR_BINS; b += THREADS) (&sh.hist[turn ^ 1][0][0])[b] = 0;
      turn ^= 1;
      __syncthreads();
      const int found = sh.found;
      if (found < 0) return;                     // (fewer than k within reach: all of them are kept)
      base = sh.found_base;
      if (shift < 0) {
        // the keys of the step: the smallest one at most so many steps below m, by 32 at a time
        if (warp < 2) {
          const int most = found - warp;
          uint32_t from = order_key<T>(-INFINITY), to = top_key;       // above: `from` is more than `most` steps below m, `to` is not
          while (most >= 0 && to - from > 1u) {
            const uint32_t step = max(1u, (uint32_t)(((u64)(to - from) + 32) / 33));
            const u64 probe = min((u64)from + (u64)(lane + 1) * step, (u64)to);
            const float s = below(key_value<T>((uint32_t)probe));
            const uint32_t in = __ballot_sync(0xffffffffu, s < (float)SR_BINS && (int)s <= most);
            const int first = __ffs(in) - 1;     // (lane 31's is `to`, or the search goes on above it)
            const uint32_t next_to = first < 0 ? to : (uint32_t)min((u64)from + (u64)(first + 1) * step, (u64)to);
            from = first < 0 ? (uint32_t)min((u64)from + 32ull * step, (u64)to) : (uint32_t)((u64)from + (u64)first * step);
            to = next_to;
          }
          if (lane == 0) sh.range[warp] = most < 0 ? top_key : warp == 0 ? to : to - 1u;
        }
        __syncthreads();
        lo = sh.range[0], hi = sh.range[1];
      } else {
        hi -= (uint32_t)found << shift;
        if (hi - lo >= 1u << shift) lo = hi - ((1u << shift) - 1u);
      }
      if (lo == hi) {
        border = hi;
        return;
      }
      shift = 0;
      while (((hi - lo) >> shift) >= (uint32_t)SR_BINS) ++shift;
    }
  };
  if (top_k >= 1 && top_k < V) select(std::false_type(), [&](u64 n, u64, int) { return n >= (u64)top_k; });
  if (top_p < 1.f) {
    double want = 0.0;
    select(std::true_type(), [&](u64 n, u64 all, int shift) {
      if (shift < 0) want = (double)top_p * (double)all;
      return n > 0 && (double)n >= want;
    });
  }

  // ---- kept weights by runs of a warp's numbers, which follow one another in the row
  const double least = fmin((double)min_p, 1.0) * SR_ONE;
  // (beyond so many steps min-p keeps nothing; a step more than that comes to, for the roundings)
  const float reach = min_p > 0.f ? fminf((float)SR_BINS, -logf(fminf(min_p, 1.f)) * ((float)SR_BINS / SR_REACH) + 1.f) : (float)SR_BINS;
  auto kept = [&](float v) -> u64 {
    if (order_key<T>(v) < border || !(below(v) < reach)) return 0;
    const u64 w = weight(v);
    return (double)w >= least ? w : 0;
  };
  u64 total = 0;
#pragma unroll 1
  for (int j = 0; j < a.turns; ++j) {
    float x[N];
    vec_values<T>(s_row[j * THREADS + t], x);
    u64 n = 0;
#pragma unroll
    for (int e = 0; e < N; ++e) n += kept(x[e]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
    if (lane == 0) sh.segment[j][warp] = n;
  }
  __syncthreads();
  if (warp == 0) {
    for (int s = lane; s < a.turns * WARPS; s += 32) total += (&sh.segment[0][0])[s];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    if (lane < C) cluster.map_shared_rank(sh.totals, lane)[rank] = total;
  }
  cluster.sync();
  u64 before = 0;
  total = 0;
  for (int c = 0; c < C; ++c) {
    if (c == rank) before = total;
    total += sh.totals[c];
  }
  const u64 target = temperature == 0.f ? 0 : min((u64)floor((double)u * (double)total), total - 1);
  if (target < before || target >= before + sh.totals[rank]) return;
  // the run that the target falls into (every warp looks for itself), and the number in it
  int run = -1;
  for (int s0 = 0; s0 < a.turns * WARPS && run < 0; s0 += 32) {
    const u64 n = s0 + lane < a.turns * WARPS ? (&sh.segment[0][0])[s0 + lane] : 0;
    u64 incl = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const u64 v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    const uint32_t past = __ballot_sync(0xffffffffu, before + incl > target);
    if (past != 0u) {
      run = s0 + __ffs(past) - 1;
      before += __shfl_sync(0xffffffffu, incl - n, __ffs(past) - 1);
    } else {
      before += __shfl_sync(0xffffffffu, incl, 31);
    }
  }
  if (run < 0 || run % WARPS != warp) return;
  const int j = run / WARPS;
  float x[N];
  vec_values<T>(s_row[j * THREADS + t], x);
  u64 w[N], n = 0;
#pragma unroll
  for (int e = 0; e < N; ++e) w[e] = kept(x[e]), n += w[e];
  u64 incl = n;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  u64 at = before + incl - n;
  if (at <= target && target < at + n) {
    int e0 = 0;
#pragma unroll
    for (int e = 0; e < N; ++e) {
      at += w[e];
      if (at <= target) e0 = e + 1;
    }
    a.tokens[r] = i0 + (j * THREADS + t) * N + e0;
  }
}

// Blocks a row: enough that a thread has at most 32 numbers, and more of them while there are few rows.
template <typename T, int THREADS>
int launch_sample(SampleArgs a, int R, int C, cudaStream_t st) {
  constexpr int N = row_vec<T>::n;
  a.turns = (a.V + N - 1 + C * THREADS * N - 1) / (C * THREADS * N);      // (a row may begin between two boundaries)
  static_assert(SR_TURNS * SR_MOST * SR_WIDE * 4 >= (1 << 18) + 3, "rows of 2^18 numbers");
  static PerDevice set;
  if (!set) {
    LL_CUDA(cudaFuncSetAttribute(sample_rows_kernel<T, THREADS>, cudaFuncAttributeMaxDynamicSharedMemorySize, SR_TURNS * THREADS * 16));
    prefer_max_smem(sample_rows_kernel<T, THREADS>);
    set.mark();
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(R * C);
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = a.turns * THREADS * 16;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = C;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  LL_CUDA(cudaLaunchKernelEx(&cfg, sample_rows_kernel<T, THREADS>, a));
  LL_LAUNCH_OK("sample_rows_kernel");
  return LL_OK;
}
template <typename T>
int sample_rows(const SampleArgs& a, int R, cudaStream_t st) {
  if (a.V <= SR_NARROW * 8) return launch_sample<T, SR_NARROW>(a, R, 1, st);
  int C = 1;
  while (C < SR_MOST && a.V > C * SR_WIDE * 32) C *= 2;
  while (C < SR_MOST && C * R <= (sm_count() > 0 ? sm_count() : 148) && a.V > 2 * C * SR_WIDE * 4) C *= 2;
  return launch_sample<T, SR_WIDE>(a, R, C, st);
}

}  // namespace
}  // namespace llb

using namespace llb;

extern "C" {

int ll_sample_rows(const void* logits, int dtype, int R, int V, long long row, const float* u, const float* temperature, float temperature_all, const int32_t* top_k,
                   int top_k_all, const float* top_p, float top_p_all, const float* min_p, float min_p_all, int64_t* tokens, ll_stream stream) {
  LL_CHECK_ARG(logits && u && tokens && R > 0 && R <= 1 << 27 && V > 0 && V <= 1 << 18, "sample_rows: %d rows of %d logits (1 to %d)", R, V, 1 << 18);
  LL_CHECK_ARG(dtype == LL_F32 || dtype == LL_BF16 || dtype == LL_F16, "sample_rows: type %d", dtype);
  LL_CHECK_ARG((uintptr_t)logits % (dtype == LL_F32 ? 4 : 2) == 0, "sample_rows: logits at %p", logits);
  const SampleArgs a{logits, row, V, 0, u, temperature, top_p, min_p, top_k, temperature_all, top_p_all, min_p_all, top_k_all, tokens};
  if (dtype == LL_F32) return sample_rows<float>(a, R, (cudaStream_t)stream);
  if (dtype == LL_BF16) return sample_rows<__nv_bfloat16>(a, R, (cudaStream_t)stream);
  return sample_rows<__half>(a, R, (cudaStream_t)stream);
}

}  // extern "C"
