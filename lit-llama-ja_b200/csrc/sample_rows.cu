// A token a row of logits from a given random number: temperature, top-k, top-p and min-p (the definition: include/llb200.h).
//
// Weights are whole numbers, w = rint(2^44 exp((l - m) / T)): V of them have a sum of 62 bits, exactly, so that neither a border of top-p nor a draw depends on
// the order of sums, and blocks may add in any order.  Both borders are values: top-k's the largest x with k logits at or above it, top-p's the largest x with
// top_p of the kept weight there.
//   top-k: counts in 1024 equal steps below m, down to where weights are 0.
//   top-p: the steps' weights, in the same pass that adds up all of them: within a step they differ by 3 %, so that 13 bits of each one's part of the step's largest
//   are enough to leave one step or two that the border can be in.
// The few numbers of those steps are then compared with one another, on top of the exact sum of what lies above; where they are many (rows of few values), the border is
// found by counts or exact weights of their keys, 1024 ranges at a time.
//
// What bounds it: 301 rows of 100 003 (fp32) under top-p and min-p 250 us, under top-p alone 310, 125 without a border (copying them takes 18): instructions (half of the issue slots)
// and the barriers of a cluster, 1 to 1.5 us each, between phases of 3 to 6 us of exponentials (ten instructions of 64 bits each), two blocks an SM.  One row of 32 000 (bf16): 5.2 us,
// 7.9 under top-k, 14 under top-p.  On the way (us, 301 rows, top-p and min-p): a block a row and bisection 3334; exact weights in all steps, two dependent additions of 32 bits in shared
// memory each, 738; steps' weights in parts, and a list of the border's numbers by remote atomics 639, by one's own 435; the exponential by a table, one block that
// finishes alone and sums by lanes 325; top-p's border not looked for where min-p's is above it 253; a number's step by one
// product 250.
//
// A cluster of blocks has a row in its shared memory, read once.
#include <cooperative_groups.h>

#include "row_values.cuh"

namespace llb {
namespace {

namespace cg = cooperative_groups;

constexpr double SR_ONE = 17592186044416.0;      // 2^44
constexpr double SR_PER = 256 * 1.4426950408889634;      // 256 / ln 2
constexpr float SR_REACH = 31.25f;               // weights are 0 from 45 ln 2 = 31.19 temperatures below m on
constexpr float SR_STEP0 = 8388608.f;            // 2^23
constexpr float SR_LEAST = 7.888609052210118e-31f;      // 2^-100: less of a temperature counts as 0
constexpr int SR_BINS = 1024, SR_LIST = 512, SR_TABLE = 256;
constexpr int SR_WIDE = 512, SR_NARROW = 128, SR_MOST = 8, SR_TURNS = 17;      // threads; blocks a row and vectors a thread, at most
typedef unsigned long long u64;

// Numbers in the order of their values, as whole numbers in the steps of their type; 0 and -0 are one.
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

// rint(2^44 exp(d / T)) for d <= 0, with c = SR_PER / T: by a table of 2^(j / 256) and a polynomial of degree 4 around its places (Tang, Table-driven
// implementation of the exponential function, 1989): at most half of ln 2 / 256 from one, so that the next term is under 2^-54 of a weight.  Before it is rounded a weight is off by
// less than 2^-6 of a whole one: by 2^-52 of |d / T| of itself with c (x exp(-x) is 0.37 at most), 2^-52 with the table and 2^-53 with the last product.  So one in some thousand weights is the
// whole number beside the nearest one.
__device__ __forceinline__ u64 weight_of(double d, double c, const double* table) {
  constexpr double SHIFT = 6755399441055744.0;   // 1.5 2^52: the sum's last bits are the nearest whole number
  constexpr double L = 0.0027076061740622863;    // ln 2 / 256
  const double shifted = fma(d, c, SHIFT);
  const int k = __double2loint(shifted);
  const double r = fma(d, c, SHIFT - shifted);
  const double p = r * fma(r, fma(r, fma(r, L * L * L * L / 24, L * L * L / 6), L * L / 2), L);
  const double at = table[k & (SR_TABLE - 1)], y = fma(at, p, at);
  const double scaled = __hiloint2double(__double2hiint(y) + ((k >> 8) << 20) + (44 << 20), __double2loint(y));
  return (u64)__double_as_longlong(scaled + 4503599627370496.0) & 0xfffffffffffffull;      // 2^52
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
  alignas(16) uint32_t hist[2][2][SR_BINS];      // two in turn: low and high halves of sums; or a block's list of numbers that a border is among
  double exps[SR_TABLE];                         // 2^(j / 256)
  alignas(16) u64 list_weight[SR_LIST];          // all blocks' lists
  alignas(16) uint32_t list_key[SR_LIST];
  u64 scan[THREADS / 32], found_base, sums[2][SR_MOST], kept[SR_MOST];
  uint32_t key[SR_MOST], warp_key[THREADS / 32], range[2], listed[2], least_key;
  int found, last;
};
static_assert(SR_LIST * 16 <= 2 * SR_BINS * 4, "a list in the place of counts");

// Another block's shared memory, asked for by its place in this one's.
__device__ __forceinline__ uint32_t there(const void* p, int rank) {
  uint32_t at;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(p)), "r"(rank));
  return at;
}
__device__ __forceinline__ uint32_t remote(uint32_t at) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
  return v;
}
template <int BINS>
__device__ __forceinline__ void remote_bins(uint32_t (&h)[BINS], uint32_t at) {
  if constexpr (BINS == 2) {
    asm volatile("ld.shared::cluster.v2.u32 {%0, %1}, [%2];" : "=r"(h[0]), "=r"(h[1]) : "r"(at) : "memory");
  } else {
#pragma unroll
    for (int b = 0; b < BINS; ++b) h[b] = remote(at + 4 * b);
  }
}

// Of the warps' sums those before this warp's, and all.
template <int WARPS>
__device__ __forceinline__ u64 warps_before(const u64* s, u64& all) {
  const int lane = threadIdx.x & 31;
  const u64 x = lane < WARPS ? s[lane] : 0;
  u64 incl = x;
#pragma unroll
  for (int o = 1; o < WARPS; o <<= 1) {
    const u64 n = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += n;
  }
  all = __shfl_sync(0xffffffffu, incl, WARPS - 1);
  return __shfl_sync(0xffffffffu, incl - x, threadIdx.x >> 5);
}
// Sum over the threads before this one, and over all.  Every thread of the block calls.
template <int THREADS>
__device__ __forceinline__ u64 threads_before(u64 v, u64* s, u64& all) {
  const int lane = threadIdx.x & 31;
  u64 incl = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 n = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += n;
  }
  if (lane == 31) s[threadIdx.x >> 5] = incl;
  __syncthreads();
  return warps_before<THREADS / 32>(s, all) + incl - v;
}

template <typename T, int THREADS>
__global__ void __launch_bounds__(THREADS, THREADS == SR_WIDE ? 2 : 8) sample_rows_kernel(const SampleArgs a) {
  constexpr int N = row_vec<T>::n, WARPS = THREADS / 32, BINS = SR_BINS / THREADS, MOST = THREADS == SR_WIDE ? SR_MOST : 1;
  __shared__ SampleShared<THREADS> sh;
  cg::cluster_group cluster = cg::this_cluster();
  cluster.barrier_arrive();                      // (other blocks' memory is touched when all of them have begun)
  const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int r = blockIdx.x / C, t = threadIdx.x, lane = t & 31, warp = t >> 5, V = a.V;
  const T* l = (const T*)a.logits + r * a.row;
  const float u = a.u[r];
  float temperature = a.temperature ? a.temperature[r] : a.temperature_all, top_p = a.top_p ? a.top_p[r] : a.top_p_all, min_p = a.min_p ? a.min_p[r] : a.min_p_all;
  int top_k = a.top_k ? a.top_k[r] : a.top_k_all;
  bool bad = !(u >= 0.f && u <= 1.f) || !(temperature >= 0.f && temperature < INFINITY) || isnan(top_p) || isnan(min_p);
  top_p = fmaxf(top_p, 0.f);
  const bool first = temperature < SR_LEAST;     // the first one of the largest
  if (first) temperature = 1.f, top_k = 1, top_p = 1.f, min_p = 0.f;

  // ---- the row, a run of it a warp, and its largest logit
  extern __shared__ uint4 s_row[];
  uint4* const mine = s_row + warp * a.turns * 32 + lane;      // the thread's vectors, 32 apart
  const int i0 = (rank * THREADS + warp * 32) * a.turns * N + lane * N - row_offset(l);      // the first one's first number
  float top = -INFINITY;
#pragma unroll 4
  for (int j = 0; j < a.turns; ++j) {
    const uint4 raw = load_vector(l, i0 + j * 32 * N, V);
    mine[j * 32] = raw;
    float x[N];
    vec_values<T>(raw, x);
#pragma unroll
    for (int e = 0; e < N; ++e) asm("max.NaN.f32 %0, %0, %1;" : "+f"(top) : "f"(x[e]));
  }
  bad |= isnan(top);
  if ((top_k >= 1 && top_k < V) || top_p < 1.f)      // (the first turn's counts; what comes after them is set to none on the way)
    for (int b = t; b < SR_BINS; b += THREADS) sh.hist[0][0][b] = 0;
  for (int b = t; b < SR_TABLE; b += THREADS) sh.exps[b] = exp2(b * (1.0 / SR_TABLE));
  if (t < 2) sh.listed[t] = 0;
  {
    const uint32_t k = __reduce_max_sync(0xffffffffu, order_bits(top));
    const bool any = __any_sync(0xffffffffu, bad);
    if (lane == 0) sh.warp_key[warp] = any ? 0xffffffffu : k;      // (above all others)
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
  float m = __uint_as_float(top_bits & 0x80000000u ? top_bits & 0x7fffffffu : ~top_bits);
  if (m == INFINITY) {                           // the limit: these alone, all alike
    m = 0.f;
    for (int j = 0; j < a.turns; ++j) {
      float x[N];
      vec_values<T>(mine[j * 32], x);
      T* to = reinterpret_cast<T*>(&mine[j * 32]);
#pragma unroll
      for (int e = 0; e < N; ++e) dt<T>::st(to, e, x[e] == INFINITY ? 0.f : -INFINITY);
    }
  }

  // ---- steps below m, and weights
  const double c64 = SR_PER / (double)temperature, m64 = m;
  const float half_m = 0.5f * m, per_half = 2.f * (SR_BINS / SR_REACH) / temperature;      // (by halves: m - v may be more than a float holds)
  const float cut = fmaxf(m - 31.5f * temperature, -3.402823466e38f);      // weights are 0 from here on; -inf is below
  auto below = [&](float v) { return __fmaf_rn(v, -0.5f, half_m); };
  // SR_STEP0 and the step that is nearest (a float past 2^23 has no fraction): one rounding of the same product wherever a number's step is asked for, which the compiler may not put together
  // in another way (with a product rounded by itself in one place and not in another, a number between two steps was counted in one and looked for in the other).  It rises as v falls.  Of numbers
  // above `cut` those of SR_BINS steps and more weigh nothing.
  auto step_at = [&](float v) { return __fmaf_rn(below(v), per_half, SR_STEP0); };
  auto step_of = [&](float at) { return __float_as_int(at) & 0x7fffff; };
  auto weight = [&](float v) { return weight_of((double)v - m64, c64, sh.exps); };      // (of numbers from `cut` on)
  float lowest = cut;                            // kept are numbers from here on
  int turn = 0, sums = 0;
  // the thread's vectors that have a number from `from` on in their warp
  auto each = [&](float from, auto visit) {
#pragma unroll 1
    for (int j = 0; j < a.turns; ++j) {
      float x[N];
      vec_values<T>(mine[j * 32], x);
      float most = x[0];
#pragma unroll
      for (int e = 1; e < N; ++e) most = fmaxf(most, x[e]);
      if (__any_sync(0xffffffffu, most >= from)) visit(x, j);
    }
  };
  // a sum of all blocks' threads' numbers, behind a barrier of the cluster; `before`: of the blocks before this one
  auto cluster_sum = [&](u64 v, u64& before) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (lane == 0) sh.scan[warp] = v;
    __syncthreads();
    if (warp == 0) {
      u64 all;
      warps_before<WARPS>(sh.scan, all);
      if (lane < C) cluster.map_shared_rank(&sh.sums[sums][0], lane)[rank] = all;
    }
    cluster.sync();
    v = 0;
    for (int c = 0; c < C; ++c) {
      if (c == rank) before = v;
      v += sh.sums[sums][c];
    }
    sums ^= 1;                                   // (read before the next barrier, and written again behind that)
    return v;
  };
  // This turn's counts of all blocks, behind a barrier of the cluster: the thread's bins, which are neighbours.
  auto counted = [&](bool high, u64 (&n)[BINS]) {
#pragma unroll
    for (int b = 0; b < BINS; ++b) n[b] = 0;
    for (int part = 0; part < (high ? 2 : 1); ++part) {
      uint32_t h[MOST][BINS];
#pragma unroll
      for (int c = 0; c < MOST; ++c)
        if (c < C) remote_bins(h[c], there(&sh.hist[turn][part][BINS * t], c));
#pragma unroll
      for (int c = 0; c < MOST; ++c)
        if (c < C)
#pragma unroll
          for (int b = 0; b < BINS; ++b) n[b] += (u64)h[c][b] << (32 * part);
    }
    if (t == 0) sh.found = -1, sh.last = SR_BINS - 1, sh.range[0] = sh.range[1] = 0;
    // (what the turn before has left has been read by every block: behind a barrier of the cluster that comes after)
    for (int b = t; b < 2 * SR_BINS; b += THREADS) (&sh.hist[turn ^ 1][0][0])[b] = 0;
    turn ^= 1;
  };
  auto bins_before = [&](const u64 (&n)[BINS]) {
    u64 all = 0;
#pragma unroll
    for (int b = 0; b < BINS; ++b) all += n[b];
    u64 total;
    return threads_before<THREADS>(all, sh.scan, total);
  };
  // The keys of the steps first_bin .. last_bin below m: the smallest key at most so many steps below, by 32 at a time.
  auto keys_of = [&](int first_bin, int last_bin) {
    if (warp < 2) {
      const int most = warp == 0 ? last_bin : first_bin - 1;
      const uint32_t top_key = order_key<T>(m);
      uint32_t from = order_key<T>(-INFINITY), to = top_key;             // `from` is more than `most` steps below m, `to` is not
      while (most >= 0 && to - from > 1u) {
        const uint32_t step = (to - from - 1u) / 33u + 1u;
        const u64 probe = min((u64)from + (u64)(lane + 1) * step, (u64)to);
        const uint32_t in = __ballot_sync(0xffffffffu, step_at(key_value<T>((uint32_t)probe)) <= SR_STEP0 + most);
        const int at = in != 0u ? __ffs(in) - 1 : 32;
        const u64 above = (u64)from + (u64)at * step;
        if (in != 0u) to = (uint32_t)min(above + step, (u64)to);
        from = (uint32_t)above;
      }
      if (lane == 0) sh.range[warp] = most < 0 ? top_key : warp == 0 ? to : to - 1u;
    }
    __syncthreads();
  };
  // (a sum of 64 bits by halves: the one that makes the lower one run over adds to the upper one)
  auto add_weight = [](uint32_t(*hist)[SR_BINS], uint32_t bin, u64 w) {
    const uint32_t part = (uint32_t)w, old = atomicAdd(&hist[0][bin], part), up = (uint32_t)(w >> 32) + (old + part < old ? 1u : 0u);
    if (up != 0u) atomicAdd(&hist[1][bin], up);
  };
  // The largest key of lo .. hi at or above which the counts (or weights) reach what they have to.  Counts of what lies above hi are known (`base`), weights are added up.
  auto by_keys = [&](auto weights, uint32_t lo, uint32_t hi, u64 base, auto reached) {
    constexpr bool WEIGHTS = decltype(weights)::value;
    const float least = fmaxf(key_value<T>(lo), lowest), most = key_value<T>(hi);
    for (bool begin = true;; begin = false) {
      int shift = 0;
      while (((hi - lo) >> shift) >= (uint32_t)SR_BINS) ++shift;
      uint32_t(*hist)[SR_BINS] = sh.hist[turn];
      u64 above = 0, none;
      each(least, [&](const float (&x)[N], int) {
#pragma unroll
        for (int e = 0; e < N; ++e) {
          if (x[e] < least) continue;
          if (x[e] > most) {
            if (WEIGHTS && begin) above += weight(x[e]);
            continue;
          }
          const uint32_t key = order_key<T>(x[e]);
          if (key < lo || key > hi) continue;
          const uint32_t bin = (hi - key) >> shift;
          if (WEIGHTS) {
            add_weight(hist, bin, weight(x[e]));
          } else {
            atomicAdd(&hist[0][bin], 1u);
          }
        }
      });
      if (WEIGHTS && begin) base = cluster_sum(above, none);
      else cluster.sync();
      u64 n[BINS];
      counted(WEIGHTS, n);
      u64 at = base + bins_before(n);
#pragma unroll
      for (int b = 0; b < BINS; ++b) {
        if (!reached(at) && reached(at + n[b])) sh.found = BINS * t + b, sh.found_base = at;
        at += n[b];
      }
      __syncthreads();
      const int found = sh.found;
      if (found < 0) return lo;                  // (there is one: a border is not looked for where it cannot be)
      base = sh.found_base;
      hi -= (uint32_t)found << shift;
      if (hi - lo >= 1u << shift) lo = hi - ((1u << shift) - 1u);
      if (lo == hi) return hi;
    }
  };
  // The same where SR_LIST numbers at most have keys lo .. hi: every block compares all of them.
  int listed = 0;
  u64 warp_above = 0;                            // of the warp's numbers what lies above hi
  auto by_list = [&](auto weights, uint32_t lo, uint32_t hi, u64 base, auto reached, int which) {
    constexpr bool WEIGHTS = decltype(weights)::value;
    const float least = fmaxf(key_value<T>(lo), lowest), most = key_value<T>(hi);
    u64* const weight_here = reinterpret_cast<u64*>(&sh.hist[turn][0][0]);      // (zeros that nobody reads)
    uint32_t* const key_here = reinterpret_cast<uint32_t*>(weight_here + SR_LIST);
    uint32_t* const warp_here = key_here + SR_LIST;
    u64 above = 0, none;
    each(least, [&](const float (&x)[N], int) {
#pragma unroll
      for (int e = 0; e < N; ++e) {
        if (x[e] < least || (!WEIGHTS && x[e] > most)) continue;
        const u64 w = WEIGHTS ? weight(x[e]) : 1;
        if (x[e] > most) {
          above += w;
        } else {
          const uint32_t at = atomicAdd(&sh.listed[which], 1u);
          if (at < SR_LIST) key_here[at] = order_key<T>(x[e]), weight_here[at] = w, warp_here[at] = warp;
        }
      }
    });
    if (WEIGHTS) base = cluster_sum(above, none), warp_above = sh.scan[warp];
    else cluster.sync();
    // all lists one after the other, a warp or some a block's
    if (t < C) sh.key[t] = min(remote(there(&sh.listed[which], t)), (uint32_t)SR_LIST);
    // (the counts before have been read by every block; the list, until the next barrier, by others)
    uint32_t(*hist)[SR_BINS] = sh.hist[turn ^ 1];
    for (int b = t; b < 2 * SR_BINS; b += THREADS) hist[0][b] = 0;
    turn ^= 1;
    __syncthreads();
    int n = 0;
    for (int c = 0; c < C; ++c) {
      const int of_c = min((int)sh.key[c], SR_LIST - n);
      if (warp % C == c)
        for (int i = lane + 32 * (warp / C); i < of_c; i += 32 * (WARPS / C)) {
          const uint32_t w = there(weight_here + i, c);
          sh.list_weight[n + i] = (u64)remote(w + 4) << 32 | remote(w);
          sh.list_key[n + i] = remote(there(key_here + i, c));
        }
      n += of_c;
    }
    __syncthreads();
    if (WEIGHTS) cluster.barrier_arrive();       // (the lists have been read; the wait stands where the kept weights are added up)
    listed = n;
    while (lo < hi) {
      int shift = 0;
      while (((hi - lo) >> shift) >= (uint32_t)SR_BINS) ++shift;
      for (int i = t; i < n; i += THREADS)
        if (const uint32_t key = sh.list_key[i]; key >= lo && key <= hi) add_weight(hist, (hi - key) >> shift, sh.list_weight[i]);
      if (t == 0) sh.found = -1;
      __syncthreads();
      u64 here[BINS];
#pragma unroll
      for (int b = 0; b < BINS; ++b) {
        uint32_t* h = &hist[0][BINS * t + b];
        here[b] = (u64)h[SR_BINS] << 32 | h[0];
        h[0] = h[SR_BINS] = 0;
      }
      u64 at = base + bins_before(here);
#pragma unroll
      for (int b = 0; b < BINS; ++b) {
        if (!reached(at) && reached(at + here[b])) sh.found = BINS * t + b, sh.found_base = at;
        at += here[b];
      }
      __syncthreads();
      const int found = sh.found;
      if (found < 0) break;                      // (there is one: a border is not looked for where it cannot be)
      base = sh.found_base;
      hi -= (uint32_t)found << shift;
      if (hi - lo >= 1u << shift) lo = hi - ((1u << shift) - 1u);
      __syncthreads();
    }
    return lo;
  };

  // ---- Where few numbers can be kept, the first block finishes alone: those up to `last` steps below m, in the order of the row, HERE at most.  `want`: the weight that top-p
  // has to reach, or less than 0: `top_p` of the weight that top-k leaves.  It compares all of them with one another, and no other barrier of the cluster follows.
  // us with it / without, top-k 50 and top-k 200 with top-p 0.9: 301 rows of 100 003 (fp32) 154 / 179 and 172 / 292, 16 rows 15.4 / 17.6 and 21 / 30; bf16, one row of
  // 32 000 (eight blocks) 9.0 / 8.0 and 13.0 / 12.6, 128 rows (two blocks) 17.1 / 14.2 and 21 / 26, 100 of 5000 (one block) 11.2 / 11.2 and 16 / 22: 16-bit numbers,
  // whose borders are found in one go, do without it where a row has several blocks, or two and no top-p.
  constexpr int HERE = THREADS == SR_WIDE ? SR_LIST : SR_LIST / 2, EACH = HERE / THREADS;
  const bool alone = sizeof(T) == 4 || C == 1 || (C == 2 && top_p < 1.f);
  auto finish_here = [&](int last, double want) {
    float* const value_here = reinterpret_cast<float*>(&sh.hist[turn][0][0]);      // (zeros that nobody reads)
    int* const place_here = reinterpret_cast<int*>(value_here + HERE);
    auto in = [&](float v) { return v >= lowest && step_at(v) <= SR_STEP0 + last; };
    int n = 0;
    each(lowest, [&](const float (&x)[N], int) {
#pragma unroll
      for (int e = 0; e < N; ++e) n += in(x[e]) ? 1 : 0;
    });
    n = __reduce_add_sync(0xffffffffu, n);
    if (lane == 0) sh.warp_key[warp] = n;
    __syncthreads();
    int at = 0, all = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      at += w < warp ? (int)sh.warp_key[w] : 0;
      all += (int)sh.warp_key[w];
    }
    each(lowest, [&](const float (&x)[N], int j) {
      int mine = 0;
#pragma unroll
      for (int e = 0; e < N; ++e) mine += in(x[e]) ? 1 : 0;
      if (!__any_sync(0xffffffffu, mine > 0)) return;
      int incl = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
      }
      int to = at + incl - mine;
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (in(x[e])) {
          if (to < HERE) value_here[to] = x[e], place_here[to] = i0 + j * 32 * N + e;
          ++to;
        }
      at += __shfl_sync(0xffffffffu, incl, 31);
    });
    if (t == 0) sh.listed[0] = (uint32_t)all;
    cluster.sync();
    float v[EACH];
    int place[EACH];
    n = 0;
    if (rank == 0) {
      if (t < C) sh.key[t] = remote(there(&sh.listed[0], t));
      __syncthreads();
#pragma unroll
      for (int q = 0; q < EACH; ++q) {
        const int i = t * EACH + q;
        int first_of = 0;
        v[q] = -INFINITY, place[q] = -1;
        for (int c = 0; c < C; ++c) {
          const int of_c = (int)sh.key[c];
          if (i >= first_of && i < first_of + of_c) {
            v[q] = __uint_as_float(remote(there(value_here + i - first_of, c)));
            place[q] = (int)remote(there(place_here + i - first_of, c));
          }
          first_of += of_c;
        }
        n = min(first_of, HERE);
        sh.list_key[i] = __float_as_uint(v[q]);
      }
    }
    cluster.sync();                              // (the other blocks may go)
    if (rank > 0) return;
    n = (n + 3) & ~3;                            // (-inf behind the last one)
    const float4* values = reinterpret_cast<const float4*>(sh.list_key);
    u64 w[EACH], sum = 0;
#pragma unroll
    for (int q = 0; q < EACH; ++q) {
      bool keep = place[q] >= 0;
      if (want < 0.0 && __any_sync(0xffffffffu, keep)) {                          // as large as the k-th largest: fewer than k are larger
        int larger = 0;
#pragma unroll 4
        for (int j = 0; j < n / 4; ++j) {
          const float4 o = values[j];
          larger += (o.x > v[q] ? 1 : 0) + (o.y > v[q] ? 1 : 0) + (o.z > v[q] ? 1 : 0) + (o.w > v[q] ? 1 : 0);
        }
        keep = keep && larger < top_k;
      }
      w[q] = keep ? weight(v[q]) : 0;
      sh.list_weight[t * EACH + q] = w[q];
      sum += w[q];
    }
    auto block_before = [&](u64 x, u64& total) {
      __syncthreads();                           // (the sums before have been read)
      return threads_before<THREADS>(x, sh.scan, total);
    };
    u64 total;
    block_before(sum, total);
    if (top_p < 1.f) {                           // what is larger does not reach it
      if (want < 0.0) want = (double)top_p * (double)total;
      const ulonglong2* weights = reinterpret_cast<const ulonglong2*>(sh.list_weight);
#pragma unroll
      for (int q = 0; q < EACH; ++q) {
        if (!__any_sync(0xffffffffu, w[q] > 0)) continue;
        u64 larger = 0;
#pragma unroll 2
        for (int j = 0; j < n / 4; ++j) {
          const float4 o = values[j];
          const ulonglong2 a = weights[2 * j], b = weights[2 * j + 1];
          larger += (o.x > v[q] ? a.x : 0) + (o.y > v[q] ? a.y : 0) + (o.z > v[q] ? b.x : 0) + (o.w > v[q] ? b.y : 0);
        }
        if (larger > 0 && (double)larger >= want) w[q] = 0;
      }
    }
    const u64 least = min_p > 0.f ? (u64)ceil((double)fminf(min_p, 1.f) * SR_ONE) : 0;
    sum = 0;
#pragma unroll
    for (int q = 0; q < EACH; ++q) {
      if (w[q] < least) w[q] = 0;
      sum += w[q];
    }
    u64 running = block_before(sum, total);
    const u64 target = first ? 0 : min((u64)floor((double)u * (double)total), total - 1);
#pragma unroll
    for (int q = 0; q < EACH; ++q) {
      if (running <= target && target < running + w[q]) a.tokens[r] = place[q];
      running += w[q];
    }
  };

  if (top_k >= 1 && top_k < V) {
    uint32_t* hist = sh.hist[turn][0];
    each(cut, [&](const float (&x)[N], int) {
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float at = step_at(x[e]);
        if (at < SR_STEP0 + SR_BINS) atomicAdd(&hist[step_of(at)], 1u);
      }
    });
    cluster.sync();
    auto reached = [&](u64 n) { return n >= (u64)top_k; };
    u64 n[BINS];
    counted(false, n);
    u64 at = bins_before(n);
#pragma unroll
    for (int b = 0; b < BINS; ++b) {
      if (!reached(at) && reached(at + n[b])) sh.found = BINS * t + b, sh.found_base = at, sh.range[0] = (uint32_t)n[b];
      at += n[b];
    }
    __syncthreads();
    const int found = sh.found;
    if (found >= 0) {                            // (else all that have a weight are kept)
      const u64 base = sh.found_base;
      const bool few = sh.range[0] <= SR_LIST;
      if (alone && base + sh.range[0] <= HERE) return finish_here(found, -1.0);
      __syncthreads();
      keys_of(found, found);
      const uint32_t lo = sh.range[0], hi = sh.range[1];
      const uint32_t border = lo == hi ? hi : few ? by_list(std::false_type(), lo, hi, base, reached, 0) : by_keys(std::false_type(), lo, hi, base, reached);
      lowest = fmaxf(lowest, key_value<T>(border));
    }
  }
  // The smallest number that min-p keeps, by 32 at a time (-inf: all).
  auto least_of = [&]() {
    if (!(min_p > 0.f)) return -INFINITY;
    if (warp == 0) {
      const u64 least = (u64)ceil((double)fminf(min_p, 1.f) * SR_ONE);
      uint32_t from = order_key<T>(lowest) - 1u, to = order_key<T>(m);     // `from` weighs less or is not kept, `to` is
      while (to - from > 1u) {
        const uint32_t step = (to - from - 1u) / 33u + 1u;
        const u64 probe = min((u64)from + (u64)(lane + 1) * step, (u64)to);
        const uint32_t in = __ballot_sync(0xffffffffu, weight(fmaxf(key_value<T>((uint32_t)probe), cut)) >= least);
        const int at = in != 0u ? __ffs(in) - 1 : 32;
        const u64 above = (u64)from + (u64)at * step;
        if (in != 0u) to = (uint32_t)min(above + step, (u64)to);
        from = (uint32_t)above;
      }
      if (lane == 0) sh.least_key = to;
    }
    __syncthreads();
    return key_value<T>(sh.least_key);
  };
  float settled = -INFINITY, least_kept = -INFINITY;      // numbers above `settled` and those of a list are all that is kept
  if (top_p < 1.f) {
    // A step's weights as parts of its middle one, in 13 bits: each off by half of one in 8067, 2^-13.98 (a part is at least exp(-15.6 / 1024)), by 2^-17.4 with
    // its place in the step (two roundings of a number of 1024 and one of what is left, times 0.03), and by 2^-27 with the series: less than 2^-13 together; and a weight, rounded to a whole
    // number, by half of one, the step's middle one too.
    u64 all = 0, none;
    uint32_t* hist = sh.hist[turn][0];
    each(lowest, [&](const float (&x)[N], int) {
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float v = fmaxf(x[e], cut), at = step_at(v), d = __fmaf_rn(below(v), per_half, SR_STEP0 - at) * (SR_REACH / SR_BINS);
        const u64 w = weight(v);
        if (x[e] >= lowest) {
          all += w;
          const float part = fmaf(fmaf(fmaf(d, -1.f / 6, 0.5f), d, -1.f) * d, 8192.f, 8192.f);
          if (at < SR_STEP0 + SR_BINS) atomicAdd(&hist[step_of(at)], (uint32_t)(__float_as_int(part + 8388608.f) & 0x7fffff));
        }
      }
    });
    all = cluster_sum(all, none);
    const double want = (double)top_p * (double)all;
    u64 n[BINS];
    uint32_t numbers[BINS];
    counted(false, n);
#pragma unroll
    for (int b = 0; b < BINS; ++b) {
      numbers[b] = ((uint32_t)n[b] + 8059u) / 8060u;         // at most
      n[b] = (u64)((double)n[b] * ((double)weight_of(-(BINS * t + b) * (double)(SR_REACH / SR_BINS), SR_PER, sh.exps) * (1.0 / 8192)));
    }
    u64 at = bins_before(n);
    constexpr double OFF = 1.0 / 8192;
    auto may = [&](u64 x) { return ((double)x + 2 * V + 1024) * (1.0 + OFF) >= want; };
    auto must = [&](u64 x) { return x > 0 && ((double)x - 2 * V - 1024) * (1.0 - OFF) >= want; };
#pragma unroll
    for (int b = 0; b < BINS; ++b) {
      if ((BINS * t + b == 0 || !may(at)) && may(at + n[b])) sh.found = BINS * t + b;
      if (!must(at) && must(at + n[b])) sh.last = BINS * t + b;
      at += n[b];
    }
    __syncthreads();
    const int from = max(sh.found, 0), to = sh.last;
#pragma unroll
    for (int b = 0; b < BINS; ++b) {
      if (BINS * t + b >= from && BINS * t + b <= to) atomicAdd(&sh.range[0], numbers[b]);
      if (BINS * t + b <= to && numbers[b] > 0) atomicAdd(&sh.range[1], numbers[b]);
    }
    __syncthreads();
    const bool few = sh.range[0] <= SR_LIST;
    if (alone && sh.range[1] <= HERE) return finish_here(to, want);
    __syncthreads();
    keys_of(from, to);
    const uint32_t lo = sh.range[0], hi = sh.range[1];
    auto reached = [&](u64 x) { return x > 0 && (double)x >= want; };
    least_kept = least_of();
    if (least_kept <= key_value<T>(hi)) {        // (else min-p keeps less than top-p)
      if (lo != hi && few) settled = key_value<T>(hi);
      const uint32_t border = lo == hi ? hi : few ? by_list(std::true_type(), lo, hi, 0, reached, 1) : by_keys(std::true_type(), lo, hi, 0, reached);
      lowest = fmaxf(lowest, key_value<T>(border));
    }
  } else {
    least_kept = least_of();
  }
  lowest = fmaxf(lowest, least_kept);

  // ---- kept weights
  auto kept = [&](float v) -> u64 {
    const u64 w = weight(fmaxf(v, cut));
    return v >= lowest ? w : 0;
  };
  u64 before = 0, total = 0;
  if (settled > -INFINITY) cluster.barrier_wait();
  if (lowest <= settled) {                       // top-p's list and what lies above it: sums of warps and blocks without another look at the row
    const uint32_t from = order_key<T>(lowest);
    const u64* const weight_here = reinterpret_cast<const u64*>(&sh.hist[turn ^ 1][0][0]);
    const uint32_t *const key_here = reinterpret_cast<const uint32_t*>(weight_here + SR_LIST), *const warp_here = key_here + SR_LIST;
    if (lane == 0) sh.scan[warp] = warp_above;
    if (t < C) sh.kept[t] = sh.sums[sums ^ 1][t];
    __syncthreads();
    for (int i = t; i < min((int)sh.listed[1], SR_LIST); i += THREADS)
      if (key_here[i] >= from) atomicAdd(&sh.scan[warp_here[i]], weight_here[i]);
    for (int i = t; i < listed; i += THREADS) {
      if (sh.list_key[i] < from) continue;
      int c = 0;
      for (int end = (int)sh.key[0]; i >= end; end += (int)sh.key[c]) ++c;
      atomicAdd(&sh.kept[c], sh.list_weight[i]);
    }
    __syncthreads();
    for (int c = 0; c < C; ++c) {
      if (c == rank) before = total;
      total += sh.kept[c];
    }
  } else {
    u64 n = 0;
    each(lowest, [&](const float (&x)[N], int) {
#pragma unroll
      for (int e = 0; e < N; ++e) n += kept(x[e]);
    });
    total = cluster_sum(n, before);
  }
  const u64 target = first ? 0 : min((u64)floor((double)u * (double)total), total - 1);
  // the warp that the target falls to goes through its run
  u64 in_block;
  before += warps_before<WARPS>(sh.scan, in_block);
  if (target < before || target >= before + sh.scan[warp]) return;
  each(lowest, [&](const float (&x)[N], int j) {
    u64 w[N], incl = 0;
#pragma unroll
    for (int e = 0; e < N; ++e) w[e] = kept(x[e]), incl += w[e];
    const u64 own = incl;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const u64 v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    u64 at = before + incl - own;
    if (at <= target && target < at + own) {
      int e0 = 0;
#pragma unroll
      for (int e = 0; e < N; ++e) {
        at += w[e];
        if (at <= target) e0 = e + 1;
      }
      a.tokens[r] = i0 + j * 32 * N + e0;
    }
    before += __shfl_sync(0xffffffffu, incl, 31);
  });
}

// Blocks a row: enough that a thread has at most 32 numbers (eight at most: 68 in rows of 2^18), and more while there are fewer blocks than SMs.  us without a border and under top-p, by
// one / two / four / eight blocks a row of 32 000 (bf16): one row 14.0, 34 / 9.0, 22 / 6.6, 17 / 5.3, 14; 64 rows 14.6, 40 / 9.6, 26 / 8.8, 23 / 12.7, 36; 128 rows 14.7, 41 / 13.2, 35 / 17.0, 45 / 24.5, 69.
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
