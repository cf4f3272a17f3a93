// Attention of prompts over the paged 4-bit cache on tcgen05: S = Q K^T and O += P V with fp32 accumulators in tensor memory.
//
// A block owns two tiles of 128 columns (queries of the heads that share a key head) of one request and walks a range of its pages of 64 keys:
//   warps 0-7, 8-15 : softmax of tile 0 / tile 1, two threads a row with 32 of its 64 scores each; before, they bring the queries as fp16
//   warps 16, 17    : one thread each issues the MMAs of a tile: the scores of the next page first, then P V of this one (18, 19: nothing)
//   warps 20-27     : two sets that take the pages in turn, a warp a slice of 16 keys: codes by bulk copies into a ring, from there as fp16 numbers into
//                     the operands.  (One set took 2600 clocks a page, and with it the block; 700 tokens over 5000 keys, 32 / 8 heads: 132 -> 125 us.)
// All operands are fp16, whatever the cache's type: its 11 bits hold a query exactly (a row under a power of two of its own) and a key or value
// c s + lo rounded once, where bf16 would lose three bits more.  Where the result is fp16, whose 11 bits show that, keys are two terms (split_terms), and
// weights too: five prompts of up to 3333, 8 heads of 64, differ from 64 bits by 0.00028 of their norm instead of 0.00064 (0.00034 with the keys' terms
// alone), in 158 us instead of 134.  (Values as two terms instead of weights: 0.00029, 180 us.  Eight warps unpack, sixteen weigh.)
// What fp16 numbers do not hold (group_fits) is left to the walk of few columns: a tile that sees such a group, or one that is no number, stores nothing and
// is named in `odd`.  (Powers of two by slices of keys cost what stands beside a large number its bits, also in rows that do not see it, and 3 to 14 us of the
// prompts here.)
// A word's codes become pairs by masks: 1024 + c under exponent bits, from which one operation takes the 1024 (of odd nibbles, 1024 + 16 c, 64 + c), and
// one more multiplies and adds.  Keys' pairs run along the dimensions, values' along the keys: values stand with the keys in a row, so that both
// operands are K-major.
// What bounds it: no pipe (issue slots 62 %, exponential unit 32, tensor pipe 31) but the chain of a page's turn, some 1.4 us: scores, their maximum, the meeting
// of a row's two threads, weights, arrivals, and the unpacking beside it; leaving either of these two out gains 8 to 15 %.  A prompt of 2048, 32 heads of 128, us:
// 92 with the queries a row a thread (8000 clocks of a block) and all walks cut, 73 with whole rows and walks as they are, 64 with two sets of unpacking warps
// and the other sequences' kernel let in at the end, 62 with waits and loops as one turn of code, 59 without powers of two; over the bf16 cache
// (csrc/attn_tc.cuh) 65.  With values that are all left to the walk of few columns 328.
// Every wait is bounded; one that runs out records a code, all roles stop, copies in flight are waited for, tensor memory is freed.
#include <type_traits>

#include "attn_tc.cuh"
#include "paged_work.cuh"

namespace llb {
namespace {

// Warps: softmax, MMA issuers (two of four), two sets of four that bring codes into operands, a page each in turn.
constexpr int KP_ROWS = 128, KP_SOFTMAX = 16, KP_FIRST = KP_SOFTMAX + 4, KP_SETS = 2, KP_DEQUANT = 4 * KP_SETS, KP_THREADS = (KP_FIRST + KP_DEQUANT) * 32;
// registers a thread: 72 at the launch; the softmax takes what the others leave
constexpr int KP_REGS = 72, KP_REGS_SOFTMAX = 88, KP_REGS_MMA = 40, KP_REGS_DEQUANT = 56;
static_assert(KP_THREADS * KP_REGS <= 65536 && KP_SOFTMAX * KP_REGS_SOFTMAX + 4 * KP_REGS_MMA + KP_DEQUANT * KP_REGS_DEQUANT <= KP_THREADS / 32 * KP_REGS, "registers");
constexpr int KP_QBOX = KP_ROWS * 128, KP_KBOX = KV4_PAGE * 128;      // 64 numbers of 16 bits a row
constexpr int KP_COPIES = 2;                                         // in flight a slice of a set
// A row's largest weight is 2^KP_UP or more, so that a weight in fp16 comes to nothing under 2^-31 of it only, and under 2^15: its scores may outgrow the
// reference by KP_SLACK before it moves.
constexpr float KP_UP = 6.f, KP_SLACK = KP_UP + AT_SLACK;

// TERMS: of a key and of a weight, two where the result is fp16.  STAGES: pages of K and of V.
template <typename T, int D, int NG>
struct KpShape {
  static constexpr int TERMS = std::is_same<T, __half>::value ? 2 : 1, STAGES = TERMS == 2 && D == 128 ? 2 : 3;
  static constexpr int NB = (D + 63) / 64, SLICE = kv4_slice_bytes(D, NG);
  static constexpr int Q = 2 * NB * KP_QBOX, K = TERMS * NB * KP_KBOX, V = D * 128;
  static constexpr int RING = KP_DEQUANT * KP_COPIES * SLICE, SPLIT = TERMS == 2 ? KP_DEQUANT * KV4_SLICE * NG * 16 : 0;
  static constexpr int SMEM = 1024 + Q + STAGES * (K + V) + RING + SPLIT + 512 + 6 * KP_ROWS * 4;
};

__device__ __forceinline__ void kp_ran_out(volatile int* fail, int* word, int code) {
  *fail = 1;
  wait_ran_out(word, 810 + code);
}
// A wait that ends: on its phase, when another role has given up, or after the limit.
__device__ __forceinline__ bool kp_wait(uint64_t* bar, uint32_t parity, volatile int* fail, int* word, int code) {
#pragma unroll 1
  for (uint32_t i = 0; !mbar_try_wait(bar, parity); ++i) {
    if ((i & 255u) != 255u) continue;
    if (*fail) return false;
    if (i >= AT_WAIT_LIMIT) {
      kp_ran_out(fail, word, code);
      return false;
    }
  }
  return true;
}
__host__ __device__ constexpr uint32_t instr_desc_f16(int M, int N) { return (1u << 4) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24); }
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }      // -126 <= e <= 127

// Whether a group of scale s and lowest value lo (the halves of a word) keeps its bits as fp16 numbers: |c s + lo| is under 2^13, and rounding it and, from bf16,
// s and lo costs 2^-10 of the group's largest (2^-11 of it over 2^-13; a bf16 scale from 2^-17 on is exact, and a smaller one is off by 2^-25, 15 codes 2^-21).
// Then weights that come to nothing (2^-31 of a row's largest) take 2^-18 from a result at most.  A group that is no number does not fit, one of zeros does.
template <typename T>
__device__ __forceinline__ bool group_fits(uint32_t w) {
  constexpr bool F = std::is_same<T, __half>::value;
  constexpr uint32_t S_LARGE = F ? 0x5c00u : 0x4380u, LO_LARGE = F ? 0x6c00u : 0x4580u;      // 2^8, 2^12
  constexpr uint32_t S_SMALL = F ? 0x0100u : 0x3780u, LO_SMALL = F ? 0x1400u : 0x3a80u;      // 2^-16, 2^-10
  const uint32_t s = w & 0x7fffu, lo = (w >> 16) & 0x7fffu;
  return s < S_LARGE && lo < LO_LARGE && (s >= S_SMALL || lo >= LO_SMALL || (s | lo) == 0u);
}
__device__ __forceinline__ __half2 as_half2(uint32_t u) { return *reinterpret_cast<const __half2*>(&u); }
__device__ __forceinline__ uint32_t as_u32(__half2 v) { return *reinterpret_cast<const uint32_t*>(&v); }
// the pairs of nibble n of a word, as c s + lo
template <int N>
__device__ __forceinline__ uint32_t word_pair(uint32_t w, __half2 s, __half2 lo) {
  const uint32_t u = N >= 2 ? w >> 8 : w;
  const __half2 c = (N & 1) ? __hfma2(as_half2((u & 0x00f000f0u) | 0x64006400u), __half2half2(__ushort_as_half(0x2c00)), __half2half2(__ushort_as_half(0xd400)))
                            : __hadd2(as_half2((u & 0x000f000fu) | 0x64006400u), __half2half2(__ushort_as_half(0xe400)));      // (1/16, -64; -1024)
  return as_u32(__hfma2(c, s, lo));
}
// Two terms of such pairs.  With m the code next to 0, s1 the first seven bits of s and s2 the others, c s + lo = (c - m) s1 + ((c - m) s2 + (lo + m s)).  The
// first term is exact in 11 bits; the second is under s where the group's range holds 0, so that its rounding is 2^-12 of s (of |lo| where it does not,
// as one term's).  x: -1024 - m, y: s1, z: s2, w: lo + m s, twice each.
__device__ __forceinline__ uint4 split_terms(uint32_t params) {
  const float2 p = __half22float2(as_half2(params));
  const float m = p.x > 0.f ? fminf(fmaxf(rintf(__fdividef(-p.y, p.x)), 0.f), 15.f) : 0.f;
  const __half2 s = as_half2(__byte_perm(params, params, 0x1010)), s1 = as_half2(as_u32(s) & 0xfff0fff0u);
  return make_uint4(as_u32(__float2half2_rn(-1024.f - m)), as_u32(s1), as_u32(__hsub2(s, s1)), as_u32(__float2half2_rn(fmaf(m, p.x, p.y))));
}
template <int N>
__device__ __forceinline__ void word_terms(uint32_t w, uint4 t, uint32_t& a, uint32_t& b) {
  const uint32_t u = N >= 2 ? w >> 8 : w;
  const __half2 even = as_half2(t.x), odd = __hadd2(even, __half2half2(__ushort_as_half(0x6380)));      // (960)
  const __half2 c = (N & 1) ? __hfma2(as_half2((u & 0x00f000f0u) | 0x64006400u), __half2half2(__ushort_as_half(0x2c00)), odd)
                            : __hadd2(as_half2((u & 0x000f000fu) | 0x64006400u), even);
  a = as_u32(__hmul2(c, as_half2(t.y))), b = as_u32(__hfma2(c, as_half2(t.z), as_half2(t.w)));
}

template <typename T, int D, int NG>
__global__ void __launch_bounds__(KP_THREADS, 1) kv4_prompt_kernel(const Kv4Attn a) {
  using Shape = KpShape<T, D, NG>;
  constexpr int TERMS = Shape::TERMS, STAGES = Shape::STAGES, NB = Shape::NB, SLICE = Shape::SLICE, W = D / 32, BYTES = kv4_bytes(D, NG);
  constexpr uint32_t TM_S = 0, TM_O = 256;            // per tile: two score buffers of 64 columns; 128 accumulator columns
  extern __shared__ __align__(1024) uint8_t smem[];
  const int item = blockIdx.x / a.G, head = blockIdx.x - item * a.G;
  const Kv4Item it = load_item(a.work, item);                           // (there is room for it: asked for together with the number of parts)
  if (item >= a.work[0]) return;
  const int R = a.H / a.G, cols_all = it.count * R, col0 = it.tile * KV4_MANY, cols = min(KV4_MANY, cols_all - col0);
  T* const y = (T*)a.y;
  if (it.row < 0) {                     // a refused sequence's tokens are no numbers
    if (threadIdx.x == 0) a.odd[blockIdx.x] = 0;
#pragma unroll 1
    for (int e = threadIdx.x; e < cols * D; e += KP_THREADS) {
      const int c = col0 + e / D;
      dt<T>::st(y, ((size_t)(it.first + c / R) * a.H + head * R + c % R) * D + e % D, NAN);
    }
    return;
  }
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem) + 1023) & ~(uintptr_t)1023);
  uint8_t* sq = base;                                 // [2 tiles][NB][128][64]
  uint8_t* sk = sq + Shape::Q;                        // [stage][NB][64 keys][64]
  uint8_t* sv = sk + STAGES * Shape::K;            // [stage][D][64 keys]
  uint8_t* ring = sv + STAGES * Shape::V;          // [slice][stage]
  uint64_t* q_full = reinterpret_cast<uint64_t*>(ring + Shape::RING + Shape::SPLIT);
  uint64_t* k_full = q_full + 1;
  uint64_t* k_empty = k_full + STAGES;
  uint64_t* v_full = k_empty + STAGES;
  uint64_t* v_empty = v_full + STAGES;
  uint64_t* s_full = v_empty + STAGES;             // [tile][buffer] scores are there
  uint64_t* p_full = s_full + 4;                      // [tile][buffer] weights are there
  uint64_t* o_full = p_full + 4;                      // [tile][buffer] P V is done
  uint64_t* r_full = o_full + 4;                      // [slice][stage]
  uint32_t* tmem_ptr = reinterpret_cast<uint32_t*>(r_full + KP_DEQUANT * KP_COPIES);
  int* s_fail = reinterpret_cast<int*>(tmem_ptr + 1);
  volatile int* s_odd = s_fail + 1;                   // [tile] whether the tile sees a group that fp16 numbers do not hold
  float* s_x = reinterpret_cast<float*>(ring + Shape::RING + Shape::SPLIT + 512);      // [tile][half][row]: what the two threads of a row tell one another
  float* s_mul = s_x + 4 * KP_ROWS;                   // [2 tiles][row] what a row's raw scores are multiplied by

  const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  // what every role walks: pages page0 .. page1; per tile the last page that one of its rows sees
  const int last = it.pos0 + column_token(col0 + cols - 1, R), page0 = it.page0;
  const int hi1 = cols > KP_ROWS ? min(it.page1, last / KV4_PAGE + 1) - 1 : -1;
  const int hi0 = min(it.page1, (it.pos0 + column_token(col0 + min(cols, KP_ROWS) - 1, R)) / KV4_PAGE + 1) - 1;
  const int page_last = max(hi0, hi1);

  const int units = page_last - page0 + 1;
  // codes into operands: the first copies are on their way before the block meets
  const int dq = warp - KP_FIRST, sl = dq & 3, set = dq >> 2;         // (the slice and the set of a warp of theirs)
  const int turns = (units - set + KP_SETS - 1) / KP_SETS;             // pages set, set + KP_SETS ..
  const int32_t* table = a.table + (size_t)it.row * a.width + page0 + set;
  const uint8_t* from = a.blocks + (size_t)head * BYTES + sl * SLICE;
  const size_t page_bytes = (size_t)a.G * BYTES;
  uint8_t* mine = ring + dq * KP_COPIES * SLICE;
  uint64_t* full = r_full + dq * KP_COPIES;
  uint8_t* split = ring + Shape::RING + dq * (KV4_SLICE * NG * 16);
  int entry = 0;
  if (dq >= 0) {
    entry = lane < turns ? table[KP_SETS * lane] : 0;
    if (lane == 0) {
      for (int i = 0; i < KP_COPIES; ++i) mbar_init(&full[i], 1);
      fence_barrier_init();
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < KP_COPIES; ++i) {
      const int page = __shfl_sync(0xffffffffu, entry, i);
      if (lane == 0 && i < turns) {
        mbar_expect_tx(&full[i], SLICE);
        bulk_load_1d(mine + i * SLICE, from + min(max(page, 0), a.pages - 1) * page_bytes, SLICE, &full[i]);
      }
    }
  }
  if (threadIdx.x == 0) {
    mbar_init(q_full, KP_SOFTMAX);
    for (int i = 0; i < STAGES; ++i) mbar_init(&k_full[i], 4), mbar_init(&k_empty[i], 2), mbar_init(&v_full[i], 4), mbar_init(&v_empty[i], 2);
    for (int i = 0; i < 4; ++i) mbar_init(&s_full[i], 1), mbar_init(&p_full[i], KP_SOFTMAX / 2), mbar_init(&o_full[i], 1);
    *s_fail = s_odd[0] = s_odd[1] = 0;
    fence_barrier_init();
  }
  if (warp == KP_SOFTMAX) tmem_alloc(tmem_ptr, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_ptr, 0);
  // (Not before the block has its tensor memory: a kernel let in that fits beside it could take that first, and then waits for this one's end.)
  pdl_launch_dependents();

  if (warp >= KP_FIRST) {
    // ===================== codes into operands =====================
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(KP_REGS_DEQUANT));
    const int t4 = lane & 3, g8 = lane >> 2;
    bool ok = true;
#pragma unroll 1
    for (int turn = 0; turn < turns; ++turn) {
      const int n = KP_SETS * turn + set, st = turn % KP_COPIES, ks = n % STAGES;
      ok = __all_sync(0xffffffffu, kp_wait(&full[st], (turn / KP_COPIES) & 1, s_fail, a.word, 1));
      if (!ok) break;
      const uint8_t* blk = mine + st * SLICE;
      uint32_t kw[2][W], vw[2][W];
      uint32_t kp[2][NG], vp[2][2][NG];               // parameters of keys g8 + 8 x and of the values of slots 2 (t4 + 4 x) + e
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        lds_words<W>(kw[x], blk + (g8 + 8 * x) * (D / 2) + t4 * 4 * W);
        lds_words<W>(vw[x], blk + kv4_v_codes(D) + (t4 + 4 * x) * D + g8 * 4 * W);
        lds_words<NG>(kp[x], blk + kv4_k_params(D) + (g8 + 8 * x) * NG * 4);
#pragma unroll
        for (int e = 0; e < 2; ++e) lds_words<NG>(vp[x][e], blk + kv4_v_params(D, NG) + (2 * (t4 + 4 * x) + e) * NG * 4);
      }
      const int page_at = page0 + n, pos = page_at * KV4_PAGE + KV4_SLICE * sl;
      {                                               // (a lane has the groups of a key or of a value)
        uint32_t mine[NG];
        lds_words<NG>(mine, blk + kv4_k_params(D) + lane * NG * 4);
        bool fits = true;
#pragma unroll
        for (int g = 0; g < NG; ++g) fits &= group_fits<T>(mine[g]);
        if (!fits && pos + (lane & (KV4_SLICE - 1)) <= last) {
          if (page_at <= hi0) s_odd[0] = 1;
          if (page_at <= hi1) s_odd[1] = 1;
        }
      }
      if (pos + KV4_SLICE - 1 > last) {               // (a slot behind the last key may hold anything)
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int g = 0; g < NG; ++g) {
            if (pos + g8 + 8 * x > last) kp[x][g] = 0u;
#pragma unroll
            for (int e = 0; e < 2; ++e)
              if (pos + 2 * (t4 + 4 * x) + e > last) vp[x][e][g] = 0u;
          }
      }
      if constexpr (TERMS == 2) {                     // (a lane splits the scales of a key's groups for the four that take the key)
#pragma unroll
        for (int z = lane; z < KV4_SLICE * NG; z += 32) {
          const uint32_t p = *reinterpret_cast<const uint32_t*>(blk + kv4_k_params(D) + 4 * z);
          reinterpret_cast<uint4*>(split)[z] = split_terms(pos + z / NG <= last ? p : 0u);
        }
      }
      const int nxt = turn + KP_COPIES;
      if ((nxt & 31) == 0) entry = nxt + lane < turns ? table[KP_SETS * (nxt + lane)] : 0;
      const int page = __shfl_sync(0xffffffffu, entry, nxt & 31);
      __syncwarp();                                   // every lane has read the slice
      if (lane == 0 && nxt < turns) {
        mbar_expect_tx(&full[st], SLICE);
        bulk_load_1d(mine + st * SLICE, from + min(max(page, 0), a.pages - 1) * page_bytes, SLICE, &full[st]);
      }
      // keys: row = slot, 8 bytes of four dimensions at a time
      ok = __all_sync(0xffffffffu, kp_wait(&k_empty[ks], ((n / STAGES) & 1) ^ 1, s_fail, a.word, 2));
      if (!ok) break;
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int r = KV4_SLICE * sl + g8 + 8 * x;
#pragma unroll
        for (int i = 0; i < W; ++i) {
          uint8_t* row = sk + ks * Shape::K + (i >> 1) * KP_KBOX + r * 128;
          const int c = 4 * (i & 1) + (t4 >> 1), b = 8 * (t4 & 1);      // 16-byte piece of dimensions 32 i + 4 t4 in the row, 8 bytes in it
          uint8_t *const first = row + ((c ^ (r & 7)) << 4) + b, *const second = row + (((c + 2) ^ (r & 7)) << 4) + b;
          if constexpr (TERMS == 2) {
            const uint4 t = reinterpret_cast<const uint4*>(split)[(g8 + 8 * x) * NG + i * NG / W];
            uint2 u, v;
            word_terms<0>(kw[x][i], t, u.x, v.x), word_terms<1>(kw[x][i], t, u.y, v.y);
            *reinterpret_cast<uint2*>(first) = u, *reinterpret_cast<uint2*>(first + NB * KP_KBOX) = v;
            word_terms<2>(kw[x][i], t, u.x, v.x), word_terms<3>(kw[x][i], t, u.y, v.y);
            *reinterpret_cast<uint2*>(second) = u, *reinterpret_cast<uint2*>(second + NB * KP_KBOX) = v;
          } else {
            const float2 p = bits_pair<T>(kp[x][i * NG / W]);
            const __half2 s = __float2half2_rn(p.x), lo = __float2half2_rn(p.y);
            *reinterpret_cast<uint2*>(first) = make_uint2(word_pair<0>(kw[x][i], s, lo), word_pair<1>(kw[x][i], s, lo));
            *reinterpret_cast<uint2*>(second) = make_uint2(word_pair<2>(kw[x][i], s, lo), word_pair<3>(kw[x][i], s, lo));
          }
        }
      }
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(&k_full[ks]);
      // values: row = dimension, a pair of slots at a time
      ok = __all_sync(0xffffffffu, kp_wait(&v_empty[ks], ((n / STAGES) & 1) ^ 1, s_fail, a.word, 3));
      if (!ok) break;
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int i = 0; i < W; ++i) {
          uint8_t* at = sv + ks * Shape::V + (32 * i + g8) * 128 + (((2 * sl + x) ^ g8) << 4) + 4 * t4;
          __half2 s, lo;
          if constexpr (TERMS == 2) {
            s = as_half2(__byte_perm(vp[x][0][i * NG / W], vp[x][1][i * NG / W], 0x5410)), lo = as_half2(__byte_perm(vp[x][0][i * NG / W], vp[x][1][i * NG / W], 0x7632));
          } else {
            const float2 p0 = bits_pair<T>(vp[x][0][i * NG / W]), p1 = bits_pair<T>(vp[x][1][i * NG / W]);
            s = __floats2half2_rn(p0.x, p1.x), lo = __floats2half2_rn(p0.y, p1.y);
          }
          *reinterpret_cast<uint32_t*>(at) = word_pair<0>(vw[x][i], s, lo);
          *reinterpret_cast<uint32_t*>(at + 8 * 128) = word_pair<1>(vw[x][i], s, lo);
          *reinterpret_cast<uint32_t*>(at + 16 * 128) = word_pair<2>(vw[x][i], s, lo);
          *reinterpret_cast<uint32_t*>(at + 24 * 128) = word_pair<3>(vw[x][i], s, lo);
        }
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(&v_full[ks]);
    }
    if (!ok && lane == 0) kv4_let_end();
    __syncwarp();
  } else if (warp >= KP_SOFTMAX) {
    // ===================== MMA issuers, one thread per tile =====================
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(KP_REGS_MMA));
    if (warp < KP_SOFTMAX + 2 && elect_one()) {
      constexpr uint32_t idesc_s = instr_desc_f16(KP_ROWS, KV4_PAGE), idesc_o = instr_desc_f16(KP_ROWS, D);
      const int i = warp - KP_SOFTMAX, myhi = i == 0 ? hi0 : hi1;
      const uint32_t tm_s = tmem + TM_S + 128u * i, tm_o = tmem + TM_O + 128u * i;
      const uint64_t qdesc = smem_desc_sw128(smem_u32(sq + i * NB * KP_QBOX));
      const uint64_t kdesc0 = smem_desc_sw128(smem_u32(sk)), vdesc0 = smem_desc_sw128(smem_u32(sv));
      auto scores = [&](int n) {
        const int ks = n % STAGES;
        if (!kp_wait(&k_full[ks], (n / STAGES) & 1, s_fail, a.word, 4)) return false;
        tc_fence_after();
        if (page0 + n <= myhi) {
          const uint32_t d = tm_s + 64u * (n & 1);
          const uint64_t kdesc = kdesc0 + (uint64_t)(ks * (Shape::K >> 4));
#pragma unroll
          for (int c = 0; c < TERMS * NB; ++c)
#pragma unroll
            for (int k = 0; k < (D < 64 ? D / 16 : 4); ++k)
              umma_bf16(d, qdesc + (uint64_t)(c % NB * (KP_QBOX >> 4) + 2 * k), kdesc + (uint64_t)(c * (KP_KBOX >> 4) + 2 * k), idesc_s, (c | k) != 0 ? 1u : 0u);
          umma_commit(&s_full[2 * i + (n & 1)]);
          umma_commit(&k_empty[ks]);
        } else {
          mbar_arrive(&k_empty[ks]);
        }
        return true;
      };
      bool ok = kp_wait(q_full, 0, s_fail, a.word, 5);
      if (ok && units > 0) ok = scores(0);
#pragma unroll 1
      for (int n = 0; ok && n < units; ++n) {
        if (n + 1 < units && !(ok = scores(n + 1))) break;
        const int vs = n % STAGES;
        if (!(ok = kp_wait(&v_full[vs], (n / STAGES) & 1, s_fail, a.word, 6))) break;
        if (page0 + n <= myhi) {
          const uint32_t buf = n & 1;
          if (!(ok = kp_wait(&p_full[2 * i + (int)buf], (n >> 1) & 1u, s_fail, a.word, 7))) break;
          tc_fence_after();
          const uint64_t vdesc = vdesc0 + (uint64_t)(vs * (Shape::V >> 4));
#pragma unroll
          for (int k = 0; k < KV4_PAGE / UMMA_K; ++k)      // 16 keys: 8 columns of packed weights, a term
#pragma unroll
            for (int t = 0; t < TERMS; ++t)
              umma_ts(tm_o, tm_s + 64u * buf + 32u * (k >> 1) + 16u * t + 8u * (k & 1), vdesc + (uint64_t)(2 * k), idesc_o, (n | k | t) != 0 ? 1u : 0u);
          umma_commit(&o_full[2 * i + (int)buf]);
          umma_commit(&v_empty[vs]);
        } else {
          mbar_arrive(&v_empty[vs]);
        }
      }
      if (!ok) kv4_let_end();
    }
    __syncwarp();
  } else {
    // ===================== queries, softmax, then the epilogue =====================
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(KP_REGS_SOFTMAX));
    const int tile = warp >> 3, half = (warp >> 2) & 1, row = (int)(threadIdx.x & (KP_ROWS - 1));
    const int c = col0 + tile * KP_ROWS + row, myhi = tile == 0 ? hi0 : hi1;
    const bool live = tile * KP_ROWS + row < cols;
    const int qt = column_token(live ? c : col0, R), qp = it.pos0 + qt;                // the row's token and its position
    const size_t out_row = (size_t)(it.first + qt) * a.H + head * R + column_head(live ? c : col0, R);
    float* const own = s_x + (tile * 2 + half) * KP_ROWS + row;
    const float* const other = s_x + (tile * 2 + (half ^ 1)) * KP_ROWS + row;
    const int bar = 1 + tile * 4 + (warp & 3);
    {
      // whole rows by neighbouring lanes (a row a thread took 32 lines a load, 8000 clocks of a block): 16 rows a warp
      constexpr int LV = D / 8, RPI = 32 / LV, N = 16 / RPI;            // lanes a row, rows a load, loads
      const int l = lane % LV;
      uint4 u[N];
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int r = 16 * warp + i * RPI + lane / LV, cc = col0 + r;
        u[i] = make_uint4(0u, 0u, 0u, 0u);
        if (r < cols) u[i] = *reinterpret_cast<const uint4*>((const T*)a.q + (long long)(it.first + column_token(cc, R)) * a.q_row + (size_t)(head * R + column_head(cc, R)) * D + 8 * l);
      }
      // rows as they stand, where every piece of eight numbers has one of 2^-4 .. 2^14, or only zeros: small ones lose 2^-25 then; else under a
      // power of two a row, its largest comes to 2^14 .. 2^15
      constexpr uint32_t SMALL = std::is_same<T, __half>::value ? 0x2c00u : 0x3d80u, LARGE = std::is_same<T, __half>::value ? 0x7400u : 0x4680u;
      uint32_t bigs[N];
      bool odd = false;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const uint32_t m = __vmaxu2(__vmaxu2(u[i].x & 0x7fff7fffu, u[i].y & 0x7fff7fffu), __vmaxu2(u[i].z & 0x7fff7fffu, u[i].w & 0x7fff7fffu));
        bigs[i] = max(m & 0xffffu, m >> 16);
        odd |= bigs[i] != 0u && (bigs[i] < SMALL || bigs[i] >= LARGE);
      }
      odd = __any_sync(0xffffffffu, odd);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int r = 16 * warp + i * RPI + lane / LV, tr = r & (KP_ROWS - 1);
        const uint32_t w[4] = {u[i].x, u[i].y, u[i].z, u[i].w};
        float up = 1.f, down = 1.f;
        if (odd) {
          uint32_t big = bigs[i];
#pragma unroll
          for (int o = LV / 2; o > 0; o >>= 1) big = max(big, __shfl_xor_sync(0xffffffffu, big, o));
          const int ex = min(max((int)(__float_as_uint(bits_pair<T>(big).x) >> 23), 15), 240);
          up = pow2(127 + 14 - ex), down = pow2(ex - 127 - 14);
        }
        if (l == 0) s_mul[r] = fmaxf(down * (a.scale * AT_LOG2E), 1.2e-38f);      // (not 0: masked scores are -inf)
        uint32_t h[4];
#pragma unroll
        for (int z = 0; z < 4; ++z) {
          if (std::is_same<T, __half>::value && !odd) {
            h[z] = w[z];
          } else {
            const float2 f = bits_pair<T>(w[z]);
            h[z] = odd ? pair_bits<__half>(f.x * up, f.y * up) : pair_bits<__half>(f.x, f.y);
          }
        }
        *reinterpret_cast<uint4*>(sq + ((r >> 7) * NB + (l >> 3)) * KP_QBOX + tr * 128 + (((l & 7) ^ (tr & 7)) << 4)) = make_uint4(h[0], h[1], h[2], h[3]);
      }
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_full);
      asm volatile("barrier.cta.sync 9, 512;" ::: "memory");
    }
    const float mul = s_mul[tile * KP_ROWS + row];                      // what a raw score is multiplied by, to units of log2
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t ts0 = tmem + lanes + TM_S + 128u * tile, to = tmem + lanes + TM_O + 128u * tile;
    float ref = -INFINITY, sum = 0.f;
    bool ok = true;
    bool far = false;                                                   // a reference past 2^24: a product and a rounded one of the same numbers differ
    const int count = max(0, myhi - page0 + 1);
#pragma unroll 1
    for (int n = 0; n < count; ++n) {
      const uint32_t ts = ts0 + 64u * (n & 1);
      ok = kp_wait(&s_full[2 * tile + (n & 1)], (n >> 1) & 1, s_fail, a.word, 8);
      __syncwarp();
      tc_fence_after();
      uint32_t sr[32];
      tmem_ld32_async(ts + 32u * half, sr);
      tmem_wait_ld();
      tie32(sr);
      const int cmax = qp - ((page0 + n) * KV4_PAGE + 32 * half);       // the row's last visible column of these 32
      const bool masked = __any_sync(0xffffffffu, cmax < 31);
      if (masked) {
#pragma unroll
        for (int e = 0; e < 32; ++e)
          if (e > cmax) sr[e] = __float_as_uint(-INFINITY);
      }
      float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int e = 0; e < 32; e += 2) m4[e >> 3] = at_max3(m4[e >> 3], __uint_as_float(sr[e]), __uint_as_float(sr[e + 1]));
      const float mx = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])) * mul;
      __syncwarp();      // the stores to tensor memory below are the whole warp's: lanes part above this line and not between it and them
      // (one barrier of the rows' two warps per page: does any row's reference have to move, has any wait run out?  The difference is exact where a sum
      // with the slack would be rounded; it is no number where a row has seen nothing.)
      if (at_any(bar, !ok || mx - ref > KP_SLACK)) {
        *own = mx;
        ok = !at_any(bar, !ok);
        if (!ok) break;
        const float nref = fmaxf(ref, fmaxf(mx, *other) - KP_UP);
        const float f = ref == -INFINITY ? 0.f : at_exp2(ref - nref);
        ref = nref;
        far = __any_sync(0xffffffffu, fabsf(ref) > 16777216.f && ref != -INFINITY);
        sum *= f;
        if (n > 0) ok = kp_wait(&o_full[2 * tile + ((n - 1) & 1)], ((n - 1) >> 1) & 1, s_fail, a.word, 9);
        __syncwarp();
        tc_fence_after();
        if (at_any(bar, !ok)) {                                         // (also: both threads of a row have read the other's)
          ok = false;
          break;
        }
        if (n > 0) {                                                    // what the pages before have added up
#pragma unroll 1
          for (int z = 32 * half; z < D; z += 64) {
            uint32_t o[32];
            tmem_ld32_async(to + (uint32_t)z, o);
            tmem_wait_ld();
            tie32(o);
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
            tmem_st16(to + (uint32_t)z, o);
            tmem_st16(to + (uint32_t)z + 16u, o + 16);
          }
        }
      }
      const float sub = ref == -INFINITY ? 0.f : -ref;
      uint32_t ph[16 * TERMS];
      // weights as a pair, and what their 11 bits leave over
      auto weights = [&](int e, float p0, float p1) {
        ph[e] = pair_bits<__half>(p0, p1);
        if constexpr (TERMS == 2) {
          const float2 f = bits_pair<__half>(ph[e]);
          ph[16 + e] = pair_bits<__half>(p0 - f.x, p1 - f.y);
        }
      };
      f2 part[2] = {f2_of(0.f, 0.f), f2_of(0.f, 0.f)};
      if (!far) {
        const f2 m2 = f2_of(mul, mul), s2 = f2_of(sub, sub);
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          float a0, a1;
          f2_split(f2_fma(f2_of(__uint_as_float(sr[2 * e]), __uint_as_float(sr[2 * e + 1])), m2, s2), a0, a1);
          const float p0 = at_exp2(a0), p1 = at_exp2(a1);
          part[e & 1] = f2_add(part[e & 1], f2_of(p0, p1));
          weights(e, p0, p1);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float s0 = __uint_as_float(sr[2 * e]), s1 = __uint_as_float(sr[2 * e + 1]);
          const float p0 = s0 == -INFINITY ? 0.f : at_exp2(__fadd_rn(__fmul_rn(s0, mul), sub)), p1 = s1 == -INFINITY ? 0.f : at_exp2(__fadd_rn(__fmul_rn(s1, mul), sub));
          part[e & 1] = f2_add(part[e & 1], f2_of(p0, p1));
          weights(e, p0, p1);
        }
      }
      float p0, p1;
      f2_split(f2_add(part[0], part[1]), p0, p1);
      sum += p0 + p1;
      // the weights go over the thread's own scores
      tmem_st16(ts + 32u * half, ph);
      if constexpr (TERMS == 2) tmem_st16(ts + 32u * half + 16u, ph + 16);
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[2 * tile + (n & 1)]);
    }
    if (ok && count > 0) ok = kp_wait(&o_full[2 * tile + ((count - 1) & 1)], ((count - 1) >> 1) & 1, s_fail, a.word, 10);
    __syncwarp();
    tc_fence_after();
    *own = sum;
    // (what a tile gives that sees a group out of range counts for nothing: kv4_few_kernel has its walk)
    if (!at_any(bar, !ok) && s_odd[tile] == 0) {
      const float den = half == 0 ? sum + *other : *other + sum;        // the halves' sums in the order of the keys
      const size_t part_at = ((size_t)(it.base + it.part) * a.G + head) * KV4_MANY + tile * KP_ROWS + row;
      const bool whole = it.parts == 1;
      if (!whole && live && half == 0)
        *reinterpret_cast<float2*>(a.part + (size_t)a.kept * a.G * KV4_MANY * D + part_at * 2) = make_float2(ref == -INFINITY ? KV4_NONE : ref, den);
      const float f = whole ? 1.f / den : 1.f;
      if (count > 0) {
#pragma unroll
        for (int z = 32 * half; z < D; z += 64) {
          uint32_t o[32];
          tmem_ld32_async(to + (uint32_t)z, o);
          tmem_wait_ld();
          tie32(o);
          if (live) {
            if (whole) {
              T* dst = y + out_row * D + z;
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                uint32_t w[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) w[j] = pair_bits<T>(__uint_as_float(o[8 * e + 2 * j]) * f, __uint_as_float(o[8 * e + 2 * j + 1]) * f);
                *reinterpret_cast<uint4*>(dst + 8 * e) = make_uint4(w[0], w[1], w[2], w[3]);
              }
            } else {
              float* dst = a.part + part_at * D + z;
#pragma unroll
              for (int e = 0; e < 8; ++e)
                *reinterpret_cast<float4*>(dst + 4 * e) = make_float4(__uint_as_float(o[4 * e]) * f, __uint_as_float(o[4 * e + 1]) * f,
                                                                      __uint_as_float(o[4 * e + 2]) * f, __uint_as_float(o[4 * e + 3]) * f);
            }
          }
          __syncwarp();
        }
      }
    }
    tc_fence_before();
  }
  __syncthreads();
  if (warp == KP_SOFTMAX) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
  if (threadIdx.x == 0) a.odd[blockIdx.x] = s_odd[0] | s_odd[1] << 1;
}

template <typename T, int D, int NG>
int prompt_launch(const Kv4Attn& a, cudaStream_t st) {
  constexpr int smem = KpShape<T, D, NG>::SMEM;
  static_assert(smem <= 227 * 1024, "shared memory of a block");
  static PerDevice set;
  if (!set) {
    LL_CUDA(cudaFuncSetAttribute(kv4_prompt_kernel<T, D, NG>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    set.mark();
  }
  kv4_prompt_kernel<T, D, NG><<<(unsigned)(a.items * a.G), KP_THREADS, smem, st>>>(a);
  LL_LAUNCH_OK("kv4_prompt_kernel");
  return LL_OK;
}

}  // namespace

int kv4_prompt_launch(const Kv4Attn& a, int dtype, int head_size, int group, cudaStream_t st) {
#define PROMPT(DD, NG)                                            \
  if (head_size == DD && group == DD / NG) {                      \
    if (dtype == LL_BF16) return prompt_launch<__nv_bfloat16, DD, NG>(a, st); \
    return prompt_launch<__half, DD, NG>(a, st);                  \
  }
  PROMPT(32, 1) PROMPT(64, 1) PROMPT(64, 2) PROMPT(128, 1) PROMPT(128, 2) PROMPT(128, 4)
#undef PROMPT
  set_error("kv4_attn: no prompt kernel for heads of %d in groups of %d", head_size, group);
  return LL_ERR_UNSUPPORTED;
}

}  // namespace llb
