// Softmax attention over the paged key/value cache in 4 bits (kv4.cuh): a step's tokens, of requests of unequal lengths, over the keys at and before
// their positions.
//
// With K = s c + lo and V alike, by groups of a head's dimensions (c: codes),
//   q.k_j = sum_g s_jg (q.c_j)_g + lo_jg (sum of q)_g           y = sum_j p_j v_j = sum_j (p_j s_jg) c_j + sum_j p_j lo_jg
// so that the products run over codes, which a mask turns into numbers of fp16 (subnormal ones, exactly), and scales meet 16 keys at a time.
//
// What bounds it: memory in a burst, 60 requests of up to 4096 keys, 32 heads of 128 in groups of 64, 579 MB in 91 us (97 % of the copy rate); in a loop,
// where the power cap takes the SMs from 1.97 to 1.64 GHz, its instructions (103 to 111 us), of which the masks are a third.  tcgen05 would not help: the walk
// needs no products faster, and a tile of 128 rows would hold one query a head.  us on the way there: a warp a key on the CUDA cores 1290; codes by
// mma.sync, a block's warps sharing a ring 185; a ring a warp and one look at all maxima 137; 32 keys a look and four columns of two each 118; the
// largest parts first 102; fewer masks (c + 16 c' in the second row half) and no looks behind a column but at a walk's end 94; loops as one turn of code 91.
#include <algorithm>
#include <climits>
#include <type_traits>

#include "paged_work.cuh"

namespace llb {
namespace {

constexpr int KF_WARPS = 4, KF_THREADS = KF_WARPS * 32;
// units of 32 keys in a warp's ring: four blocks an SM
__host__ __device__ constexpr int kf_stages(int D, int groups) { return 4 * KF_WARPS * 3 * 2 * kv4_slice_bytes(D, groups) <= 222 * 1024 ? 3 : 2; }
constexpr float KF_LOG2E = 1.4426950408889634f, KF_SLACK = 8.f;      // a column's scores may outgrow its reference by 2^8 before it moves
// Weights are at most 2^KF_SLACK, and scales at most KF_SCALES of what a column's sums stand under unless the unit is looked at: 2^15 in fp16.
constexpr float KF_SCALES = 128.f, KF_LEAST = 1.17549435082228751e-38f;      // (2^-126)
constexpr uint32_t KF_WAIT_LIMIT = 1u << 20;

__device__ __forceinline__ float kf_exp2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// the power of two at or under x, and one over it (2^-126 <= x <= 2^126)
__device__ __forceinline__ float pow2_of(float x) { return __uint_as_float(__float_as_uint(x) & 0x7f800000u); }
__device__ __forceinline__ float one_over_pow2(float x) { return __uint_as_float((254u << 23) - (__float_as_uint(x) & 0x7f800000u)); }
// D(16x8, f32) += A(16x16, f16, by rows) * B(16x8, f16, by columns)
__device__ __forceinline__ void mma_f16_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t movmatrix(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ void add_pair(float& a, float& b, float x, float y) {
  asm("{\n\t.reg .b64 p, q;\n\tmov.b64 p, {%0, %1};\n\tmov.b64 q, {%2, %3};\n\tadd.rn.f32x2 p, p, q;\n\tmov.b64 {%0, %1}, p;\n\t}" : "+f"(a), "+f"(b) : "f"(x), "f"(y));
}
__device__ __forceinline__ uint32_t half_bits(float a, float b) { return pair_bits<__half>(a, b); }

__device__ __forceinline__ void mbar_inval(uint64_t* bar) { asm volatile("mbarrier.inval.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory"); }

// One warp's wait for its copy: bounded; one that runs out leaves a code for the host.
__device__ __forceinline__ bool kf_wait(uint64_t* bar, uint32_t parity, int* word) {
  if (mbar_try_wait(bar, parity)) return true;
#pragma unroll 1
  for (uint32_t i = 0; i < KF_WAIT_LIMIT; ++i)
    if (mbar_try_wait(bar, parity)) return true;
  wait_ran_out(word, 801);
  return false;
}

// Few queries a request: a block walks a range of one request's pages for one key head and a tile of columns (a column: one query of one of the heads
// that share the key head).  Warp w takes half w & 1 of every other page, 32 keys, through a ring and with references of its own; the four join at the end.
// CPL = 1: up to four columns, each of which has two of the product's eight, so that a lane has one column's scores and not those of columns that are
// not there (drafts of four tokens, 12 requests of up to 3000 keys, 40 heads: 35 us, with eight columns 39); CPL = 2: eight columns, and 16 with NB = 2.
// Weights enter the second product as fp16, half a place (2^-11) of which a bf16 result does not show; where the result is fp16 as two terms, with CPL = 1 the
// second one in the odd column.
template <int COLS, int STAGES>
struct KfShared {
  uint64_t full[KF_WARPS][STAGES];
  float ref[KF_WARPS][COLS], sum[KF_WARPS][COLS];
};
// Where a part's sums go: [parts there is room for][G][stride] of D sums, then of (reference, sum of weights), from column `at` of a walk's.
struct KfPart {
  float* part;
  int kept, stride, at;
};
// Columns col0 .. of an item's walk.  False where a wait ran out; every thread of the block calls.
template <typename T, int D, int NG, int CPL, int NB>
__device__ __forceinline__ bool few_walk(const Kv4Attn& a, const Kv4Item& it, int head, int col0, const KfPart to, uint8_t* smem,
                                         KfShared<4 * CPL * NB, kf_stages(D, NG)>& sh) {
  constexpr int W = D / 32, KS = D / 16, COLS = 4 * CPL * NB, BYTES = kv4_bytes(D, NG), SLICE = kv4_slice_bytes(D, NG), SPG = KS / NG, STAGES = kf_stages(D, NG);
  constexpr bool FINE = std::is_same<T, __half>::value;                  // the result keeps 11 bits
  constexpr int TERMS = CPL == 2 && FINE ? 2 : 1;
  const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31, R = a.H / a.G;
  const int first = it.first, n = it.count, row = it.row, cols = min(COLS, n * R - col0);
  T* y = (T*)a.y;
  const int pos0 = it.pos0;
  const int last = pos0 + column_token(col0 + cols - 1, R);                    // position of the tile's last column: keys up to here are in sight
  const int page0 = it.page0 + (warp >> 1), page1 = min(it.page1, last / KV4_PAGE + 1), half32 = 32 * (warp & 1);
  // the warp's pages: page0, page0 + 2 ..; the last one only where its half holds keys in sight
  const int units = page0 >= page1 ? 0 : (page1 - page0 + 1) / 2 - ((page0 + ((page1 - page0 - 1) & ~1)) * KV4_PAGE + half32 > last ? 1 : 0);
  const int32_t* table = a.table + (size_t)row * a.width + page0;
  uint8_t* ring = smem + warp * STAGES * 2 * SLICE;
  uint64_t* full = sh.full[warp];
  const uint8_t* from = a.blocks + (size_t)head * BYTES + (warp & 1) * 2 * SLICE;
  const size_t page_bytes = (size_t)a.G * BYTES;

  int entry = lane < units ? table[2 * lane] : 0;                       // the table's entries of 32 pages, a lane each
  if (lane == 0) {
    for (int i = 0; i < STAGES; ++i) mbar_init(&full[i], 1);
    fence_barrier_init();
  }
  __syncwarp();
#pragma unroll
  for (int i = 0; i < STAGES; ++i) {
    const int page = __shfl_sync(0xffffffffu, entry, i);
    if (lane == 0 && i < units) {
      mbar_expect_tx(&full[i], 2 * SLICE);
      bulk_load_1d(ring + i * 2 * SLICE, from + min(max(page, 0), a.pages - 1) * page_bytes, 2 * SLICE, &full[i]);
    }
  }

  float o[NB][KS][4];
  float ref[NB][CPL], sum[NB][CPL], sumlo[NB][NG][CPL];      // references in the products' units
  // About the largest product of a weight and a scale so far, whose power of two a column's sums over codes stand under: neither a scale that the column does
  // not weigh nor one that it does not see costs the others their bits.
  float most[NB][NG][CPL];
#pragma unroll
  for (int b = 0; b < NB; ++b) {
#pragma unroll
    for (int r = 0; r < KS; ++r) o[b][r][0] = o[b][r][1] = o[b][r][2] = o[b][r][3] = 0.f;
#pragma unroll
    for (int e = 0; e < CPL; ++e) {
      ref[b][e] = KV4_NONE;
      sum[b][e] = 0.f;
#pragma unroll
      for (int g = 0; g < NG; ++g) sumlo[b][g][e] = 0.f, most[b][g][e] = KF_LEAST;
    }
  }

  const int t4 = lane & 3, g8 = lane >> 2;
  // queries as the products' second operand: the product's column g8, dimensions 16 s + 4 t4 .. + 3; the largest of a column is brought to
  // 2^14 .. 2^15, the dimensions of odd nibbles are 16 times smaller
  uint32_t qb[NB][KS][2];
  float kq[NB][CPL], qn[NB][NG][CPL];
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    const int mine = CPL == 2 ? 8 * b + g8 : g8 >> 1, c = col0 + mine;
    const bool live = mine < cols && (CPL == 2 || (g8 & 1) == 0);
    const T* q = (const T*)a.q + (long long)(first + (live ? column_token(c, R) : 0)) * a.q_row + (size_t)(head * R + (live ? column_head(c, R) : 0)) * D;
    uint2 raw[KS];
    uint32_t big = 0;                                                   // sizes of numbers rise with their bits
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      raw[s] = live ? *reinterpret_cast<const uint2*>(q + 16 * s + 4 * t4) : make_uint2(0u, 0u);
      big = __vmaxu2(__vmaxu2(big, raw[s].x & 0x7fff7fffu), raw[s].y & 0x7fff7fffu);
    }
    big = __vmaxu2(big, __shfl_xor_sync(0xffffffffu, big, 1));
    big = __vmaxu2(big, __shfl_xor_sync(0xffffffffu, big, 2));
    const float2 mx2 = bits_pair<T>(big);
    const float mx = fmaxf(mx2.x, mx2.y);
    const int ex = min(max((int)(__float_as_uint(mx) >> 23), 15), 240);            // biased exponent of the largest
    const float up = __uint_as_float((uint32_t)(127 + 14 + 127 - ex) << 23);       // 2^(14 - (ex - 127))
    float gs[NG];
#pragma unroll
    for (int g = 0; g < NG; ++g) gs[g] = 0.f;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const float2 u = bits_pair<T>(raw[s].x), v = bits_pair<T>(raw[s].y);
      qb[b][s][0] = half_bits(u.x * up, u.y * up);
      qb[b][s][1] = half_bits(v.x * (up * 0.0625f), v.y * (up * 0.0625f));
      gs[s / SPG] += (u.x + u.y) + (v.x + v.y);
    }
    // 2^24 of the codes and 2^(ex - 127 - 14) of the queries, times the scores' scale in units of log2.  (Less than 1e-36 is what queries of nearly nothing
    // come to under a scale of nearly nothing: scores of 0 either way.)
    const float back = fmaxf(__uint_as_float((uint32_t)(ex - 14 + 24) << 23) * (a.scale * KF_LOG2E), 1e-36f);      // (masked scores are -inf, and a first one is more than KF_SLACK from KV4_NONE)
#pragma unroll
    for (int e = 0; e < CPL; ++e) kq[b][e] = __shfl_sync(0xffffffffu, back, 4 * (2 * t4 + e));
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      gs[g] += __shfl_xor_sync(0xffffffffu, gs[g], 1);
      gs[g] += __shfl_xor_sync(0xffffffffu, gs[g], 2);
#pragma unroll
      for (int e = 0; e < CPL; ++e) qn[b][g][e] = __shfl_sync(0xffffffffu, gs[g] * (up * 5.9604644775390625e-8f), 4 * (2 * t4 + e));      // (2^-24)
    }
  }
  const int first_pos = pos0 + column_token(col0, R);                              // every column sees the keys up to here

  bool ok = true;
  int st = 0;
  uint32_t parity = 0;
#pragma unroll 1
  for (int i = 0; i < units; ++i) {
    ok = __all_sync(0xffffffffu, kf_wait(&full[st], parity, a.word));
    if (!ok) break;
    const uint8_t* const unit = ring + st * 2 * SLICE;
    const int j = (page0 + 2 * i) * KV4_PAGE + half32 + g8;             // the lane's keys: j, j + 8, j + 16, j + 24
    // scores, in the products' units
    float s[4][NB][CPL];
    float2 pv[4][NG];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint8_t* const blk = unit + h * SLICE;
      uint32_t kw[2][W], kp[2][NG], vp[2][NG];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        lds_words<W>(kw[x], blk + (g8 + 8 * x) * (D / 2) + t4 * 4 * W);
        lds_words<NG>(kp[x], blk + kv4_k_params(D) + (g8 + 8 * x) * NG * 4);
        lds_words<NG>(vp[x], blk + kv4_v_params(D, NG) + (g8 + 8 * x) * NG * 4);
      }
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        float acc[NB][4];
#pragma unroll
        for (int b = 0; b < NB; ++b) acc[b][0] = acc[b][1] = acc[b][2] = acc[b][3] = 0.f;
#pragma unroll
        for (int e = 0; e < SPG; ++e) {
          const int k = g * SPG + e;
          const uint32_t w0 = (k & 1) ? kw[0][k >> 1] >> 8 : kw[0][k >> 1], w1 = (k & 1) ? kw[1][k >> 1] >> 8 : kw[1][k >> 1];
#pragma unroll
          for (int b = 0; b < NB; ++b)
            mma_f16_16816(acc[b], w0 & 0x000f000fu, w1 & 0x000f000fu, w0 & 0x00f000f0u, w1 & 0x00f000f0u, qb[b][k][0], qb[b][k][1]);
        }
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const float2 p = bits_pair<T>(kp[x][g]);
          pv[2 * h + x][g] = bits_pair<T>(vp[x][g]);
#pragma unroll
          for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int e = 0; e < CPL; ++e)
              s[2 * h + x][b][e] = fmaf(p.x, acc[b][2 * x + e], g == 0 ? p.y * qn[b][g][e] : fmaf(p.y, qn[b][g][e], s[2 * h + x][b][e]));
        }
      }
    }
    // which keys a column sees: all of them but at the end of its walk, where a slot behind the last key may hold anything
    bool none = false;                                                  // whether the unit's values have to be looked at one by one
    if (j - g8 + 31 > first_pos) {
#pragma unroll
      for (int x = 0; x < 4; ++x) {
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
          for (int e = 0; e < CPL; ++e)
            if (j + 8 * x > pos0 + column_token(min(col0 + 8 * b + CPL * t4 + e, col0 + cols - 1), R)) s[x][b][e] = -INFINITY;
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          if (j + 8 * x > last) pv[x][g] = make_float2(0.f, 0.f);
          none |= isnan(pv[x][g].y);
        }
      }
      none = __any_sync(0xffffffffu, none);                             // (a value that is none, maybe behind a column: 0 * NaN)
    }
    // do references have to move, or what the sums stand under?
    bool grow = false;
    float top[NG];                                                      // the largest scale of the lane's keys
#pragma unroll
    for (int g = 0; g < NG; ++g) top[g] = fmaxf(fmaxf(pv[0][g].x, pv[1][g].x), fmaxf(pv[2][g].x, pv[3][g].x));
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int e = 0; e < CPL; ++e) {
        grow |= (fmaxf(fmaxf(s[0][b][e], s[1][b][e]), fmaxf(s[2][b][e], s[3][b][e])) - ref[b][e]) * kq[b][e] > KF_SLACK;
#pragma unroll
        for (int g = 0; g < NG; ++g) grow |= top[g] * one_over_pow2(most[b][g][e]) > KF_SCALES;
      }
    if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int e = 0; e < CPL; ++e) {
          float m = fmaxf(fmaxf(s[0][b][e], s[1][b][e]), fmaxf(s[2][b][e], s[3][b][e]));
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
          m = fmaxf(m, ref[b][e]);
          const float fe = kf_exp2((ref[b][e] - m) * kq[b][e]);
          ref[b][e] = m;
          sum[b][e] *= fe;
#pragma unroll
          for (int g = 0; g < NG; ++g) {
            sumlo[b][g][e] *= fe;
            // the largest product of the 32 keys (one that is none is passed over: such a group's results are none whatever they stand under) and the
            // largest scale: what a column's lanes agree on.  Up to four times the largest product, where the scales are within bounds then.
            float now = 0.f, scale = top[g];
#pragma unroll
            for (int x = 0; x < 4; ++x) now = fmaxf(now, kf_exp2((s[x][b][e] - m) * kq[b][e]) * pv[x][g].x);
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) now = fmaxf(now, __shfl_xor_sync(0xffffffffu, now, d)), scale = fmaxf(scale, __shfl_xor_sync(0xffffffffu, scale, d));
            now = fmaxf(most[b][g][e] * fe, fmaxf(now, fminf(4.f * now, scale * (1.f / KF_SCALES))));
            now = fminf(fmaxf(now, KF_LEAST), 1.f / KF_LEAST);
            const float f = fe * pow2_of(most[b][g][e]) * one_over_pow2(now);
            most[b][g][e] = now;
            none |= scale * one_over_pow2(now) > KF_SCALES;
#pragma unroll
            for (int r = 0; r < SPG; ++r) {
              o[b][g * SPG + r][e] *= f, o[b][g * SPG + r][2 + e] *= f;
              if (CPL == 1) o[b][g * SPG + r][1] *= f, o[b][g * SPG + r][3] *= f;
            }
          }
        }
      none = __any_sync(0xffffffffu, none);                             // (a scale that a column does not weigh: its product is taken before it is brought under E)
    }
    // weights (the difference first: of scores past 2^27 a product and a rounded one of the same numbers are too far apart)
#pragma unroll
    for (int x = 0; x < 4; ++x)
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int e = 0; e < CPL; ++e) {
          s[x][b][e] = kf_exp2((s[x][b][e] - ref[b][e]) * kq[b][e]);
          sum[b][e] += s[x][b][e];
        }
    // y += (p s) c, p lo: by groups, p s under what the column's sums stand under, and so under 2^15.  Of a word's nibbles 0 and 1 (2 and 3) the rows of
    // the second tile half take both as they stand, c + 16 c': the end takes c from it.  Where the result is fp16, the sums of
    // 16 keys are added in fp32, and codes are four times as large: the tensor pipe cuts products off two bits below the last one of the sum that they join, and
    // those of a subnormal number as if it were the smallest normal one.  (130 000 keys of like weights, whose values leave a 40th of a scale: 0.00021 of
    // the norm off, as a rounded exact result is, instead of 0.00028 with the sums around code 8 in the pipe, which also took 45 us instead of 40; eight columns
    // 0.00022 instead of 0.00066 around code 0, 60 us instead of 58.)
    auto add_values = [&](auto careful) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t vw[2][W];
#pragma unroll
        for (int x = 0; x < 2; ++x) lds_words<W>(vw[x], unit + h * SLICE + kv4_v_codes(D) + (t4 + 4 * x) * D + g8 * 4 * W);
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          uint32_t bw[NB][TERMS][2];
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const float2 p = pv[2 * h + x][g];
#pragma unroll
            for (int b = 0; b < NB; ++b) {
              float w[2] = {0.f, 0.f};
#pragma unroll
              for (int e = 0; e < CPL; ++e) {
                const float pe = s[2 * h + x][b][e];
                w[e] = careful.value ? pe * p.x * one_over_pow2(most[b][g][e]) : pe * (p.x * one_over_pow2(most[b][g][e]));
                if (careful.value && pe == 0.f) w[e] = 0.f;
                else sumlo[b][g][e] = fmaf(pe, p.y, sumlo[b][g][e]);
              }
              if (CPL == 1) {
                if (FINE) {                                             // the odd column: what 11 bits leave over
                  const float hi = __uint_as_float(__float_as_uint(w[0]) & 0xffffe000u);
                  w[1] = w[0] - hi;
                  w[0] = hi;
                }
                bw[b][0][x] = movmatrix(half_bits(w[0], w[1]));
              } else {
                const uint32_t hi = half_bits(w[0], w[1]);
                bw[b][0][x] = movmatrix(hi);
                if (TERMS == 2) {
                  const float2 f = bits_pair<__half>(hi);
                  bw[b][TERMS - 1][x] = movmatrix(half_bits(w[0] - f.x, w[1] - f.y));
                }
              }
            }
          }
#pragma unroll
          for (int e = 0; e < SPG; ++e) {
            const int r = g * SPG + e;
            auto codes = [](uint32_t w, bool upper) {
              if (FINE) return (upper ? w >> 6 : w << 2) & 0x03fc03fcu;
              return upper ? __byte_perm(w, 0u, 0x4341) : w & 0x00ff00ffu;
            };
            constexpr uint32_t LOW = FINE ? 0x003c003cu : 0x000f000fu;
            const uint32_t w0 = codes(vw[0][r >> 1], (r & 1) != 0), w1 = codes(vw[1][r >> 1], (r & 1) != 0);
#pragma unroll
            for (int b = 0; b < NB; ++b) {
              float t[4] = {0.f, 0.f, 0.f, 0.f};
              float (&sums)[4] = FINE ? t : o[b][r];
#pragma unroll
              for (int x = 0; x < TERMS; ++x) mma_f16_16816(sums, w0 & LOW, w0, w1 & LOW, w1, bw[b][x][0], bw[b][x][1]);
              if (FINE)
#pragma unroll
                for (int x = 0; x < 4; x += 2) add_pair(o[b][r][x], o[b][r][x + 1], t[x], t[x + 1]);
            }
          }
        }
      }
    };
    if (none) add_values(std::true_type());
    else add_values(std::false_type());
    // the next 32 keys for this place of the ring
    const int nxt = i + STAGES;
    if ((nxt & 31) == 0) entry = nxt + lane < units ? table[2 * (nxt + lane)] : 0;
    const int page = __shfl_sync(0xffffffffu, entry, nxt & 31);
    __syncwarp();                                                       // every lane has read the unit
    if (lane == 0 && nxt < units) {
      mbar_expect_tx(&full[st], 2 * SLICE);
      bulk_load_1d(ring + st * 2 * SLICE, from + min(max(page, 0), a.pages - 1) * page_bytes, 2 * SLICE, &full[st]);
    }
    if (++st == STAGES) st = 0, parity ^= 1;
  }
  if (!ok) kv4_let_end();                                               // copies that were asked for end before the block does
  // a column's sums over the lanes that share it
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int e = 0; e < CPL; ++e)
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) {
        sum[b][e] += __shfl_xor_sync(0xffffffffu, sum[b][e], d);
#pragma unroll
        for (int g = 0; g < NG; ++g) sumlo[b][g][e] += __shfl_xor_sync(0xffffffffu, sumlo[b][g][e], d);
      }
  if (g8 == 0)
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int e = 0; e < CPL; ++e) sh.ref[warp][8 * b + CPL * t4 + e] = ref[b][e] == KV4_NONE ? KV4_NONE : ref[b][e] * kq[b][e], sh.sum[warp][8 * b + CPL * t4 + e] = sum[b][e];
  if (__syncthreads_or(!ok)) return false;    // every unit has been read: the rings hold the warps' sums now
  pdl_launch_dependents();
  float* so = reinterpret_cast<float*>(smem);                           // [warp][column][D + 4]
  constexpr int LD = D + 4;
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int r = 0; r < KS; ++r) {
#pragma unroll
      for (int e = 0; e < CPL; ++e) {                                   // (codes were 2^-24 of themselves, or 2^-22)
        const float up = pow2_of(most[b][r / SPG][e]);
        const float c = CPL == 2 ? o[b][r][e] : o[b][r][0] + o[b][r][1], both = CPL == 2 ? o[b][r][2 + e] : o[b][r][2] + o[b][r][3];
        float* const at = so + (warp * COLS + 8 * b + CPL * t4 + e) * LD + 16 * r + g8;
        at[0] = fmaf(c * (FINE ? 4194304.f : 16777216.f), up, sumlo[b][r / SPG][e]);
        at[8] = fmaf((both - c) * (FINE ? 262144.f : 1048576.f), up, sumlo[b][r / SPG][e]);
      }
    }
  __syncthreads();
  // the four warps' parts; the block's are stored as they are, or as the result where there is no other part
#pragma unroll 1
  for (int x = threadIdx.x; x < cols * (D / 4); x += KF_THREADS) {
    const int c = x / (D / 4), d = x % (D / 4) * 4;
    float m = sh.ref[0][c];
#pragma unroll
    for (int w = 1; w < KF_WARPS; ++w) m = fmaxf(m, sh.ref[w][c]);
    float l = 0.f, v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < KF_WARPS; ++w) {
      const float f = kf_exp2(sh.ref[w][c] - m);
      const float4 u = *reinterpret_cast<const float4*>(so + (w * COLS + c) * LD + d);
      l = fmaf(sh.sum[w][c], f, l);
      v[0] = fmaf(u.x, f, v[0]), v[1] = fmaf(u.y, f, v[1]), v[2] = fmaf(u.z, f, v[2]), v[3] = fmaf(u.w, f, v[3]);
    }
    if (it.parts == 1) {
      const int cc = col0 + c;
      const uint2 out = make_uint2(pair_bits<T>(v[0] / l, v[1] / l), pair_bits<T>(v[2] / l, v[3] / l));
      *reinterpret_cast<uint2*>(y + ((size_t)(first + column_token(cc, R)) * a.H + head * R + column_head(cc, R)) * D + d) = out;
    } else {
      const size_t at = ((size_t)(it.base + it.part) * a.G + head) * to.stride + to.at + c;
      *reinterpret_cast<float4*>(to.part + at * D + d) = make_float4(v[0], v[1], v[2], v[3]);
      if (d == 0) *reinterpret_cast<float2*>(to.part + (size_t)to.kept * a.G * to.stride * D + at * 2) = make_float2(m, l);
    }
  }
  return true;
}

// A block an item and key head of the list `a`.  BESIDE a list `m` of the many there are blocks more, which go through the tiles that kv4_prompt_kernel has
// left (groups that fp16 numbers do not hold), KV4_FEW_BESIDE columns at a time.  (A kernel of its own: with that walk in it too, twelve drafts of eight tokens
// took 37 us instead of 36.)
template <typename T, int D, int NG, int CPL, int NB, bool BESIDE>
__global__ void __launch_bounds__(KF_THREADS, NB == 1 ? 4 : 2) kv4_few_kernel(const Kv4Attn a, const Kv4Attn m) {
  constexpr int COLS = 4 * CPL * NB;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ KfShared<COLS, kf_stages(D, NG)> sh;
  // (launched when the last blocks of the prompts' kernel of the same call run: what is read here was there before that one.  The last block ends after
  // it, so that what waits for this kernel waits for both.)
  if (blockIdx.x == gridDim.x - 1) pdl_wait();
  const int R = a.H / a.G, blocks = a.items * a.G;
  if constexpr (BESIDE) {
    if ((int)blockIdx.x >= blocks) {      // (what these read the prompts' kernel has left)
      constexpr int SUBS = KV4_MANY / COLS;
      __shared__ uint32_t s_left[KF_WARPS];
      pdl_launch_dependents();
      pdl_wait();
      const int again = gridDim.x - blocks;
      const int32_t* work = after_wait(m.work);
      const int* odd = after_wait(m.odd);
      const long long units = (long long)min(work[0], m.items) * a.G * SUBS;
#pragma unroll 1
      for (long long u0 = blockIdx.x - blocks; u0 < units; u0 += (long long)again * KF_THREADS) {
        const long long mine = u0 + (long long)again * threadIdx.x;
        const uint32_t left = __ballot_sync(0xffffffffu, mine < units && (odd[mine / SUBS] >> (mine % SUBS / (SUBS / 2)) & 1) != 0);
        __syncthreads();
        if ((threadIdx.x & 31) == 0) s_left[threadIdx.x >> 5] = left;
        __syncthreads();
#pragma unroll 1
        for (int w = 0; w < KF_WARPS; ++w)
#pragma unroll 1
          for (uint32_t bits = s_left[w]; bits != 0u; bits &= bits - 1) {
            const long long unit = u0 + (long long)again * (32 * w + __ffs(bits) - 1);
            const int block = (int)(unit / SUBS), item = block / a.G, head = block - item * a.G, at = (int)(unit % SUBS) * COLS;
            const Kv4Item it = load_item(work, item);
            const int col0 = it.tile * KV4_MANY + at;
            if (col0 >= it.count * R) continue;
            if (!few_walk<T, D, NG, CPL, NB>(a, it, head, col0, KfPart{m.part, m.kept, KV4_MANY, at}, smem, sh)) return;
            fence_proxy_async();                                        // (the rings' memory has been written and read by threads: copies come next)
            __syncthreads();
            if ((threadIdx.x & 31) == 0)
              for (int i = 0; i < kf_stages(D, NG); ++i) mbar_inval(&sh.full[threadIdx.x >> 5][i]);
            __syncwarp();
          }
      }
      return;
    }
  }
  const int item = blockIdx.x / a.G, head = blockIdx.x - item * a.G;
  const Kv4Item it = load_item(a.work, item);                           // (there is room for it: asked for together with the number of parts)
  if (item >= a.work[0]) return;
  const int col0 = it.tile * COLS;
  if (it.row < 0) {                     // a refused sequence's tokens are no numbers
    const int cols = min(COLS, it.count * R - col0);
#pragma unroll 1
    for (int e = threadIdx.x; e < cols * D; e += KF_THREADS) {
      const int c = col0 + e / D;
      dt<T>::st((T*)a.y, ((size_t)(it.first + column_token(c, R)) * a.H + head * R + column_head(c, R)) * D + e % D, NAN);
    }
    return;
  }
  few_walk<T, D, NG, CPL, NB>(a, it, head, col0, KfPart{a.part, a.kept, COLS, 0}, smem, sh);
}

// Joins the parts of walks.  Of the few columns a block has one at a time, a warp every KJ-th part (a long walk is in hundreds of parts); of the
// tcgen05 kernel's tiles a warp has one (these are in a few).
constexpr int KJ = 8;
template <int D>
struct KjSum {
  float m = KV4_NONE, l = 0.f, o[D / 32] = {};
  __device__ __forceinline__ void add(float2 u, const float* part, int lane) {      // u: reference and sum of weights
    if (u.y == 0.f) return;                    // (a part that holds no key of the column's)
    const float mn = fmaxf(m, u.x), f = kf_exp2(m - mn), w = kf_exp2(u.x - mn);
    m = mn;
    l = fmaf(l, f, u.y * w);
#pragma unroll
    for (int e = 0; e < D / 32; ++e) o[e] = fmaf(o[e], f, part[lane + 32 * e] * w);
  }
};
template <typename T, int D, int COLS>
__global__ void __launch_bounds__(KJ * 32) kv4_join_kernel(const Kv4Attn few, const Kv4Attn many) {
  __shared__ float s_m[KJ], s_l[KJ], s_o[KJ][D];
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, G = few.G, R = few.H / few.G;
  T* const y = (T*)few.y;
  if (few.items > 0) {
    const int32_t* work = after_wait(few.work);
    const float* part = after_wait(few.part);
    const float2* ml = reinterpret_cast<const float2*>(part + (size_t)few.kept * G * COLS * D);
    const int units = work[1] * G * few.cols;
    for (int u = blockIdx.x; u < units; u += gridDim.x) {
      const int j = u / (G * few.cols), head = u / few.cols % G, c = u % few.cols;
      const int4 a = joins_of(work, few.items)[2 * j], b = joins_of(work, few.items)[2 * j + 1];
      const int first = a.x, col = a.z * COLS + c, parts = a.w;
      if (col >= a.y * R) continue;
      KjSum<D> s;
#pragma unroll 4
      for (int k = warp; k < parts; k += KJ) {
        const size_t at = ((size_t)(b.x + k) * G + head) * COLS + c;
        s.add(ml[at], part + at * D, lane);
      }
      __syncthreads();                         // (the unit before this one has been read)
      if (lane == 0) s_m[warp] = s.m, s_l[warp] = s.l;
#pragma unroll
      for (int e = 0; e < D / 32; ++e) s_o[warp][lane + 32 * e] = s.o[e];
      __syncthreads();
      const int d = threadIdx.x;
      if (d < D) {
        float m = s_m[0], num = 0.f, den = 0.f;
#pragma unroll
        for (int w = 1; w < KJ; ++w) m = fmaxf(m, s_m[w]);
#pragma unroll
        for (int w = 0; w < KJ; ++w) {
          const float f = kf_exp2(s_m[w] - m);
          num = fmaf(s_o[w][d], f, num);
          den = fmaf(s_l[w], f, den);
        }
        dt<T>::st(y, ((size_t)(first + column_token(col, R)) * few.H + head * R + column_head(col, R)) * D + d, num / den);
      }
    }
  }
  if (many.items > 0) {
    const int32_t* work = after_wait(many.work);
    const float* part = after_wait(many.part);
    const float2* ml = reinterpret_cast<const float2*>(part + (size_t)many.kept * G * KV4_MANY * D);
    const int units = work[1] * G * (KV4_MANY / KJ);
    for (int u = blockIdx.x; u < units; u += gridDim.x) {
      const int j = u / (G * (KV4_MANY / KJ)), head = u / (KV4_MANY / KJ) % G, c = u % (KV4_MANY / KJ) * KJ + warp;
      const int4 a = joins_of(work, many.items)[2 * j], b = joins_of(work, many.items)[2 * j + 1];
      const int first = a.x, col = a.z * KV4_MANY + c, parts = a.w;
      if (col >= a.y * R) continue;
      KjSum<D> s;
#pragma unroll 2
      for (int k = 0; k < parts; ++k) {
        const size_t at = ((size_t)(b.x + k) * G + head) * KV4_MANY + c;
        s.add(ml[at], part + at * D, lane);
      }
#pragma unroll
      for (int e = 0; e < D / 32; ++e)
        dt<T>::st(y, ((size_t)(first + column_token(col, R)) * few.H + head * R + column_head(col, R)) * D + lane + 32 * e, s.o[e] / s.l);
    }
  }
}

}  // namespace
}  // namespace llb

using namespace llb;

extern "C" {

size_t ll_kv4_attn_scratch_bytes(const ll_kv4_cache* cache, int B, int T, int max_count) {
  if (!kv4_step_ok(cache, B, T, max_count)) return 0;
  return Kv4Lists(B, T, max_count, cache->heads, cache->kv_heads, cache->max_length).bytes(cache->kv_heads, cache->head_size);
}

int ll_kv4_attn(const ll_kv4_cache* cache, const void* blocks, const void* q, long long q_row, const int32_t* work, void* y, int B, int T, int max_count,
                float scale, void* scratch, ll_stream stream) {
  LL_CHECK_ARG(cache != nullptr, "kv4_attn: no cache");
  const int dtype = cache->dtype, H = cache->heads, G = cache->kv_heads, head_size = cache->head_size, group = cache->group;
  LL_CHECK_ARG(kv4_shape_ok(head_size, group), "kv4_attn: heads of %d in groups of %d (32, 64 or 128 each)", head_size, group);
  LL_CHECK_ARG(dtype == LL_BF16 || dtype == LL_F16, "kv4_attn: type %d (bf16 or fp16)", dtype);
  LL_CHECK_ARG(q && blocks && cache->table && work && y && scratch && B > 0 && T > 0 && max_count >= 0 && G > 0 && G <= 65535 && H > 0 && H % G == 0 && cache->width > 0 &&
                   cache->pages > 0 && cache->max_length > 0 && (long long)T * H <= INT_MAX,
               "kv4_attn: %d tokens of %d heads, %d cached", T, H, G);
  LL_CHECK_ARG(scale > 0.f && scale < INFINITY, "kv4_attn: scores times %g (more than 0, and a number of 32 bits)", scale);
  LL_CHECK_ARG((((uintptr_t)q | (uintptr_t)y | (uintptr_t)blocks | (uintptr_t)scratch | (uintptr_t)work) & 15) == 0 && q_row % 8 == 0,
               "kv4_attn: rows have to start on 16-byte boundaries");
  const Kv4Lists l(B, T, max_count, H, G, cache->max_length);
  LL_CHECK_ARG(l.few_items * G <= INT_MAX && l.many_items * G <= INT_MAX, "kv4_attn: %d sequences of %d tokens, %d heads", B, T, H);
  const int R = l.R, cols = l.cols, used = (int)std::min((long long)cols, (long long)max_count * R);
  const Kv4Attn a{q, q_row, (const uint8_t*)blocks, cache->table, work, y, (float*)scratch, H, G, cache->width, cache->pages, (int)l.few_items, l.few_kept(), used, scale,
                  wait_word(), nullptr};
  Kv4Attn m = a;
  m.items = 0;
  cudaStream_t st = (cudaStream_t)stream;
  if (l.many) {
    m.work = work + l.few_ints();
    m.part = (float*)scratch + l.few_floats(G, head_size);
    m.odd = (int*)(m.part + l.many_floats(G, head_size));
    m.items = (int)l.many_items;
    m.kept = l.many_kept();
    if (int r = kv4_prompt_launch(m, dtype, head_size, group, st)) return r;
  }
  // The sequences of few columns fill the end of the prompts' kernel, which lets them in when it has begun.  The join waits for both (kv4_few_kernel's last blocks).
  // (None where walks are not cut, or where no sequence may bring a token: then all that bring some are refused.)
  const unsigned join_blocks =
      l.few_cut || l.many ? (unsigned)std::min<long long>(4ll * kv4_sms(), (long long)l.few_joins() * G * used + (l.many ? (long long)l.many_joins() * G * (KV4_MANY / KJ) : 0)) : 0;
  LL_CHECK_ARG(l.few_items * G + 4ll * kv4_sms() <= INT_MAX, "kv4_attn: %d sequences of %d tokens, %d heads", B, T, H);
  const unsigned few_blocks = (unsigned)(l.few_items * G) + (l.many ? 4u * kv4_sms() : 0u);
#define FEW(TT, DD, NG, CPL, NB, BESIDE)                                                                                                      \
  {                                                                                                                                           \
    static_assert(!BESIDE || 4 * CPL * NB == KV4_FEW_BESIDE, "columns beside the many");                                                      \
    constexpr int COLS = 4 * CPL * NB, ring = KF_WARPS * kf_stages(DD, NG) * 2 * kv4_slice_bytes(DD, NG), join = KF_WARPS * COLS * (DD + 4) * 4; \
    constexpr int smem = ring > join ? ring : join;                                                                                           \
    static PerDevice set;                                                                                                                     \
    if (!set) {                                                                                                                               \
      LL_CUDA(cudaFuncSetAttribute(kv4_few_kernel<TT, DD, NG, CPL, NB, BESIDE>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));                  \
      prefer_max_smem(kv4_few_kernel<TT, DD, NG, CPL, NB, BESIDE>);                                                                                   \
      set.mark();                                                                                                                             \
    }                                                                                                                                         \
    LL_CUDA(launch(kv4_few_kernel<TT, DD, NG, CPL, NB, BESIDE>, dim3(few_blocks), dim3(KF_THREADS), smem, st, l.many, a, m));           \
    LL_LAUNCH_OK("kv4_few_kernel");                                                                                                           \
    if (join_blocks > 0) LL_CUDA(launch(kv4_join_kernel<TT, DD, COLS>, dim3(join_blocks), dim3(KJ * 32), 0, st, true, a, m));                          \
  }
#define FEW_COLS(TT, DD, NG)                          \
  if (l.many) FEW(TT, DD, NG, 2, 1, true)             \
  else if (cols == 4) FEW(TT, DD, NG, 1, 1, false)    \
  else if (cols == 8) FEW(TT, DD, NG, 2, 1, false)    \
  else FEW(TT, DD, NG, 2, 2, false)
#define ATTN(DD, NG)                                      \
  if (dtype == LL_BF16) { FEW_COLS(__nv_bfloat16, DD, NG) } \
  else { FEW_COLS(__half, DD, NG) }
  KV4_SHAPES(head_size, group, ATTN)
#undef ATTN
#undef FEW_COLS
#undef FEW
  LL_LAUNCH_OK("kv4_join_kernel");
  return LL_OK;
}

}  // extern "C"
