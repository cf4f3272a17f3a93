// Softmax attention over the paged key/value cache in 4 bits (kv4.cuh): a step's tokens, of requests of unequal lengths, over the keys at and before
// their positions.
//
// With K = s c + lo and V alike, by groups of a head's dimensions (c: codes),
//   q.k_j = sum_g s_jg (q.c_j)_g + lo_jg (sum of q)_g           y = sum_j p_j v_j = sum_j (p_j s_jg) c_j + sum_j p_j lo_jg
// so that the products run over codes, which a mask turns into numbers of fp16 (subnormal ones, exactly), and scales meet 16 keys at a time.
#include <type_traits>

#include "kv4.cuh"

namespace llb {
namespace {

struct Kv4Attn {
  const void* q;
  long long q_row;
  const uint8_t* blocks;
  const int32_t *table, *starts, *ends, *request, *work;
  void* y;
  float* part;         // [items][G][COLS] of D sums, then [items][G][COLS] of (reference, sum of weights)
  int H, G, width, pages, B, max_items;
  float scale;
  int* word;           // wait_word()
};

constexpr int KF_WARPS = 4, KF_THREADS = KF_WARPS * 32, KF_STAGES = 4;
constexpr float KF_LOG2E = 1.4426950408889634f, KF_SLACK = 8.f;      // a column's scores may outgrow its reference by 2^8 before it moves
constexpr float KF_NONE = -1e37f;                                       // the reference of a column that has seen no key
constexpr uint32_t KF_WAIT_LIMIT = 1u << 20;

__device__ __forceinline__ float kf_exp2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
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
template <int W> __device__ __forceinline__ void lds_words(uint32_t (&w)[W], const uint8_t* p) {
  if constexpr (W == 4) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    w[0] = u.x, w[1] = u.y, w[2] = u.z, w[3] = u.w;
  } else if constexpr (W == 2) {
    const uint2 u = *reinterpret_cast<const uint2*>(p);
    w[0] = u.x, w[1] = u.y;
  } else {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  }
}
__device__ __forceinline__ uint32_t half_bits(float a, float b) { return pair_bits<__half>(a, b); }

// One warp's wait for its copy: bounded; one that runs out leaves a code for the host.
__device__ __forceinline__ bool kf_wait(uint64_t* bar, uint32_t parity, int* word) {
  if (mbar_try_wait(bar, parity)) return true;
  for (uint32_t i = 0; i < KF_WAIT_LIMIT; ++i)
    if (mbar_try_wait(bar, parity)) return true;
  wait_ran_out(word, 701);
  return false;
}

// Few queries a request: a block walks a range of one request's pages for one key head and up to 8 NB columns (a column: one query of one of the heads
// that share the key head).  Each of its four warps takes a slice of 16 keys of every page through a ring of its own, with references of its own; they
// join at the end.
// Weights enter the second product as fp16 (TERMS 1), or as two such terms where the result is fp16, too.
template <typename T, int D, int NG, int NB>
__global__ void __launch_bounds__(KF_THREADS, NB == 1 ? 4 : 2) kv4_few_kernel(const Kv4Attn a) {
  constexpr int W = D / 32, KS = D / 16, COLS = 8 * NB, BYTES = kv4_bytes(D, NG), SLICE = kv4_slice_bytes(D, NG), SPG = KS / NG;
  constexpr int TERMS = std::is_same<T, __half>::value ? 2 : 1;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint64_t s_full[KF_WARPS][KF_STAGES];
  __shared__ int s_fail;
  __shared__ float s_ref[KF_WARPS][COLS], s_sum[KF_WARPS][COLS];
  const int item = blockIdx.x, head = blockIdx.y;
  if (item >= a.work[0]) return;
  const int4 it = reinterpret_cast<const int4*>(a.work)[1 + item];      // sequence, tile of columns, part, parts
  const int step = a.work[1], warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31, R = a.H / a.G;
  const int seq = it.x, first = a.starts[seq], n = a.starts[seq + 1] - first, row = a.request[seq];
  const int col0 = it.y * COLS, cols = min(COLS, n * R - col0);
  T* y = (T*)a.y;
  if (row < 0) {                        // a refused sequence's tokens are no numbers
    for (int e = threadIdx.x; e < cols * D; e += KF_THREADS) {
      const int c = col0 + e / D;
      dt<T>::st(y, ((size_t)(first + c / R) * a.H + head * R + c % R) * D + e % D, NAN);
    }
    return;
  }
  const int pos0 = a.ends[seq] - n;                                     // position of the sequence's first token
  const int last = pos0 + (col0 + cols - 1) / R;                        // position of the tile's last column: keys up to here are in sight
  const int page0 = it.z * step, pages = min(page0 + step, last / KV4_PAGE + 1) - page0;
  // the warp's slices: of the last page only what holds keys in sight
  const int slices = pages <= 0 ? 0 : pages - ((page0 + pages - 1) * KV4_PAGE + 16 * warp > last ? 1 : 0);
  const int32_t* table = a.table + (size_t)row * a.width + page0;
  uint8_t* ring = smem + warp * KF_STAGES * SLICE;
  uint64_t* full = s_full[warp];
  const uint8_t* from = a.blocks + (size_t)head * BYTES + warp * SLICE;
  const size_t page_bytes = (size_t)a.G * BYTES;

  int entry = lane < slices ? table[lane] : 0;                          // the table's entries of 32 pages, a lane each
  if (threadIdx.x == 0) s_fail = 0;
  if (lane == 0) {
    for (int i = 0; i < KF_STAGES; ++i) mbar_init(&full[i], 1);
    fence_barrier_init();
  }
  __syncwarp();
#pragma unroll
  for (int i = 0; i < KF_STAGES; ++i) {
    const int page = __shfl_sync(0xffffffffu, entry, i);
    if (lane == 0 && i < slices) {
      mbar_expect_tx(&full[i], SLICE);
      bulk_load_1d(ring + i * SLICE, from + min(max(page, 0), a.pages - 1) * page_bytes, SLICE, &full[i]);
    }
  }

  float o[NB][KS][4];
  float ref[NB][2], sum[NB][2], sumlo[NB][NG][2];      // references in units of log2
  uint32_t ev[NG];                                     // exponents of the values' scales so far, as powers of two's bits
#pragma unroll
  for (int b = 0; b < NB; ++b) {
#pragma unroll
    for (int r = 0; r < KS; ++r) o[b][r][0] = o[b][r][1] = o[b][r][2] = o[b][r][3] = 0.f;
    ref[b][0] = ref[b][1] = KF_NONE;
    sum[b][0] = sum[b][1] = 0.f;
#pragma unroll
    for (int g = 0; g < NG; ++g) sumlo[b][g][0] = sumlo[b][g][1] = 0.f;
  }
#pragma unroll
  for (int g = 0; g < NG; ++g) ev[g] = 1u << 23;

  const int t4 = lane & 3, g8 = lane >> 2;
  // queries as the products' second operand: column g8, dimensions 16 s + 4 t4 .. + 3; the largest of a column is brought to 2^14 .. 2^15, the
  // dimensions of odd nibbles are 16 times smaller
  uint32_t qb[NB][KS][2];
  float kq[NB][2], qn[NB][NG][2];
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    const int c = col0 + 8 * b + g8;
    const bool live = 8 * b + g8 < cols;
    const T* q = (const T*)a.q + (long long)(first + (live ? c / R : 0)) * a.q_row + (size_t)(head * R + (live ? c % R : 0)) * D;
    uint2 raw[KS];
    float mx = 0.f;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      raw[s] = live ? *reinterpret_cast<const uint2*>(q + 16 * s + 4 * t4) : make_uint2(0u, 0u);
      const float2 u = bits_pair<T>(raw[s].x), v = bits_pair<T>(raw[s].y);
      mx = fmaxf(fmaxf(mx, fmaxf(fabsf(u.x), fabsf(u.y))), fmaxf(fabsf(v.x), fabsf(v.y)));
    }
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
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
      const float2 x = bits_pair<__half>(qb[b][s][0]), z = bits_pair<__half>(qb[b][s][1]);
      gs[s / SPG] += (x.x + x.y) + 16.f * (z.x + z.y);
    }
    // 2^24 of the codes and 2^(ex - 127 - 14) of the queries, times the scores' scale in units of log2
    const float back = __uint_as_float((uint32_t)(ex - 14 + 24) << 23) * (a.scale * KF_LOG2E);
#pragma unroll
    for (int e = 0; e < 2; ++e) kq[b][e] = __shfl_sync(0xffffffffu, back, 4 * (2 * t4 + e));
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      gs[g] += __shfl_xor_sync(0xffffffffu, gs[g], 1);
      gs[g] += __shfl_xor_sync(0xffffffffu, gs[g], 2);
#pragma unroll
      for (int e = 0; e < 2; ++e) qn[b][g][e] = __shfl_sync(0xffffffffu, gs[g], 4 * (2 * t4 + e)) * 5.9604644775390625e-8f;      // 2^-24
    }
  }
  const int first_pos = pos0 + col0 / R;                                // every column sees the keys up to here

  bool ok = true;
  int st = 0;
  uint32_t parity = 0;
  for (int i = 0; i < slices; ++i) {
    ok = __all_sync(0xffffffffu, kf_wait(&full[st], parity, a.word));
    if (!ok) break;
    const uint8_t* blk = ring + st * SLICE;
    uint32_t kw[2][W], vw[2][W], kp[2][NG], vp[2][NG];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      lds_words<W>(kw[x], blk + (g8 + 8 * x) * (D / 2) + t4 * 4 * W);
      lds_words<NG>(kp[x], blk + kv4_k_params(D) + (g8 + 8 * x) * NG * 4);
      lds_words<W>(vw[x], blk + kv4_v_codes(D) + (t4 + 4 * x) * D + g8 * 4 * W);
      lds_words<NG>(vp[x], blk + kv4_v_params(D, NG) + (g8 + 8 * x) * NG * 4);
    }
    // the next slice for this place of the ring
    const int nxt = i + KF_STAGES;
    if ((nxt & 31) == 0) entry = nxt + lane < slices ? table[nxt + lane] : 0;
    const int page = __shfl_sync(0xffffffffu, entry, nxt & 31);
    __syncwarp();                                                       // every lane has read the slice
    if (lane == 0 && nxt < slices) {
      mbar_expect_tx(&full[st], SLICE);
      bulk_load_1d(ring + st * SLICE, from + min(max(page, 0), a.pages - 1) * page_bytes, SLICE, &full[st]);
    }
    if (++st == KF_STAGES) st = 0, parity ^= 1;
    const int j = (page0 + i) * KV4_PAGE + 16 * warp + g8;              // the lane's keys: j, j + 8
    // scores, in the products' units
    float s[NB][4];
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
      const float2 p0 = bits_pair<T>(kp[0][g]), p1 = bits_pair<T>(kp[1][g]);
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 p = e < 2 ? p0 : p1;
          s[b][e] = fmaf(p.x, acc[b][e], g == 0 ? p.y * qn[b][g][e & 1] : fmaf(p.y, qn[b][g][e & 1], s[b][e]));
        }
    }
    float2 pv[2][NG];
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int g = 0; g < NG; ++g) pv[x][g] = bits_pair<T>(vp[x][g]);
    // which keys a column sees: all of them but at the end of its walk, where a slot behind the last key may hold anything
    const bool masked = j - g8 + 15 > first_pos;
    if (masked) {
#pragma unroll
      for (int x = 0; x < 2; ++x) {
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            if (j + 8 * x > pos0 + min(col0 + 8 * b + 2 * t4 + e, col0 + cols - 1) / R) s[b][2 * x + e] = -INFINITY;
        if (j + 8 * x > last)
#pragma unroll
          for (int g = 0; g < NG; ++g) pv[x][g] = make_float2(0.f, 0.f);
      }
    }
    // do references or exponents have to move?
    bool grow = false;
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int e = 0; e < 2; ++e) grow |= fmaxf(s[b][e], s[b][e + 2]) * kq[b][e] > ref[b][e] + KF_SLACK;
#pragma unroll
    for (int g = 0; g < NG; ++g) grow |= fmaxf(pv[0][g].x, pv[1][g].x) > 2.f * __uint_as_float(ev[g]);
    if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float m = fmaxf(s[b][e], s[b][e + 2]) * kq[b][e];
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
          m = fmaxf(m, ref[b][e]);
          const float f = kf_exp2(ref[b][e] - m);
          ref[b][e] = m;
          sum[b][e] *= f;
#pragma unroll
          for (int g = 0; g < NG; ++g) sumlo[b][g][e] *= f;
#pragma unroll
          for (int r = 0; r < KS; ++r) o[b][r][e] *= f, o[b][r][e + 2] *= f;
        }
#pragma unroll
      for (int g = 0; g < NG; ++g) {      // (scales are not negative: their bits rise with them; infinite ones and those that are none are passed over)
        const uint32_t e0 = __float_as_uint(pv[0][g].x), e1 = __float_as_uint(pv[1][g].x);
        const uint32_t big = __reduce_max_sync(0xffffffffu, max(e0 < 0x7f800000u ? e0 : 0u, e1 < 0x7f800000u ? e1 : 0u)) & 0x7f800000u;
        if (big > ev[g]) {
          const float f = __uint_as_float(max((int)ev[g] - (int)big + (127 << 23), 0));
          ev[g] = big;
#pragma unroll
          for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int r = 0; r < SPG; ++r)
#pragma unroll
              for (int e = 0; e < 4; ++e) o[b][g * SPG + r][e] *= f;
        }
      }
    }
    // weights
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[b][e] = kf_exp2(fmaf(s[b][e], kq[b][e & 1], -ref[b][e & 1]));
        sum[b][e & 1] += s[b][e];
      }
    // y += (p s) c, p lo: by groups, the scales brought under 4 by a power of two that only grows
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      const float inv = __uint_as_float((254u << 23) - ev[g]);
      const float s0 = pv[0][g].x * inv, s1 = pv[1][g].x * inv;
      uint32_t bw[NB][TERMS][2];
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        float w[4] = {s[b][0] * s0, s[b][1] * s0, s[b][2] * s1, s[b][3] * s1};
        if (masked) {                                                   // (a value that is no number, behind a column: no trace of it)
          float l[4] = {s[b][0] * pv[0][g].y, s[b][1] * pv[0][g].y, s[b][2] * pv[1][g].y, s[b][3] * pv[1][g].y};
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (s[b][e] == 0.f) w[e] = 0.f, l[e] = 0.f;
          sumlo[b][g][0] += l[0] + l[2];
          sumlo[b][g][1] += l[1] + l[3];
        } else {
          sumlo[b][g][0] = fmaf(s[b][0], pv[0][g].y, fmaf(s[b][2], pv[1][g].y, sumlo[b][g][0]));
          sumlo[b][g][1] = fmaf(s[b][1], pv[0][g].y, fmaf(s[b][3], pv[1][g].y, sumlo[b][g][1]));
        }
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const uint32_t h = half_bits(w[2 * x], w[2 * x + 1]);
          bw[b][0][x] = movmatrix(h);
          if (TERMS == 2) {
            const float2 f = bits_pair<__half>(h);
            bw[b][TERMS - 1][x] = movmatrix(half_bits(w[2 * x] - f.x, w[2 * x + 1] - f.y));
          }
        }
      }
#pragma unroll
      for (int e = 0; e < SPG; ++e) {
        const int r = g * SPG + e;
        const uint32_t w0 = (r & 1) ? vw[0][r >> 1] >> 8 : vw[0][r >> 1], w1 = (r & 1) ? vw[1][r >> 1] >> 8 : vw[1][r >> 1];
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
          for (int x = 0; x < TERMS; ++x)
            mma_f16_16816(o[b][r], w0 & 0x000f000fu, w0 & 0x00f000f0u, w1 & 0x000f000fu, w1 & 0x00f000f0u, bw[b][x][0], bw[b][x][1]);
      }
    }
  }
  if (!ok) {
    s_fail = 1;
    for (int w = 0; w < 2048; ++w) __nanosleep(512);                    // copies that were asked for end before the block does
  }
  // a column's sums over the lanes that share it
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int e = 0; e < 2; ++e)
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
      for (int e = 0; e < 2; ++e) s_ref[warp][8 * b + 2 * t4 + e] = ref[b][e], s_sum[warp][8 * b + 2 * t4 + e] = sum[b][e];
  __syncthreads();                      // every slice has been read: the rings hold the warps' sums now
  if (s_fail) return;
  pdl_launch_dependents();
  float* so = reinterpret_cast<float*>(smem);                           // [warp][column][D + 4]
  constexpr int LD = D + 4;
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int r = 0; r < KS; ++r) {
      const float up = __uint_as_float(ev[r / SPG]);
#pragma unroll
      for (int e = 0; e < 4; ++e)                                       // (codes were 2^-24 and, of odd nibbles, 2^-20 of themselves)
        so[(warp * COLS + 8 * b + 2 * t4 + (e & 1)) * LD + 16 * r + 8 * (e >> 1) + g8] =
            fmaf(o[b][r][e] * (e < 2 ? 16777216.f : 1048576.f), up, sumlo[b][r / SPG][e & 1]);
    }
  __syncthreads();
  // the four warps' parts; the block's are stored as they are, or as the result where there is no other part
  for (int x = threadIdx.x; x < cols * (D / 4); x += KF_THREADS) {
    const int c = x / (D / 4), d = x % (D / 4) * 4;
    float m = s_ref[0][c];
#pragma unroll
    for (int w = 1; w < KF_WARPS; ++w) m = fmaxf(m, s_ref[w][c]);
    float l = 0.f, v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < KF_WARPS; ++w) {
      const float f = kf_exp2(s_ref[w][c] - m);
      const float4 u = *reinterpret_cast<const float4*>(so + (w * COLS + c) * LD + d);
      l = fmaf(s_sum[w][c], f, l);
      v[0] = fmaf(u.x, f, v[0]), v[1] = fmaf(u.y, f, v[1]), v[2] = fmaf(u.z, f, v[2]), v[3] = fmaf(u.w, f, v[3]);
    }
    if (it.w == 1) {
      const int cc = col0 + c;
      const uint2 out = make_uint2(pair_bits<T>(v[0] / l, v[1] / l), pair_bits<T>(v[2] / l, v[3] / l));
      *reinterpret_cast<uint2*>(y + ((size_t)(first + cc / R) * a.H + head * R + cc % R) * D + d) = out;
    } else {
      const size_t at = ((size_t)item * a.G + head) * COLS + c;
      *reinterpret_cast<float4*>(a.part + at * D + d) = make_float4(v[0], v[1], v[2], v[3]);
      if (d == 0) *reinterpret_cast<float2*>(a.part + (size_t)a.max_items * a.G * COLS * D + at * 2) = make_float2(m, l);
    }
  }
}

// Joins the parts of a request's walk: a block a column, a warp every KJ-th part.
constexpr int KJ = 8;
template <typename T, int D, int NB>
__global__ void __launch_bounds__(KJ * 32) kv4_join_kernel(const Kv4Attn a) {
  constexpr int COLS = 8 * NB, E = D / 32;
  __shared__ float s_m[KJ], s_l[KJ], s_o[KJ][D];
  pdl_wait();
  const int item = blockIdx.x, head = blockIdx.y, c = blockIdx.z;
  const int32_t* work = after_wait(a.work);
  if (item >= work[0]) return;
  const int4 it = reinterpret_cast<const int4*>(work)[1 + item];
  if (it.z != 0 || it.w == 1) return;
  const int seq = it.x, first = a.starts[seq], n = a.starts[seq + 1] - first, R = a.H / a.G, col = it.y * COLS + c;
  if (a.request[seq] < 0 || col >= n * R) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const float* part = after_wait(a.part);
  const float2* ml = reinterpret_cast<const float2*>(part + (size_t)a.max_items * a.G * COLS * D);
  float m = KF_NONE, l = 0.f, o[E];
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = 0.f;
#pragma unroll 4
  for (int k = warp; k < it.w; k += KJ) {
    const size_t at = ((size_t)(item + k) * a.G + head) * COLS + c;
    const float2 u = ml[at];
    const float mn = fmaxf(m, u.x), f = kf_exp2(m - mn), w = kf_exp2(u.x - mn);
    m = mn;
    l = fmaf(l, f, u.y * w);
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = fmaf(o[e], f, part[at * D + lane * E + e] * w);
  }
  if (lane == 0) s_m[warp] = m, s_l[warp] = l;
#pragma unroll
  for (int e = 0; e < E; ++e) s_o[warp][lane * E + e] = o[e];
  __syncthreads();
  const int d = threadIdx.x;
  if (d >= D) return;
  float mm = s_m[0], num = 0.f, den = 0.f;
#pragma unroll
  for (int w = 1; w < KJ; ++w) mm = fmaxf(mm, s_m[w]);
#pragma unroll
  for (int w = 0; w < KJ; ++w) {
    const float f = kf_exp2(s_m[w] - mm);
    num = fmaf(s_o[w][d], f, num);
    den = fmaf(s_l[w], f, den);
  }
  dt<T>::st((T*)a.y, ((size_t)(first + col / R) * a.H + head * R + col % R) * D + d, num / den);
}

// ------------------------------------------------------------------ the division of a step's walks
constexpr int KW_THREADS = 1024;

__device__ __forceinline__ int block_sum(int v, int* s_warp) {
  v = __reduce_add_sync(0xffffffffu, v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) s_warp[threadIdx.x >> 5] = v;
  __syncthreads();
  return __reduce_add_sync(0xffffffffu, s_warp[threadIdx.x & 31]);
}

// Parts of `step` pages at most, step the smallest with which a step's walks are cut no more than `parts` times.
__global__ void __launch_bounds__(KW_THREADS) kv4_work_kernel(const int32_t* __restrict__ starts, const int32_t* __restrict__ ends,
                                                             const int32_t* __restrict__ request, int B, int R, int cols, int least, int longest, int parts,
                                                             int max_items, int32_t* __restrict__ work) {
  __shared__ int s_warp[32];
  auto walks = [&](int i) { return ((starts[i + 1] - starts[i]) * R + cols - 1) / cols; };
  auto pages = [&](int i) { return request[i] >= 0 ? max(1, (ends[i] + KV4_PAGE - 1) / KV4_PAGE) : 1; };
  auto total = [&](int step) {
    int v = 0;
    for (int i = threadIdx.x; i < B; i += KW_THREADS) v += walks(i) * ((pages(i) + step - 1) / step);
    return block_sum(v, s_warp);
  };
  const int most = parts + total(longest);
  int lo = least, hi = max(least, longest);
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (total(mid) <= most) hi = mid;
    else lo = mid + 1;
  }
  // a warp a sequence: its place among the items is the sum before it, taken 1024 sequences at a time
  int base = 0;
  for (int i0 = 0; i0 < B; i0 += KW_THREADS) {
    const int i = i0 + threadIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int w = i < B ? walks(i) : 0, k = i < B ? (pages(i) + lo - 1) / lo : 0;
    int incl = w * k;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, incl, d);
      if (lane >= d) incl += u;
    }
    __syncthreads();
    if (lane == 31) s_warp[warp] = incl;
    __syncthreads();
    int before = base;
    for (int x = 0; x < warp; ++x) before += s_warp[x];
    const int mine = before + incl - w * k;
    for (int x = 0; x < 32; ++x) base += s_warp[x];
    for (int l = 0; l < 32; ++l) {
      const int at = __shfl_sync(0xffffffffu, mine, l), n = __shfl_sync(0xffffffffu, w * k, l), kk = __shfl_sync(0xffffffffu, k, l), seq = i0 + 32 * warp + l;
      for (int e = lane; e < n; e += 32)
        if (at + e < max_items) reinterpret_cast<int4*>(work)[1 + at + e] = make_int4(seq, e / kk, e % kk, kk);
    }
  }
  if (threadIdx.x == 0) {
    work[0] = min(base, max_items);
    work[1] = lo;
  }
}

}  // namespace

// How many items a step's division has at most.
static int kf_parts(int G) { return ((sm_count() > 0 ? sm_count() : 148) * 4 + G - 1) / G; }
static int kf_cols(int max_count, int R) { return (long long)max_count * R <= 8 ? 8 : 16; }
static long long kf_items(int B, int T, int max_count, int H, int G) {
  const int R = H / G, cols = kf_cols(max_count, R);
  const long long walks = (long long)T * R / cols + B;
  const int parts = kf_parts(G);
  return walks + parts;
}

}  // namespace llb

using namespace llb;

extern "C" {

size_t ll_kv4_work_ints(int B, int T, int max_count, int H, int G) { return 4 + 4 * (size_t)kf_items(B, T, max_count, H, G); }

int ll_kv4_work(const int32_t* plan, int B, int T, int max_count, int H, int G, int max_length, int32_t* work, ll_stream stream) {
  LL_CHECK_ARG(plan && work && B > 0 && T >= 0 && max_count >= 0 && G > 0 && H > 0 && H % G == 0 && max_length > 0, "kv4_work: %d sequences of %d tokens, %d heads over %d",
               B, T, H, G);
  kv4_work_kernel<<<1, KW_THREADS, 0, (cudaStream_t)stream>>>(plan, plan + B + 1, plan + 3 * (size_t)B + 1, B, H / G, kf_cols(max_count, H / G), 1,
                                                              (max_length + KV4_PAGE - 1) / KV4_PAGE, kf_parts(G), (int)kf_items(B, T, max_count, H, G), work);
  LL_LAUNCH_OK("kv4_work_kernel");
  return LL_OK;
}

size_t ll_kv4_attn_scratch_bytes(int B, int T, int max_count, int H, int G, int head_size) {
  return sizeof(float) * (size_t)kf_items(B, T, max_count, H, G) * G * kf_cols(max_count, H / G) * (head_size + 2);
}

int ll_kv4_attn(const void* q, long long q_row, const void* blocks, const int32_t* table, const int32_t* plan, const int32_t* work, void* y, int dtype, int B, int T,
                int max_count, int H, int G, int head_size, int group, int width, int pages, float scale, void* scratch, ll_stream stream) {
  LL_CHECK_ARG(kv4_shape_ok(head_size, group), "kv4_attn: heads of %d in groups of %d (32, 64 or 128 each)", head_size, group);
  LL_CHECK_ARG(dtype == LL_BF16 || dtype == LL_F16, "kv4_attn: type %d (bf16 or fp16)", dtype);
  LL_CHECK_ARG(q && blocks && table && plan && work && y && scratch && B > 0 && T > 0 && max_count >= 0 && G > 0 && G <= 65535 && H > 0 && H % G == 0 && width > 0 && pages > 0,
               "kv4_attn: %d tokens of %d heads, %d cached", T, H, G);
  LL_CHECK_ARG(scale > 0.f, "kv4_attn: scores times %g (more than 0)", scale);
  LL_CHECK_ARG((((uintptr_t)q | (uintptr_t)y | (uintptr_t)blocks | (uintptr_t)scratch | (uintptr_t)work) & 15) == 0 && q_row % 8 == 0,
               "kv4_attn: rows have to start on 16-byte boundaries");
  const int R = H / G, cols = kf_cols(max_count, R), items = (int)kf_items(B, T, max_count, H, G);
  const Kv4Attn a{q, q_row, (const uint8_t*)blocks, table, plan, plan + B + 1, plan + 3 * (size_t)B + 1, work, y, (float*)scratch, H, G, width, pages, B, items, scale, wait_word()};
  cudaStream_t st = (cudaStream_t)stream;
#define FEW(TT, DD, NG, NB)                                                                                                                   \
  {                                                                                                                                           \
    constexpr int ring = KF_STAGES * kv4_bytes(DD, NG), join = KF_WARPS * 8 * NB * (DD + 4) * 4, smem = ring > join ? ring : join;            \
    static PerDevice set;                                                                                                                     \
    if (!set) {                                                                                                                               \
      LL_CUDA(cudaFuncSetAttribute(kv4_few_kernel<TT, DD, NG, NB>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));                       \
      prefer_max_smem(kv4_few_kernel<TT, DD, NG, NB>);                                                                                        \
      set.mark();                                                                                                                             \
    }                                                                                                                                         \
    kv4_few_kernel<TT, DD, NG, NB><<<dim3(items, G), KF_THREADS, smem, st>>>(a);                                                              \
    LL_LAUNCH_OK("kv4_few_kernel");                                                                                                           \
    LL_CUDA(launch(kv4_join_kernel<TT, DD, NB>, dim3(items, G, (unsigned)min((long long)cols, (long long)max_count * R)), dim3(KJ * 32), 0, st, true, a));                                      \
  }
#define ATTN(DD, NG)                                                   \
  if (dtype == LL_BF16 && cols == 8) FEW(__nv_bfloat16, DD, NG, 1)     \
  else if (dtype == LL_BF16) FEW(__nv_bfloat16, DD, NG, 2)             \
  else if (cols == 8) FEW(__half, DD, NG, 1)                           \
  else FEW(__half, DD, NG, 2)
  KV4_SHAPES(head_size, group, ATTN)
#undef ATTN
#undef FEW
  LL_LAUNCH_OK("kv4_join_kernel");
  return LL_OK;
}

}  // extern "C"
