// The paged key/value cache in 4 bits: which pages and slots a step's tokens get, how they give them back, and the rounding of keys and values into
// their slots.  Layout: kv4.cuh; the attention that reads it: paged_attn.cu.
#include <climits>

#include "kv4.cuh"

namespace llb {
namespace {

enum Kv4Status { KV4_OK = 0, KV4_NO_PAGES = 1, KV4_TOO_LONG = 2, KV4_BAD_ROW = 3, KV4_BEHIND = 4 };

struct Kv4Pool {
  int32_t* table;      // [requests][width] page of 64 slots, or -1
  int32_t* lengths;    // [requests]
  int32_t* free;       // [pages] a stack: the last of n_free is given out next
  int32_t* n_free;     // [1]
  int32_t* stamp;      // [requests] which sequence of a step names the request first
  int requests, width, pages, max_length;
};

struct Kv4Plan {
  int32_t* starts;     // [B + 1]
  int32_t* ends;       // [B]
  int32_t* status;     // [B]
  int32_t* request;    // [B] the request, or -1 where a sequence is refused
  int32_t* positions;  // [T]
  int32_t* slots;      // [T]
  int32_t* sequence;   // [T]
};

constexpr int PLAN_THREADS = 1024;

// Sum over the threads before this one; `total` of all of them.  Every thread of the block calls.
template <typename V>
__device__ __forceinline__ V block_before(V v, V* s_warp, V& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  V incl = v;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const V u = __shfl_up_sync(0xffffffffu, incl, d);
    if (lane >= d) incl += u;
  }
  __syncthreads();                     // (the sums of a scan before this one have been read)
  if (lane == 31) s_warp[warp] = incl;
  __syncthreads();
  if (warp == 0) {
    V w = lane < PLAN_THREADS / 32 ? s_warp[lane] : V(0);
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const V u = __shfl_up_sync(0xffffffffu, w, d);
      if (lane >= d) w += u;
    }
    s_warp[lane] = w;
  }
  __syncthreads();
  total = s_warp[31];
  return (warp > 0 ? s_warp[warp - 1] : V(0)) + incl - v;
}

__device__ __forceinline__ int pages_of(int tokens) { return (tokens + KV4_PAGE - 1) / KV4_PAGE; }

// The first sequence that names a request has it: an ordered claim, so that a request named twice is the same one's in every run.
__device__ __forceinline__ void claim_requests(const int32_t* rows, const int32_t* wants, bool any_want, int B, const Kv4Pool& c) {
  for (int i = threadIdx.x; i < B; i += blockDim.x)
    if ((any_want || wants[i] > 0) && rows[i] >= 0 && rows[i] < c.requests) c.stamp[rows[i]] = INT_MAX;
  __syncthreads();
  for (int i = threadIdx.x; i < B; i += blockDim.x)
    if ((any_want || wants[i] > 0) && rows[i] >= 0 && rows[i] < c.requests) atomicMin(&c.stamp[rows[i]], i);
  __syncthreads();
}

// Pages of a step: prefix sums over the sequences in one block.
__global__ void __launch_bounds__(PLAN_THREADS) kv4_plan_kernel(const int32_t* __restrict__ rows, const int32_t* __restrict__ counts, int B, int T,
                                                               int max_count, Kv4Pool c, Kv4Plan p) {
  __shared__ long long s_sum[32];
  __shared__ int s_need[32];
  __shared__ int s_row[PLAN_THREADS], s_first[PLAN_THREADS], s_pages[PLAN_THREADS], s_used[PLAN_THREADS];
  const int n_free = min(max(*c.n_free, 0), c.pages);
  claim_requests(rows, counts, false, B, c);
  long long tokens = 0, wanted = 0;      // of the sequences before this round
  int given = 0;
  for (int i0 = 0; i0 < B; i0 += PLAN_THREADS) {
    const int i = i0 + threadIdx.x;
    const int row = i < B ? rows[i] : -1, count = i < B ? counts[i] : 0, n = max(count, 0);
    const bool named = row >= 0 && row < c.requests;
    const int old = named ? c.lengths[row] : 0;
    long long total;
    const long long first = tokens + block_before<long long>(n, s_sum, total);
    tokens += total;
    int status = KV4_OK;
    if (count < 0 || (n > 0 && (!named || c.stamp[row] != i))) status = KV4_BAD_ROW;
    else if (first + n > T) status = KV4_BEHIND;
    else if (n > max_count || (long long)old + n > c.max_length) status = KV4_TOO_LONG;
    const int page0 = pages_of(old), need = status == KV4_OK && n > 0 ? pages_of(old + n) - page0 : 0;
    const long long before = wanted + block_before<long long>(need, s_sum, total);
    wanted += total;
    if (need > 0 && before + need > n_free) status = KV4_NO_PAGES;      // and so does every one after it that wants a page
    const bool ok = status == KV4_OK;
    int all;
    block_before<int>(ok ? need : 0, s_need, all);
    given += all;
    s_row[threadIdx.x] = row;
    s_first[threadIdx.x] = page0;
    s_pages[threadIdx.x] = ok ? need : 0;
    s_used[threadIdx.x] = (int)min(before, (long long)n_free);
    if (i < B) {
      if (i == 0) p.starts[0] = 0;
      p.starts[i + 1] = (int)min(first + n, (long long)T);
      p.status[i] = status;
      p.request[i] = ok && n > 0 ? row : -1;
      if (ok && n > 0) c.lengths[row] = old + n;
    }
    __syncthreads();
    // the new entries of the table, a warp a sequence
    const int lane = threadIdx.x & 31;
    for (int j = threadIdx.x >> 5; j < min(PLAN_THREADS, B - i0); j += PLAN_THREADS / 32)
      for (int k = lane; k < s_pages[j]; k += 32) c.table[(size_t)s_row[j] * c.width + s_first[j] + k] = c.free[n_free - 1 - s_used[j] - k];
    __syncthreads();
  }
  if (threadIdx.x == 0) *c.n_free = n_free - given;
  for (int i = threadIdx.x; i < B; i += PLAN_THREADS) {      // (when all lengths are the step's: an idle sequence may name another one's request)
    const int row = rows[i];
    p.ends[i] = p.status[i] == KV4_OK && row >= 0 && row < c.requests ? c.lengths[row] : 0;
  }
}

// Positions and slots of a step's tokens.
__global__ void __launch_bounds__(256) kv4_tokens_kernel(int B, int T, Kv4Pool c, Kv4Plan p) {
  const int t = blockIdx.x * blockDim.x + threadIdx.x;
  if (t >= T) return;
  int lo = 0, hi = B;                  // the first sequence that ends behind t
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (p.starts[mid + 1] > t) hi = mid;
    else lo = mid + 1;
  }
  int pos = -1, slot = -1, row;
  if (lo < B && (row = p.request[lo]) >= 0) {
    pos = p.ends[lo] - (p.starts[lo + 1] - t);
    slot = c.table[(size_t)row * c.width + pos / KV4_PAGE] * KV4_PAGE + pos % KV4_PAGE;
  }
  p.positions[t] = pos;
  p.slots[t] = slot;
  p.sequence[t] = lo < B ? lo : -1;
}

// The way back: requests are cut to `keep` tokens, the pages behind go to the stack in the order that a plan would take them in again.
__global__ void __launch_bounds__(PLAN_THREADS) kv4_truncate_kernel(const int32_t* __restrict__ rows, const int32_t* __restrict__ keep, int B, Kv4Pool c) {
  __shared__ int s_sum[32];
  __shared__ int s_row[PLAN_THREADS], s_first[PLAN_THREADS], s_pages[PLAN_THREADS], s_used[PLAN_THREADS];
  const int n_free = min(max(*c.n_free, 0), c.pages);
  claim_requests(rows, keep, true, B, c);
  int total = 0;                        // the pages of all sequences have to be known before the first goes back
  for (int i0 = 0; i0 < B; i0 += PLAN_THREADS) {
    const int i = i0 + threadIdx.x, row = i < B ? rows[i] : -1;
    int n = 0, all;
    if (row >= 0 && row < c.requests && c.stamp[row] == i && keep[i] >= 0 && keep[i] < c.lengths[row]) n = pages_of(c.lengths[row]) - pages_of(keep[i]);
    block_before<int>(n, s_sum, all);
    total += all;
  }
  int done = 0;
  for (int i0 = 0; i0 < B; i0 += PLAN_THREADS) {
    const int i = i0 + threadIdx.x, row = i < B ? rows[i] : -1;
    int n = 0, first = 0, all;
    const bool cut = row >= 0 && row < c.requests && c.stamp[row] == i && keep[i] >= 0 && keep[i] < c.lengths[row];
    if (cut) first = pages_of(keep[i]), n = pages_of(c.lengths[row]) - first;
    const int before = done + block_before<int>(n, s_sum, all);
    done += all;
    s_row[threadIdx.x] = row;
    s_first[threadIdx.x] = first;
    s_pages[threadIdx.x] = n;
    s_used[threadIdx.x] = before;
    __syncthreads();
    if (cut) c.lengths[row] = keep[i];
    const int lane = threadIdx.x & 31;
    for (int j = threadIdx.x >> 5; j < min(PLAN_THREADS, B - i0); j += PLAN_THREADS / 32)
      for (int k = lane; k < s_pages[j]; k += 32) {
        int32_t* e = c.table + (size_t)s_row[j] * c.width + s_first[j] + k;
        const int at = n_free + total - 1 - s_used[j] - k;
        if (at < c.pages) c.free[at] = *e;
        *e = -1;
      }
    __syncthreads();
  }
  if (threadIdx.x == 0) *c.n_free = min(n_free + total, c.pages);
}

// ------------------------------------------------------------------ append
struct Kv4Rows {
  const void* q;
  const void* k;
  const void* v;
  long long q_row, k_row, v_row;       // distances of a token's rows, in numbers; heads follow one another
};

// One warp a vector of a token: a query to turn, a key to turn and round, a value to round.  E numbers a lane.
template <typename T, int D, int NG, bool TURN>
__global__ void __launch_bounds__(256) kv4_append_kernel(Kv4Rows in, const float* __restrict__ rope, const int32_t* __restrict__ positions,
                                                         const int32_t* __restrict__ slots, T* __restrict__ q_out, uint8_t* __restrict__ blocks, int H, int G) {
  constexpr int E = D == 128 ? 4 : 2, LANES = D / E, GL = LANES / NG;
  const int t = blockIdx.x, lane = threadIdx.x & 31, vec = blockIdx.y * 8 + (threadIdx.x >> 5);
  const int nq = TURN ? H : 0;
  if (vec >= nq + 2 * G) return;
  const int slot = slots[t], pos = positions[t];
  const bool is_q = vec < nq, is_k = !is_q && vec < nq + G;
  const int head = is_q ? vec : is_k ? vec - nq : vec - nq - G;
  if (!is_q && slot < 0) return;
  const T* row = is_q ? (const T*)in.q + t * in.q_row : is_k ? (const T*)in.k + t * in.k_row : (const T*)in.v + t * in.v_row;
  row += head * D;
  const bool live = lane < LANES;
  const int d0 = lane * E;
  float x[E];
#pragma unroll
  for (int e = 0; e < E; e += 2) {
    const float2 f = live ? bits_pair<T>(*reinterpret_cast<const uint32_t*>(row + d0 + e)) : make_float2(0.f, 0.f);
    x[e] = f.x, x[e + 1] = f.y;
  }
  if (TURN && (is_q || is_k)) {
    const float* cs = rope + (size_t)max(pos, 0) * D;
#pragma unroll
    for (int e = 0; e < E; e += 2) {
      const float2 f = live ? *reinterpret_cast<const float2*>(cs + d0 + e) : make_float2(0.f, 0.f);
      const float a = __fsub_rn(__fmul_rn(x[e], f.x), __fmul_rn(x[e + 1], f.y)), b = __fadd_rn(__fmul_rn(x[e + 1], f.x), __fmul_rn(x[e], f.y));
      x[e] = a, x[e + 1] = b;
    }
  }
  if (is_q) {
    if (live) {
      T* o = q_out + ((size_t)t * H + head) * D + d0;
#pragma unroll
      for (int e = 0; e < E; e += 2) *reinterpret_cast<uint32_t*>(o + e) = pos < 0 ? pair_bits<T>(NAN, NAN) : pair_bits<T>(x[e], x[e + 1]);
    }
    return;
  }
  // the numbers as the cache's type has them, their smallest and largest by groups of GL lanes
  float lo = INFINITY, hi = -INFINITY;
#pragma unroll
  for (int e = 0; e < E; e += 2) {
    const float2 f = bits_pair<T>(pair_bits<T>(x[e], x[e + 1]));
    x[e] = f.x, x[e + 1] = f.y;
    lo = fminf(lo, fminf(f.x, f.y));
    hi = fmaxf(hi, fmaxf(f.x, f.y));
    if (!(fabsf(f.x) < INFINITY) || !(fabsf(f.y) < INFINITY)) lo = -INFINITY, hi = INFINITY;
  }
#pragma unroll
  for (int o = GL / 2; o > 0; o >>= 1) {
    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
  }
  uint32_t params = pair_bits<T>(__fmul_rn(__fsub_rn(hi, lo), (float)(1.0 / 15.0)), lo);
  float s = bits_pair<T>(params).x;
  if (!(s < INFINITY)) {               // a group with a number that is none, or infinite, or too wide: it stands for no numbers
    params = pair_bits<T>(NAN, NAN);
    s = 0.f;
  }
  uint32_t code[E];
#pragma unroll
  for (int e = 0; e < E; ++e) code[e] = s > 0.f ? (uint32_t)fminf(fmaxf(rintf(__fdiv_rn(__fsub_rn(x[e], lo), s)), 0.f), 15.f) : 0u;
  uint8_t* blk = blocks + ((size_t)(slot / KV4_PAGE) * G + head) * kv4_bytes(D, NG) + slot % KV4_PAGE / KV4_SLICE * kv4_slice_bytes(D, NG);
  const int at = slot % KV4_SLICE;
  if (live && lane % GL == 0)
    reinterpret_cast<uint32_t*>(blk + (is_k ? kv4_k_params(D) : kv4_v_params(D, NG)))[at * NG + lane / GL] = params;
  if (is_k) {
    // a word's codes lie in the lanes that differ in the nibble number
    uint32_t w = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) w |= code[e] << kv4_k_bit(d0 + e);
    if (E == 2) w |= __shfl_xor_sync(0xffffffffu, w, 1);
    w |= __shfl_xor_sync(0xffffffffu, w, E == 4 ? 4 : 8);
    if (live && (lane & (E == 4 ? 4 : 9)) == 0) reinterpret_cast<uint32_t*>(blk)[at * (D / 8) + kv4_k_word(D, d0)] = w;
  } else {
    // 16 bits of a word: nibbles 0 - 3 of one slot
    unsigned long long w = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) w |= (unsigned long long)code[e] << (16 * e + kv4_v_bit(d0 + e));
    w |= __shfl_xor_sync(0xffffffffu, w, E == 4 ? 2 : 4);
    w |= __shfl_xor_sync(0xffffffffu, w, E == 4 ? 4 : 8);
    const int e = E == 4 ? (lane >> 1) & 3 : (lane >> 2) & 3;      // which of the chunks this lane stores
    if (live && e < E) {
      const int d = d0 % 8 + e + 32 * (d0 / 32);                   // nibble 0's dimension
      reinterpret_cast<uint16_t*>(blk + kv4_v_codes(D))[2 * ((at / 2) * (D / 4) + kv4_v_word(D, d)) + (at & 1)] = (uint16_t)(w >> (16 * e));
    }
  }
}

// The values that slots stand for.
template <typename T, int D, int NG>
__global__ void __launch_bounds__(D) kv4_read_kernel(const uint8_t* __restrict__ blocks, const int32_t* __restrict__ slots, T* __restrict__ k_out,
                                                     T* __restrict__ v_out, int G, int pages) {
  const int t = blockIdx.x, head = blockIdx.y, d = threadIdx.x, slot = slots[t];
  float k = NAN, v = NAN;
  if (slot >= 0 && slot < pages * KV4_PAGE) {
    const uint8_t* blk = blocks + ((size_t)(slot / KV4_PAGE) * G + head) * kv4_bytes(D, NG) + slot % KV4_PAGE / KV4_SLICE * kv4_slice_bytes(D, NG);
    const int at = slot % KV4_SLICE, g = d / (D / NG);
    const uint32_t kw = reinterpret_cast<const uint32_t*>(blk)[at * (D / 8) + kv4_k_word(D, d)];
    const uint32_t vw = reinterpret_cast<const uint32_t*>(blk + kv4_v_codes(D))[(at / 2) * (D / 4) + kv4_v_word(D, d)];
    const float2 kp = bits_pair<T>(reinterpret_cast<const uint32_t*>(blk + kv4_k_params(D))[at * NG + g]);
    const float2 vp = bits_pair<T>(reinterpret_cast<const uint32_t*>(blk + kv4_v_params(D, NG))[at * NG + g]);
    k = __fadd_rn(__fmul_rn((float)((kw >> kv4_k_bit(d)) & 15u), kp.x), kp.y);
    v = __fadd_rn(__fmul_rn((float)((vw >> (16 * (at & 1) + kv4_v_bit(d))) & 15u), vp.x), vp.y);
  }
  const size_t o = ((size_t)t * G + head) * D + d;
  dt<T>::st(k_out, o, k);
  dt<T>::st(v_out, o, v);
}

bool pool_ok(const Kv4Pool& c) {
  return c.table && c.lengths && c.free && c.n_free && c.stamp && c.requests > 0 && c.width > 0 && c.pages > 0 && c.pages <= INT_MAX / KV4_PAGE &&
         c.max_length > 0 && (c.max_length - 1) / KV4_PAGE < c.width;
}

}  // namespace
}  // namespace llb

using namespace llb;

extern "C" {

size_t ll_kv4_page_bytes(int head_size, int group) { return kv4_shape_ok(head_size, group) ? (size_t)kv4_bytes(head_size, head_size / group) : 0; }

int ll_kv4_plan(const int32_t* rows, const int32_t* counts, int B, int T, int max_count, int32_t* table, int32_t* lengths, int32_t* free_pages, int32_t* n_free,
                int32_t* stamp, int requests, int width, int pages, int max_length, int32_t* out, ll_stream stream) {
  const Kv4Pool c{table, lengths, free_pages, n_free, stamp, requests, width, pages, max_length};
  LL_CHECK_ARG(rows && counts && out && B > 0 && T >= 0 && max_count >= 0 && pool_ok(c), "kv4_plan: %d sequences of %d tokens, %d requests of up to %d in %d pages",
               B, T, requests, max_length, pages);
  const Kv4Plan p{out, out + B + 1, out + 2 * (size_t)B + 1, out + 3 * (size_t)B + 1, out + 4 * (size_t)B + 1, out + 4 * (size_t)B + 1 + T,
                  out + 4 * (size_t)B + 1 + 2 * (size_t)T};
  cudaStream_t st = (cudaStream_t)stream;
  kv4_plan_kernel<<<1, PLAN_THREADS, 0, st>>>(rows, counts, B, T, max_count, c, p);
  LL_LAUNCH_OK("kv4_plan_kernel");
  if (T > 0) {
    kv4_tokens_kernel<<<(T + 255) / 256, 256, 0, st>>>(B, T, c, p);
    LL_LAUNCH_OK("kv4_tokens_kernel");
  }
  return LL_OK;
}

int ll_kv4_truncate(const int32_t* rows, const int32_t* keep, int B, int32_t* table, int32_t* lengths, int32_t* free_pages, int32_t* n_free, int32_t* stamp,
                    int requests, int width, int pages, int max_length, ll_stream stream) {
  const Kv4Pool c{table, lengths, free_pages, n_free, stamp, requests, width, pages, max_length};
  LL_CHECK_ARG(rows && keep && B > 0 && pool_ok(c), "kv4_truncate: %d sequences, %d requests of up to %d in %d pages", B, requests, max_length, pages);
  kv4_truncate_kernel<<<1, PLAN_THREADS, 0, (cudaStream_t)stream>>>(rows, keep, B, c);
  LL_LAUNCH_OK("kv4_truncate_kernel");
  return LL_OK;
}

int ll_kv4_append(const void* q, long long q_row, const void* k, long long k_row, const void* v, long long v_row, const float* rope, const int32_t* positions,
                  const int32_t* slots, void* q_out, void* blocks, int dtype, int T, int H, int G, int head_size, int group, ll_stream stream) {
  LL_CHECK_ARG(kv4_shape_ok(head_size, group), "kv4_append: heads of %d in groups of %d (32, 64 or 128 each)", head_size, group);
  LL_CHECK_ARG(dtype == LL_BF16 || dtype == LL_F16, "kv4_append: type %d (bf16 or fp16)", dtype);
  LL_CHECK_ARG(k && v && positions && slots && blocks && (!rope || (q && q_out)) && T > 0 && H > 0 && G > 0, "kv4_append: %d tokens of %d heads, %d cached", T, H, G);
  const uintptr_t a = (uintptr_t)(rope ? q : nullptr) | (uintptr_t)k | (uintptr_t)v | (uintptr_t)rope | (uintptr_t)q_out | (uintptr_t)blocks;
  LL_CHECK_ARG((a & 15) == 0 && ((rope ? q_row : 0) | k_row | v_row) % 8 == 0, "kv4_append: rows have to start on 16-byte boundaries");
  const Kv4Rows in{q, k, v, q_row, k_row, v_row};
  cudaStream_t st = (cudaStream_t)stream;
  const dim3 grid(T, ((rope ? H : 0) + 2 * G + 7) / 8);
#define APPEND(DD, NG)                                                                                                                              \
  if (dtype == LL_BF16 && rope) kv4_append_kernel<__nv_bfloat16, DD, NG, true><<<grid, 256, 0, st>>>(in, rope, positions, slots, (__nv_bfloat16*)q_out, (uint8_t*)blocks, H, G); \
  else if (dtype == LL_BF16) kv4_append_kernel<__nv_bfloat16, DD, NG, false><<<grid, 256, 0, st>>>(in, rope, positions, slots, (__nv_bfloat16*)q_out, (uint8_t*)blocks, H, G);    \
  else if (rope) kv4_append_kernel<__half, DD, NG, true><<<grid, 256, 0, st>>>(in, rope, positions, slots, (__half*)q_out, (uint8_t*)blocks, H, G);  \
  else kv4_append_kernel<__half, DD, NG, false><<<grid, 256, 0, st>>>(in, rope, positions, slots, (__half*)q_out, (uint8_t*)blocks, H, G);
  KV4_SHAPES(head_size, group, APPEND)
#undef APPEND
  LL_LAUNCH_OK("kv4_append_kernel");
  return LL_OK;
}

int ll_kv4_read(const void* blocks, const int32_t* slots, void* k, void* v, int dtype, int n, int G, int head_size, int group, int pages, ll_stream stream) {
  LL_CHECK_ARG(kv4_shape_ok(head_size, group), "kv4_read: heads of %d in groups of %d (32, 64 or 128 each)", head_size, group);
  LL_CHECK_ARG(dtype == LL_BF16 || dtype == LL_F16, "kv4_read: type %d (bf16 or fp16)", dtype);
  LL_CHECK_ARG(blocks && slots && k && v && n > 0 && G > 0 && G <= 65535 && pages > 0, "kv4_read: %d slots of %d heads", n, G);
  cudaStream_t st = (cudaStream_t)stream;
  const dim3 grid(n, G);
#define READ(DD, NG)                                                                                                                                   \
  if (dtype == LL_BF16) kv4_read_kernel<__nv_bfloat16, DD, NG><<<grid, DD, 0, st>>>((const uint8_t*)blocks, slots, (__nv_bfloat16*)k, (__nv_bfloat16*)v, G, pages); \
  else kv4_read_kernel<__half, DD, NG><<<grid, DD, 0, st>>>((const uint8_t*)blocks, slots, (__half*)k, (__half*)v, G, pages);
  KV4_SHAPES(head_size, group, READ)
#undef READ
  LL_LAUNCH_OK("kv4_read_kernel");
  return LL_OK;
}

}  // extern "C"
