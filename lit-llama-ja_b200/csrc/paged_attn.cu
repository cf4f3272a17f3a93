// Softmax attention over the paged key/value cache in 4 bits (kv4.cuh): a step's tokens, of requests of unequal lengths, over the keys at and before
// their positions.
#include "kv4.cuh"

namespace llb {
namespace {

struct Kv4Attn {
  const void* q;
  long long q_row;
  const uint8_t* blocks;
  const int32_t *table, *starts, *ends, *request, *positions, *sequence;
  void* y;
  int H, G, width, pages;
  float scale;
};

// A block a token and head, a warp a key at a time with a running maximum of its own; the warps' parts are joined at the end.
template <typename T, int D, int NG>
__global__ void __launch_bounds__(128) kv4_attn_simple_kernel(const Kv4Attn a) {
  constexpr int E = D / 32;
  __shared__ float s_m[4], s_l[4], s_o[4][D];
  const int t = blockIdx.x, h = blockIdx.y, g = h / (a.H / a.G), lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int seq = a.sequence[t];
  if (seq < 0) return;
  const int row = a.request[seq];
  T* y = (T*)a.y + ((size_t)t * a.H + h) * D;
  if (row < 0) {
    for (int d = threadIdx.x; d < D; d += 128) dt<T>::st(y, d, NAN);
    return;
  }
  const T* q = (const T*)a.q + t * a.q_row + (size_t)h * D;
  float x[E], o[E], m = -INFINITY, l = 0.f;
  for (int e = 0; e < E; ++e) x[e] = dt<T>::ld(q, lane + 32 * e), o[e] = 0.f;
  const int pos = a.positions[t];
  for (int j = warp; j <= pos; j += 4) {
    const int page = min(max(a.table[(size_t)row * a.width + j / KV4_PAGE], 0), a.pages - 1), at = j % KV4_PAGE;
    const uint8_t* blk = a.blocks + ((size_t)page * a.G + g) * kv4_bytes(D, NG);
    float s = 0.f;
    for (int e = 0; e < E; ++e) {
      const int d = lane + 32 * e, gr = d / (D / NG);
      const uint32_t w = reinterpret_cast<const uint32_t*>(blk)[at * (D / 8) + kv4_k_word(D, d)];
      const float2 p = bits_pair<T>(reinterpret_cast<const uint32_t*>(blk + kv4_k_params(D))[at * NG + gr]);
      s += x[e] * ((float)((w >> kv4_k_bit(d)) & 15u) * p.x + p.y);
    }
    s = warp_sum(s) * a.scale;
    const float mn = fmaxf(m, s), f = m == -INFINITY ? 0.f : __expf(m - mn), p = __expf(s - mn);
    m = mn;
    l = l * f + p;
    for (int e = 0; e < E; ++e) {
      const int d = lane + 32 * e, gr = d / (D / NG);
      const uint32_t w = reinterpret_cast<const uint32_t*>(blk + kv4_v_codes(D))[(at / 2) * (D / 4) + kv4_v_word(D, d)];
      const float2 v = bits_pair<T>(reinterpret_cast<const uint32_t*>(blk + kv4_v_params(D, NG))[at * NG + gr]);
      o[e] = o[e] * f + p * ((float)((w >> (16 * (at & 1) + kv4_v_bit(d))) & 15u) * v.x + v.y);
    }
  }
  if (lane == 0) s_m[warp] = m, s_l[warp] = l;
  for (int e = 0; e < E; ++e) s_o[warp][lane + 32 * e] = o[e];
  __syncthreads();
  for (int d = threadIdx.x; d < D; d += 128) {
    float mm = s_m[0], n = 0.f, s = 0.f;
    for (int w = 1; w < 4; ++w) mm = fmaxf(mm, s_m[w]);
    for (int w = 0; w < 4; ++w) {
      const float f = s_m[w] == -INFINITY ? 0.f : __expf(s_m[w] - mm);
      n += s_o[w][d] * f;
      s += s_l[w] * f;
    }
    dt<T>::st(y, d, n / s);
  }
}

}  // namespace
}  // namespace llb

using namespace llb;

extern "C" {

int ll_kv4_attn(const void* q, long long q_row, const void* blocks, const int32_t* table, const int32_t* plan, void* y, int dtype, int B, int T, int H, int G,
                int head_size, int group, int width, int pages, float scale, ll_stream stream) {
  LL_CHECK_ARG(kv4_shape_ok(head_size, group), "kv4_attn: heads of %d in groups of %d (32, 64 or 128 each)", head_size, group);
  LL_CHECK_ARG(dtype == LL_BF16 || dtype == LL_F16, "kv4_attn: type %d (bf16 or fp16)", dtype);
  LL_CHECK_ARG(q && blocks && table && plan && y && B > 0 && T > 0 && G > 0 && H > 0 && H % G == 0 && H <= 65535 && width > 0 && pages > 0, "kv4_attn: %d tokens of %d heads, %d cached",
               T, H, G);
  LL_CHECK_ARG((((uintptr_t)q | (uintptr_t)y | (uintptr_t)blocks) & 15) == 0 && q_row % 8 == 0, "kv4_attn: rows have to start on 16-byte boundaries");
  const Kv4Attn a{q, q_row, (const uint8_t*)blocks, table, plan, plan + B + 1, plan + 3 * (size_t)B + 1, plan + 4 * (size_t)B + 1,
                  plan + 4 * (size_t)B + 1 + 2 * (size_t)T, y, H, G, width, pages, scale};
  cudaStream_t st = (cudaStream_t)stream;
#define ATTN(DD, NG)                                                                                  \
  if (dtype == LL_BF16) kv4_attn_simple_kernel<__nv_bfloat16, DD, NG><<<dim3(T, H), 128, 0, st>>>(a); \
  else kv4_attn_simple_kernel<__half, DD, NG><<<dim3(T, H), 128, 0, st>>>(a);
  KV4_SHAPES(head_size, group, ATTN)
#undef ATTN
  LL_LAUNCH_OK("kv4_attn_simple_kernel");
  return LL_OK;
}

}  // extern "C"
