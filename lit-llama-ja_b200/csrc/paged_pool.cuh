// The pool of the paged key/value cache as one block of threads works on it: requests' tables, the stack of free pages, who names a request first.
#pragma once
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

constexpr int PLAN_THREADS = 1024;      // of such a block, at most

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
  V sums = lane < (int)(blockDim.x >> 5) ? s_warp[lane] : V(0);       // (every warp sums the warps' sums for itself)
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const V u = __shfl_up_sync(0xffffffffu, sums, d);
    if (lane >= d) sums += u;
  }
  total = __shfl_sync(0xffffffffu, sums, 31);
  const V before = __shfl_sync(0xffffffffu, sums, warp > 0 ? warp - 1 : 0);
  return (warp > 0 ? before : V(0)) + incl - v;
}

__device__ __forceinline__ int pages_of(int tokens) { return (tokens + KV4_PAGE - 1) / KV4_PAGE; }

// The first sequence that names a request has it, so that a request named twice is the same one's in every run.  Up to PLAN_NEAR sequences look
// through the names before theirs in shared memory; more leave an ordered claim with the request.
constexpr int PLAN_NEAR = 256;
__device__ __forceinline__ void claim_requests(const int32_t* rows, const int32_t* wants, bool any_want, int B, const Kv4Pool& c) {
  if (B <= PLAN_NEAR) return;
  for (int i = threadIdx.x; i < B; i += blockDim.x)
    if ((any_want || wants[i] > 0) && rows[i] >= 0 && rows[i] < c.requests) c.stamp[rows[i]] = INT_MAX;
  __syncthreads();
  for (int i = threadIdx.x; i < B; i += blockDim.x)
    if ((any_want || wants[i] > 0) && rows[i] >= 0 && rows[i] < c.requests) atomicMin(&c.stamp[rows[i]], i);
  __syncthreads();
}
// Whether sequence i's claim on `row` holds (`claims`: it has one).  Every thread of the block calls.
__device__ __forceinline__ bool claimed(int i, int row, bool claims, int B, const Kv4Pool& c, int* s_name) {
  if (B > PLAN_NEAR) return claims && c.stamp[row] == i;
  if (i < PLAN_NEAR) s_name[i] = claims ? row : -1;
  __syncthreads();
  bool first = claims;
  if (claims) {
    const int4* names = reinterpret_cast<const int4*>(s_name);
    for (int j = 0; 4 * j < i; ++j) {
      const int4 n = names[j];
      first &= !(n.x == row && 4 * j < i) && !(n.y == row && 4 * j + 1 < i) && !(n.z == row && 4 * j + 2 < i) && !(n.w == row && 4 * j + 3 < i);
    }
  }
  return first;
}

inline int check_cache(const ll_kv4_cache* c, const char* who) {
  LL_CHECK_ARG(c != nullptr, "%s: no cache", who);
  LL_CHECK_ARG(kv4_shape_ok(c->head_size, c->group), "%s: kv4 heads of %d in groups of %d (32, 64 or 128 each)", who, c->head_size, c->group);
  LL_CHECK_ARG(c->dtype == LL_BF16 || c->dtype == LL_F16, "%s: kv4 cache of type %d (bf16 or fp16)", who, c->dtype);
  LL_CHECK_ARG(c->table && c->lengths && c->free_pages && c->n_free && c->stamp && c->requests > 0 && c->width > 0 && c->pages > 0 && c->pages <= INT_MAX / KV4_PAGE &&
                   c->max_length > 0 && c->max_length <= (1 << 30) && (c->max_length - 1) / KV4_PAGE < c->width && c->kv_heads > 0 && c->kv_heads <= 65535 && c->heads > 0 && c->heads % c->kv_heads == 0,
               "%s: kv4 cache of %d requests of up to %d tokens in %d pages, %d heads over %d", who, c->requests, c->max_length, c->pages, c->heads, c->kv_heads);
  return LL_OK;
}
inline Kv4Pool pool_of(const ll_kv4_cache* c) {
  return Kv4Pool{c->table, c->lengths, c->free_pages, c->n_free, c->stamp, c->requests, c->width, c->pages, c->max_length};
}

}  // namespace
}  // namespace llb
