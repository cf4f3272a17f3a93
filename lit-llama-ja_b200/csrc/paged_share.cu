// Requests of the paged cache that share pages: copies of a request (fork), cuts into pages that others hold, and the copies of pages that both need.
//
// A page that a request still writes, its last one while that is not full, is the request's own: so neither a plan nor an append asks who else holds a page.
// A fork shares the whole pages and copies a last one that is not full; a cut that ends inside a page which others hold copies that one.  shared[p] counts the
// holders of page p beyond the first one (0 for free pages and for a request's own), so that a plan, which gives out free pages, need not know of it.
#include <algorithm>

#include "paged_pool.cuh"

namespace llb {
namespace {

// What a call notes of its sequences, [B] each: a page to copy and where to (-1: none), entries of the table that are given back, pages that become free
// (then: those of the sequences before).
struct ShareWork {
  int32_t *src, *dst, *first, *end, *freed;
  __host__ __device__ ShareWork(int32_t* w, int B) : src(w), dst(w + B), first(w + 2 * (size_t)B), end(w + 3 * (size_t)B), freed(w + 4 * (size_t)B) {}
};

// Empty requests into[i] become copies of rows[i], both as they are before the call.  One block: a thread a sequence decides, a warp a sequence copies its
// entries of the table.
__global__ void __launch_bounds__(PLAN_THREADS) kv4_fork_kernel(const int32_t* __restrict__ rows, const int32_t* __restrict__ into, int B, Kv4Pool c,
                                                               int32_t* __restrict__ shared, int32_t* __restrict__ status, ShareWork w) {
  __shared__ int s_sum[32];
  __shared__ int s_from[PLAN_THREADS], s_to[PLAN_THREADS], s_whole[PLAN_THREADS], s_new[PLAN_THREADS];
  __shared__ __align__(16) int s_name[PLAN_NEAR];
  const int n_free = min(max(*c.n_free, 0), c.pages), nt = blockDim.x, lane = threadIdx.x & 31;
  claim_requests(into, into, true, B, c);
  long long wanted = 0;
  int given = 0;
  for (int i0 = 0; i0 < B; i0 += nt) {
    const int i = i0 + threadIdx.x, from = i < B ? rows[i] : -1, to = i < B ? into[i] : -1;
    const bool named = to >= 0 && to < c.requests && from >= 0 && from < c.requests;
    const bool mine = claimed(i, to, to >= 0 && to < c.requests, B, c, s_name) && named && c.lengths[max(to, 0)] == 0;
    const int held = mine ? c.lengths[from] : 0, whole = held / KV4_PAGE, part = held % KV4_PAGE != 0 ? 1 : 0;
    int all;
    const long long before = wanted + block_before<int>(part, s_sum, all);
    wanted += all;
    const bool fits = part == 0 || before < n_free, ok = mine && fits, copy = ok && part != 0;
    block_before<int>(copy ? 1 : 0, s_sum, all);
    given += all;
    s_from[threadIdx.x] = from;
    s_to[threadIdx.x] = to;
    s_whole[threadIdx.x] = ok ? whole : 0;
    const int page = copy ? c.free[n_free - 1 - (int)before] : -1;
    s_new[threadIdx.x] = page;
    if (i < B) {
      status[i] = !mine ? KV4_BAD_ROW : fits ? KV4_OK : KV4_NO_PAGES;
      w.src[i] = copy ? c.table[(size_t)from * c.width + whole] : -1;
      w.dst[i] = page;
      w.end[i] = ok ? held : 0;
    }
    __syncthreads();
    for (int j = threadIdx.x >> 5; j < min(nt, B - i0); j += nt >> 5) {
      if (s_whole[j] == 0 && s_new[j] < 0) continue;
      const int32_t* a = c.table + (size_t)s_from[j] * c.width;
      int32_t* b = c.table + (size_t)s_to[j] * c.width;
      for (int k = lane; k < s_whole[j]; k += 32) {
        const int p = a[k];
        b[k] = p;
        atomicAdd(&shared[p], 1);
      }
      if (lane == 0 && s_new[j] >= 0) b[s_whole[j]] = s_new[j];
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) *c.n_free = n_free - given;
  for (int i = threadIdx.x; i < B; i += nt)      // (lengths change when all have been read: a request may be a copy and have one that names it)
    if (w.end[i] > 0) c.lengths[into[i]] = w.end[i];
}

// Requests are cut to `keep` tokens.  All decisions are taken on the pool as it is before the call: a cut inside a page that others hold needs a free page
// for its copy, and is refused where there is none.  A page goes back to the stack when its last holder has given it back, in the order of the sequences, and
// by the last of those that give it back in one call: whoever comes first makes no difference.
__global__ void __launch_bounds__(PLAN_THREADS) kv4_release_kernel(const int32_t* __restrict__ rows, const int32_t* __restrict__ keep, int B, Kv4Pool c,
                                                                  int32_t* __restrict__ shared, int32_t* __restrict__ status, ShareWork w) {
  __shared__ int s_sum[32];
  __shared__ __align__(16) int s_name[PLAN_NEAR];
  const int n_free = min(max(*c.n_free, 0), c.pages), nt = blockDim.x, lane = threadIdx.x & 31;
  int32_t* const latest = shared + c.pages;      // the last sequence that gives a page back (-1 between calls)
  claim_requests(rows, keep, true, B, c);
  int copies = 0;
  long long wanted = 0;
  for (int i0 = 0; i0 < B; i0 += nt) {
    const int i = i0 + threadIdx.x, row = i < B ? rows[i] : -1, to = i < B ? keep[i] : -1;
    const bool named = row >= 0 && row < c.requests;
    const int old = named ? c.lengths[row] : 0;
    const bool cut = claimed(i, row, named, B, c, s_name) && to >= 0 && to < old;
    const int page = cut && to % KV4_PAGE != 0 ? c.table[(size_t)row * c.width + to / KV4_PAGE] : -1;
    const int part = page >= 0 && shared[page] > 0 ? 1 : 0;
    int all;
    const long long before = wanted + block_before<int>(part, s_sum, all);
    wanted += all;
    const bool fits = part == 0 || before < n_free, copy = part != 0 && fits;
    block_before<int>(copy ? 1 : 0, s_sum, all);
    copies += all;
    if (i < B) {
      status[i] = fits ? KV4_OK : KV4_NO_PAGES;
      w.src[i] = copy ? page : -1;
      w.dst[i] = copy ? c.free[n_free - 1 - (int)before] : -1;
      w.first[i] = copy ? to / KV4_PAGE : cut ? pages_of(to) : 0;
      w.end[i] = cut && fits ? pages_of(old) : -1;
    }
  }
  __syncthreads();
  auto entries = [&](auto visit) {               // a warp a sequence: its entries that are given back
    for (int i = threadIdx.x >> 5; i < B; i += nt >> 5) {
      if (w.end[i] < 0) continue;
      const int32_t* t = c.table + (size_t)rows[i] * c.width;
      for (int k0 = w.first[i]; k0 < w.end[i]; k0 += 32) visit(i, k0 + lane < w.end[i] ? k0 + lane : -1, t);
    }
    __syncthreads();
  };
  entries([&](int i, int k, const int32_t* t) {
    if (k < 0) return;
    atomicSub(&shared[t[k]], 1);
    atomicMax(&latest[t[k]], i);
  });
  // (counters that atomics have changed are read past L1)
  auto frees = [&](int i, int page) { return __ldcg(&shared[page]) < 0 && __ldcg(&latest[page]) == i; };
  for (int i = threadIdx.x; i < B; i += nt) w.freed[i] = 0;
  __syncthreads();
  entries([&](int i, int k, const int32_t* t) {
    const uint32_t with = __ballot_sync(0xffffffffu, k >= 0 && frees(i, t[max(k, 0)]));
    if (lane == 0) w.freed[i] += __popc(with);
  });
  int total = 0;
  for (int i0 = 0; i0 < B; i0 += nt) {
    const int i = i0 + threadIdx.x, n = i < B ? w.freed[i] : 0;
    int all;
    const int before = total + block_before<int>(n, s_sum, all);
    total += all;
    if (i < B) w.freed[i] = before;
  }
  __syncthreads();
  const int top = n_free - copies + total - 1;
  entries([&](int i, int k, const int32_t* t) {
    const bool mine = k >= 0 && frees(i, t[max(k, 0)]);
    const uint32_t with = __ballot_sync(0xffffffffu, mine);
    const int at = top - w.freed[i] - __popc(with & ((1u << lane) - 1u));
    if (mine && at >= 0 && at < c.pages) c.free[at] = t[k];
    __syncwarp();
    if (lane == 0) w.freed[i] += __popc(with);
    __syncwarp();
  });
  entries([&](int i, int k, const int32_t* t) {
    if (k < 0) return;
    atomicMax(&shared[t[k]], 0);
    latest[t[k]] = -1;
    const_cast<int32_t*>(t)[k] = -1;
  });
  for (int i = threadIdx.x; i < B; i += nt) {
    if (w.end[i] < 0) continue;
    if (w.dst[i] >= 0) c.table[(size_t)rows[i] * c.width + w.first[i]] = w.dst[i];
    c.lengths[rows[i]] = keep[i];
  }
  if (threadIdx.x == 0) *c.n_free = min(max(n_free - copies + total, 0), c.pages);
}

// Pages src[i] to dst[i], all layers: a block 16 kB of one.
constexpr int COPY_THREADS = 256, COPY_BLOCK = 4 * COPY_THREADS;      // threads, vectors of 16 bytes
__global__ void __launch_bounds__(COPY_THREADS) kv4_copy_kernel(uint4* __restrict__ blocks, long long layer, int page, const int32_t* __restrict__ src,
                                                               const int32_t* __restrict__ dst) {
  const int from = src[blockIdx.x], to = dst[blockIdx.x];
  if (from < 0 || to < 0) return;
  const uint4* a = blocks + blockIdx.z * layer + (long long)from * page;
  uint4* b = blocks + blockIdx.z * layer + (long long)to * page;
  const int at = blockIdx.y * COPY_BLOCK + threadIdx.x;
  uint4 v[4];
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (at + k * COPY_THREADS < page) v[k] = a[at + k * COPY_THREADS];
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (at + k * COPY_THREADS < page) b[at + k * COPY_THREADS] = v[k];
}

int copy_pages(const ll_kv4_cache* c, void* blocks, int layers, const ShareWork& w, int B, cudaStream_t st) {
  const long long page = (long long)c->kv_heads * kv4_bytes(c->head_size, c->head_size / c->group) / 16;
  const dim3 grid(B, (unsigned)((page + COPY_BLOCK - 1) / COPY_BLOCK), layers);
  kv4_copy_kernel<<<grid, COPY_THREADS, 0, st>>>((uint4*)blocks, page * c->pages, (int)page, w.src, w.dst);
  LL_LAUNCH_OK("kv4_copy_kernel");
  return LL_OK;
}
int check_share(const ll_kv4_cache* c, const void* blocks, int layers, const void* shared, const void* a, const void* b, int B, const void* status, const void* work,
                const char* who) {
  if (int r = check_cache(c, who)) return r;
  LL_CHECK_ARG(blocks && shared && a && b && status && work && B > 0 && layers > 0 && layers <= 65535 && ((uintptr_t)blocks & 15) == 0,
               "%s: %d sequences, %d layers", who, B, layers);
  LL_CHECK_ARG((long long)c->kv_heads * kv4_bytes(c->head_size, c->head_size / c->group) / 16 <= 65535ll * COPY_BLOCK, "%s: %d heads of %d", who, c->kv_heads, c->head_size);
  return LL_OK;
}

}  // namespace
}  // namespace llb

using namespace llb;

extern "C" {

int ll_kv4_fork(const ll_kv4_cache* cache, void* blocks, int layers, int32_t* shared, const int32_t* rows, const int32_t* into, int B, int32_t* status, int32_t* work,
                ll_stream stream) {
  if (int r = check_share(cache, blocks, layers, shared, rows, into, B, status, work, "kv4_fork")) return r;
  const ShareWork w(work, B);
  kv4_fork_kernel<<<1, B <= 32 ? 256 : PLAN_THREADS, 0, (cudaStream_t)stream>>>(rows, into, B, pool_of(cache), shared, status, w);
  LL_LAUNCH_OK("kv4_fork_kernel");
  return copy_pages(cache, blocks, layers, w, B, (cudaStream_t)stream);
}

int ll_kv4_release(const ll_kv4_cache* cache, void* blocks, int layers, int32_t* shared, const int32_t* rows, const int32_t* keep, int B, int32_t* status, int32_t* work,
                   ll_stream stream) {
  if (int r = check_share(cache, blocks, layers, shared, rows, keep, B, status, work, "kv4_release")) return r;
  const ShareWork w(work, B);
  kv4_release_kernel<<<1, B <= 32 ? 256 : PLAN_THREADS, 0, (cudaStream_t)stream>>>(rows, keep, B, pool_of(cache), shared, status, w);
  LL_LAUNCH_OK("kv4_release_kernel");
  return copy_pages(cache, blocks, layers, w, B, (cudaStream_t)stream);
}

}  // extern "C"
