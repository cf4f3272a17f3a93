// Requests of the paged cache that share pages: copies of a request (fork), cuts into pages that others hold, and the copies of pages that both need.
//
// A page that a request still writes, its last one while that is not full, is the request's own: so neither a plan nor an append asks who else holds a page.
// A fork shares the whole pages and copies a last one that is not full; a cut that ends inside a page which others hold copies that one.  shared[p] counts the
// holders of page p beyond the first one (0 for free pages and for a request's own), so that a plan, which gives out free pages, need not know of it.
#include <algorithm>

#include "paged_pool.cuh"

namespace llb {
namespace {

// What a call notes: of its sequences, [B] each, entries of the table that are shared or given back and a number of tokens (-1: nothing to do); and its copies of pages,
// one after the other, their number behind them.
struct ShareWork {
  int32_t *first, *end, *tokens, *src, *dst, *copies;
  int B;
  __host__ __device__ ShareWork(int32_t* w, int B)
      : first(w), end(w + B), tokens(w + 2 * (size_t)B), src(w + 3 * (size_t)B), dst(w + 4 * (size_t)B), copies(w + 5 * (size_t)B), B(B) {}
};

// The entries of a round of sequences (as many as the block has threads), one after the other: a thread has SHARE_EACH neighbours, whichever sequences these are of.
// What bounds both kernels are dependent loads, atomics and sums of one block; with a warp a sequence, 203 sequences of 17 entries each, a fork took 11 us and a cut 27, now
// 10 and 17.
constexpr int SHARE_EACH = 4;
struct ShareRound {
  int sum[32], row[PLAN_THREADS], first[PLAN_THREADS], at[PLAN_THREADS + 1];
};
// Threads bring their sequence's request (or -1), first entry and number of entries; returns the entries of all.
__device__ __forceinline__ int round_entries(ShareRound& s, int row, int first, int n) {
  int all;
  const int before = block_before<int>(n, s.sum, all);
  s.row[threadIdx.x] = row;
  s.first[threadIdx.x] = first;
  s.at[threadIdx.x] = before;
  if (threadIdx.x == 0) s.at[blockDim.x] = all;
  __syncthreads();
  return all;
}
// Entries e0 .. e0 + SHARE_EACH - 1: their sequences in the round, and their places in the tables.
__device__ __forceinline__ void find_entries(const ShareRound& s, int e0, int all, int (&seq)[SHARE_EACH], int (&entry)[SHARE_EACH]) {
  int lo = 0, hi = blockDim.x;                   // the last sequence that begins at e0 or before it, and has entries
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (s.at[mid + 1] > e0) hi = mid;
    else lo = mid + 1;
  }
#pragma unroll
  for (int q = 0; q < SHARE_EACH; ++q) {
    const int e = e0 + q;
    if (e < all)
      while (s.at[lo + 1] <= e) ++lo;
    seq[q] = e < all ? lo : -1;
    entry[q] = e < all ? s.first[lo] + e - s.at[lo] : 0;
  }
}

// Empty requests into[i] become copies of rows[i], both as they are before the call.
__global__ void __launch_bounds__(PLAN_THREADS) kv4_fork_kernel(const int32_t* __restrict__ rows, const int32_t* __restrict__ into, Kv4Pool c,
                                                               int32_t* __restrict__ shared, int32_t* __restrict__ status, ShareWork w) {
  __shared__ ShareRound s;
  __shared__ int s_to[PLAN_THREADS];
  __shared__ __align__(16) int s_name[PLAN_NEAR];
  const int n_free = min(max(*c.n_free, 0), c.pages), nt = blockDim.x, B = w.B;
  claim_requests(into, into, true, B, c);
  long long wanted = 0;
  int given = 0;
  for (int i0 = 0; i0 < B; i0 += nt) {
    const int i = i0 + threadIdx.x, from = i < B ? rows[i] : -1, to = i < B ? into[i] : -1;
    const bool named = to >= 0 && to < c.requests && from >= 0 && from < c.requests;
    const bool mine = claimed(i, to, to >= 0 && to < c.requests, B, c, s_name) && named && c.lengths[max(to, 0)] == 0;
    const int held = mine ? c.lengths[from] : 0, whole = held / KV4_PAGE, part = held % KV4_PAGE != 0 ? 1 : 0;
    int all;
    const long long before = wanted + block_before<int>(part, s.sum, all);
    wanted += all;
    const bool fits = part == 0 || before < n_free, ok = mine && fits, copy = ok && part != 0;
    given += __syncthreads_count(copy);
    if (copy) {                                  // (all that wanted a page before have one)
      const int page = c.free[n_free - 1 - (int)before];
      w.src[before] = c.table[(size_t)from * c.width + whole];
      w.dst[before] = page;
      c.table[(size_t)to * c.width + whole] = page;
    }
    if (i < B) {
      status[i] = !mine ? KV4_BAD_ROW : fits ? KV4_OK : KV4_NO_PAGES;
      w.tokens[i] = ok ? held : 0;
    }
    s_to[threadIdx.x] = to;
    const int entries = round_entries(s, from, 0, ok ? whole : 0);
    for (int e0 = SHARE_EACH * threadIdx.x; e0 < entries; e0 += SHARE_EACH * nt) {
      int seq[SHARE_EACH], entry[SHARE_EACH], page[SHARE_EACH];
      find_entries(s, e0, entries, seq, entry);
#pragma unroll
      for (int q = 0; q < SHARE_EACH; ++q)
        if (seq[q] >= 0) page[q] = c.table[(size_t)s.row[seq[q]] * c.width + entry[q]];
#pragma unroll
      for (int q = 0; q < SHARE_EACH; ++q)
        if (seq[q] >= 0) {
          c.table[(size_t)s_to[seq[q]] * c.width + entry[q]] = page[q];
          atomicAdd(&shared[page[q]], 1);
        }
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) *c.n_free = n_free - given, *w.copies = given;
  for (int i = threadIdx.x; i < B; i += nt)      // (lengths change when all have been read: a request may be a copy and have one that names it)
    if (w.tokens[i] > 0) c.lengths[into[i]] = w.tokens[i];
}

// Requests are cut to `keep` tokens.  All decisions are taken on the pool as it is before the call: a cut inside a page that others hold needs a free page
// for its copy, and is refused where there is none.  A page goes back to the stack when its last holder has given it back, in the order of the sequences, and
// by the last of those that give it back in one call: whoever comes first makes no difference.
__global__ void __launch_bounds__(PLAN_THREADS) kv4_release_kernel(const int32_t* __restrict__ rows, const int32_t* __restrict__ keep, Kv4Pool c,
                                                                  int32_t* __restrict__ shared, int32_t* __restrict__ status, ShareWork w) {
  __shared__ ShareRound s;
  __shared__ int s_freed;
  __shared__ __align__(16) int s_name[PLAN_NEAR];
  const int n_free = min(max(*c.n_free, 0), c.pages), nt = blockDim.x, B = w.B;
  int32_t* const latest = shared + c.pages;      // the last sequence that gives a page back (-1 between calls)
  claim_requests(rows, keep, true, B, c);
  if (threadIdx.x == 0) s_freed = 0;
  int copies = 0, row = -1, first = 0, end = -1, to = -1;
  long long wanted = 0;
  for (int i0 = 0; i0 < B; i0 += nt) {
    const int i = i0 + threadIdx.x;
    row = i < B ? rows[i] : -1, to = i < B ? keep[i] : -1;
    const bool named = row >= 0 && row < c.requests;
    const int old = named ? c.lengths[row] : 0;
    const bool cut = claimed(i, row, named, B, c, s_name) && to >= 0 && to < old;
    const int page = cut && to % KV4_PAGE != 0 ? c.table[(size_t)row * c.width + to / KV4_PAGE] : -1;
    const int part = page >= 0 && shared[page] > 0 ? 1 : 0;
    int all;
    const long long before = wanted + block_before<int>(part, s.sum, all);
    wanted += all;
    const bool fits = part == 0 || before < n_free, copy = part != 0 && fits;
    copies += __syncthreads_count(copy);
    if (copy) w.src[before] = page, w.dst[before] = c.free[n_free - 1 - (int)before];      // (all that wanted a page before have one)
    first = copy ? to / KV4_PAGE : pages_of(max(to, 0));
    end = cut && fits ? pages_of(old) : -1;
    if (i < B) {
      status[i] = fits ? KV4_OK : KV4_NO_PAGES;
      w.first[i] = first;
      w.end[i] = end;
      w.tokens[i] = copy ? (int)before : -1;
    }
  }
  if (threadIdx.x == 0) *w.copies = copies;
  __syncthreads();
  // the rounds' entries that are given back: visit(sequences, places in the table, pages) of SHARE_EACH a thread
  int entries = 0, round0 = 0;
  auto rounds = [&](bool again, auto visit) {
    for (int i0 = 0; i0 < B; i0 += nt) {
      round0 = i0;
      if (B > nt || !again) {                    // (one round's entries are still there)
        const int i = i0 + threadIdx.x;
        const int f = B <= nt ? first : i < B ? w.first[i] : 0, l = B <= nt ? end : i < B ? w.end[i] : -1;
        entries = round_entries(s, B <= nt ? row : i < B ? rows[i] : -1, f, max(l - f, 0));
      }
      for (int b0 = 0; b0 < entries; b0 += SHARE_EACH * nt) {
        int seq[SHARE_EACH], entry[SHARE_EACH], page[SHARE_EACH];
        find_entries(s, b0 + SHARE_EACH * threadIdx.x, entries, seq, entry);
#pragma unroll
        for (int q = 0; q < SHARE_EACH; ++q) page[q] = seq[q] >= 0 ? c.table[(size_t)s.row[seq[q]] * c.width + entry[q]] : -1;
        visit(seq, entry, page);
      }
      __syncthreads();
    }
  };
  int freed = 0;
  rounds(false, [&](const int(&seq)[SHARE_EACH], const int(&)[SHARE_EACH], const int(&page)[SHARE_EACH]) {
#pragma unroll
    for (int q = 0; q < SHARE_EACH; ++q)
      if (page[q] >= 0) {
        freed += atomicSub(&shared[page[q]], 1) == 0 ? 1 : 0;      // (one of a page that becomes free meets this)
        atomicMax(&latest[page[q]], round0 + seq[q]);
      }
  });
  if (freed > 0) atomicAdd(&s_freed, freed);
  __syncthreads();
  const int total = s_freed;
  int top = n_free - copies + total - 1;
  rounds(true, [&](const int(&seq)[SHARE_EACH], const int(&entry)[SHARE_EACH], const int(&page)[SHARE_EACH]) {
    // (counters that atomics have changed are read past L1; who gives a page back last sets them back, which makes no difference to the others)
    bool last[SHARE_EACH], free[SHARE_EACH];
    int n = 0;
#pragma unroll
    for (int q = 0; q < SHARE_EACH; ++q) {
      last[q] = page[q] >= 0 && __ldcg(&latest[max(page[q], 0)]) == round0 + seq[q];
      free[q] = last[q] && __ldcg(&shared[max(page[q], 0)]) < 0;
      n += free[q] ? 1 : 0;
    }
    int all;
    int at = top - block_before<int>(n, s.sum, all);
    top -= all;
#pragma unroll
    for (int q = 0; q < SHARE_EACH; ++q) {
      if (free[q]) {
        if (at >= 0 && at < c.pages) c.free[at] = page[q];
        --at;
        shared[page[q]] = 0;
      }
      if (last[q]) latest[page[q]] = -1;
      if (page[q] >= 0) c.table[(size_t)s.row[seq[q]] * c.width + entry[q]] = -1;
    }
  });
  for (int i = threadIdx.x; i < B; i += nt) {
    if (w.end[i] < 0) continue;
    if (w.tokens[i] >= 0) c.table[(size_t)rows[i] * c.width + w.first[i]] = w.dst[w.tokens[i]];
    c.lengths[rows[i]] = keep[i];
  }
  if (threadIdx.x == 0) *c.n_free = min(max(n_free - copies + total, 0), c.pages);
}

// The copies, all layers: blocks take 16 kB of one each, copies of a page next to one another.  203 copies of pages of 41 kB in five layers: 9 us for 43 MB.
constexpr int COPY_THREADS = 256, COPY_BLOCK = 4 * COPY_THREADS;      // threads, vectors of 16 bytes
__global__ void __launch_bounds__(COPY_THREADS) kv4_copy_kernel(uint4* __restrict__ blocks, long long layer, int page, int layers, ShareWork w) {
  pdl_wait();
  const int copies = *after_wait(w.copies), parts = (page + COPY_BLOCK - 1) / COPY_BLOCK;
  const int32_t *src = after_wait(w.src), *dst = after_wait(w.dst);
  const long long units = (long long)copies * parts * layers;
  for (long long u = blockIdx.x; u < units; u += gridDim.x) {
    const int i = (int)(u % copies), part = (int)(u / copies % parts), l = (int)(u / copies / parts);
    const uint4* a = blocks + l * layer + (long long)src[i] * page;
    uint4* b = blocks + l * layer + (long long)dst[i] * page;
    const int at = part * COPY_BLOCK + threadIdx.x;
    uint4 v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (at + k * COPY_THREADS < page) v[k] = a[at + k * COPY_THREADS];
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (at + k * COPY_THREADS < page) b[at + k * COPY_THREADS] = v[k];
  }
}

int copy_pages(const ll_kv4_cache* c, void* blocks, int layers, const ShareWork& w, cudaStream_t st) {
  const long long page = (long long)c->kv_heads * kv4_bytes(c->head_size, c->head_size / c->group) / 16;
  const long long units = (page + COPY_BLOCK - 1) / COPY_BLOCK * layers * w.B;
  const int sms = sm_count() > 0 ? sm_count() : 148;
  LL_CUDA(launch(kv4_copy_kernel, dim3((unsigned)std::min<long long>(units, 8ll * sms)), dim3(COPY_THREADS), 0, st, true, (uint4*)blocks, page * c->pages, (int)page, layers, w));
  LL_LAUNCH_OK("kv4_copy_kernel");
  return LL_OK;
}
int check_share(const ll_kv4_cache* c, const void* blocks, int layers, const void* shared, const void* a, const void* b, int B, const void* status, const void* work,
                const char* who) {
  if (int r = check_cache(c, who)) return r;
  LL_CHECK_ARG(blocks && shared && a && b && status && work && B > 0 && layers > 0 && layers <= 65535 && ((uintptr_t)blocks & 15) == 0,
               "%s: %d sequences, %d layers", who, B, layers);
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
  kv4_fork_kernel<<<1, B <= 64 ? 256 : PLAN_THREADS, 0, (cudaStream_t)stream>>>(rows, into, pool_of(cache), shared, status, w);
  LL_LAUNCH_OK("kv4_fork_kernel");
  return copy_pages(cache, blocks, layers, w, (cudaStream_t)stream);
}

int ll_kv4_release(const ll_kv4_cache* cache, void* blocks, int layers, int32_t* shared, const int32_t* rows, const int32_t* keep, int B, int32_t* status, int32_t* work,
                   ll_stream stream) {
  if (int r = check_share(cache, blocks, layers, shared, rows, keep, B, status, work, "kv4_release")) return r;
  const ShareWork w(work, B);
  kv4_release_kernel<<<1, B <= 64 ? 256 : PLAN_THREADS, 0, (cudaStream_t)stream>>>(rows, keep, pool_of(cache), shared, status, w);
  LL_LAUNCH_OK("kv4_release_kernel");
  return copy_pages(cache, blocks, layers, w, (cudaStream_t)stream);
}

}  // extern "C"
