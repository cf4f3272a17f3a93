// The paged key/value cache in 4 bits: which pages and slots a step's tokens get, how they give them back, and the rounding of keys and values into
// their slots.  Layout: kv4.cuh; the attention that reads it: paged_attn.cu, paged_prompt.cu.
//
// A plan is a chain of dependent loads, sums and stores of one block: 64 requests 11 us, with the division of the step's attention (4 of them), 200 prompts of
// 182 000 tokens 36 and 5 for the tokens' grid.  It is made once a step and serves all layers.
#include <climits>

#include "paged_pool.cuh"
#include "paged_work.cuh"

namespace llb {
namespace {

struct Kv4Plan {
  int32_t* starts;     // [B + 1]
  int32_t* ends;       // [B]
  int32_t* status;     // [B]
  int32_t* request;    // [B] the request, or -1 where a sequence is refused
  int32_t* positions;  // [T]
  int32_t* slots;      // [T]
};

constexpr int PLAN_HELD = 1024;      // sequences whose numbers the block holds

// What the sequences of a step came to: in shared memory where there is room, else where the plan keeps it.
struct PlanView {
  static constexpr bool SHARED = false;
  const int32_t *starts, *ends, *request;
  int B;
  __device__ __forceinline__ int tokens(int i) const { return starts[i + 1] - starts[i]; }
  __device__ __forceinline__ int4 place(int i) const { return make_int4(request[i], starts[i], tokens(i), ends[i] - tokens(i)); }
};

// Walks of a step whose sequences share pages.  0 .. B - 1: the sequences, from the first page on that is theirs alone; B ..: groups of sequences that follow one
// another, over the pages that all of them have, for all of their columns.  Of the groups those count that `most` columns lie on one side of.
struct ShareView {
  static constexpr bool SHARED = true;
  PlanView v;
  const int32_t *first_page, *group_first, *group_last;      // [v.B], [groups] first and last sequence
  int2* note;                                                // [B] parts of a walk (of each of its tiles), and where they are kept
  int B, R, most;
  bool larger;
  __device__ __forceinline__ int tokens(int i) const {
    if (i < v.B) return larger || v.request[i] < 0 ? 0 : v.tokens(i);      // (refused ones: kv4_join_shared_kernel)
    const int n = v.starts[group_last[i - v.B] + 1] - v.starts[group_first[i - v.B]];
    return ((long long)n * R > most) == larger ? n : 0;
  }
  __device__ __forceinline__ int shared_pages(int i) const { return first_page[group_last[i - v.B]]; }
  __device__ __forceinline__ int from(int i) const { return i < v.B ? first_page[i] : 0; }
  __device__ __forceinline__ int pages(int i) const {
    if (i >= v.B) return shared_pages(i);
    return (v.ends[i] - 1) / KV4_PAGE + 1 - first_page[i];
  }
  __device__ __forceinline__ int4 place(int i) const {
    if (i < v.B) return v.place(i);
    const int g = group_first[i - v.B];                      // (behind all of these pages' keys)
    return make_int4(v.request[g], v.starts[g], tokens(i), shared_pages(i) * KV4_PAGE);
  }
  // parts that say whether an item's sums are the result: those of groups and of their sequences never are
  __device__ __forceinline__ int parts(int i, int k) const { return i >= v.B || first_page[i] > 0 ? max(k, 2) : k; }
};

// First sequence that ends behind token t (B: none).
__device__ __forceinline__ int sequence_of(const PlanView& v, int t) {
  int lo = 0, hi = v.B;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (v.starts[mid + 1] > t) hi = mid;
    else lo = mid + 1;
  }
  return lo;
}
// position and slot of token t
__device__ __forceinline__ void place_token(const PlanView& v, const Kv4Pool& c, const Kv4Plan& p, int t) {
  const int i = sequence_of(v, t);
  int pos = -1, slot = -1, row;
  if (i < v.B && (row = v.request[i]) >= 0) {
    pos = v.ends[i] - (v.starts[i + 1] - t);
    slot = c.table[(size_t)row * c.width + pos / KV4_PAGE] * KV4_PAGE + pos % KV4_PAGE;
  }
  p.positions[t] = pos;
  p.slots[t] = slot;
}

// ---- the division of a step's attention
struct PlanWork {
  int R, few, cols, longest;           // columns a token, most columns of the few, columns of a tile; most pages of a request
  int parts, max_items, max_joins;     // places for blocks (a key head), items and joins there is room for
  float fixed, joined;                 // what a part costs beside its pages, and what parts that have to be joined cost the step, in pages
  bool cut;                            // whether walks may be cut
  int32_t* work;
  int cuts = KV4_CUTS;                 // how many rounds of parts cuts may add
};
constexpr int PW_SIZES = 512;          // sizes of parts told apart (where there are more, by twos, fours and so on)
constexpr int PW_TRIES = 48;

// Parts of `step` pages at most, every walk in equal ones.  Parts of a size stand together, the largest first: blocks take them in that order, and the
// short ones fill the end.  step is the one of PW_TRIES that leaves the step the shortest, by what such an order comes to: the load a place, and
// of the round that is not full the time of the shortest parts, but no less than the longest part.  Walks for several rounds even out by
// themselves and stay whole.
// MANY false: the sequences of up to `few` columns, whose tiles count as long as the last one; true: the others.
template <bool MANY, class View>
__device__ __forceinline__ void divide_work(const View& v, const PlanWork& d, int* s_count, int* s_size, int2* s_walk) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  auto tokens = [&](int i) { return v.tokens(i); };
  auto tiles = [&](int i) {
    const uint32_t c = (uint32_t)tokens(i) * (uint32_t)d.R;          // (tokens times heads fit 31 bits)
    return (c > (uint32_t)d.few) == MANY ? (int)((c + (uint32_t)d.cols - 1) / (uint32_t)d.cols) : 0;
  };
  // pages that a tile's last column sees
  auto pages = [&](int i, int tile) {
    if constexpr (View::SHARED) return v.pages(i);
    else if (v.request[i] < 0) return 1;
    else {
    const int n = tokens(i);
    return (v.ends[i] - n + (MANY ? min(n - 1, (int)(((uint32_t)(tile + 1) * (uint32_t)d.cols - 1) / (uint32_t)d.R)) : n - 1)) / KV4_PAGE + 1;
    }
  };
  // tiles of the sequences, and pages of their last one, where the block can hold them; all walks
  const bool held = v.B <= PLAN_HELD;
  __syncthreads();
  if (threadIdx.x == 0) s_count[0] = 0;
  __syncthreads();
  for (int i0 = 0; i0 < v.B; i0 += blockDim.x) {
    const int i = i0 + threadIdx.x, w = i < v.B ? tiles(i) : 0, n = __reduce_add_sync(0xffffffffu, w);
    if (held && i < v.B) s_walk[i] = make_int2(w, w > 0 ? pages(i, w - 1) : 0);
    if (lane == 0 && n > 0) atomicAdd(&s_count[0], n);
  }
  __syncthreads();
  const int walks = s_count[0];
  __syncthreads();                     // (the word counts the joins next: every warp has read the walks)
  auto walk_of = [&](int i) {
    if (held) return s_walk[i];
    const int w = tiles(i);
    return make_int2(w, w > 0 ? pages(i, w - 1) : 0);
  };
  if (walks == 0) {
    if (threadIdx.x == 0) d.work[0] = d.work[1] = 0;
    return;
  }
  int step = d.longest;
  if (d.cut && walks < KV4_ROUNDS * d.parts) {
    // how long the step takes with parts of `step` pages at most, by one warp
    auto length = [&](int step) {
      int n = 0, sum = 0, most = 0, least = INT_MAX;
      auto add = [&](int w, int p) {
        const int k = (p + step - 1) / step, each = (p + k - 1) / k;
        n += w * k, sum += w * p, most = max(most, each), least = min(least, each);
      };
      for (int i0 = 0; i0 < v.B; i0 += 32) {
        const int2 wp = i0 + lane < v.B ? walk_of(i0 + lane) : make_int2(0, 0);
        const int w = wp.x;
        if (MANY) {
          for (uint32_t with = __ballot_sync(0xffffffffu, w > 0); with != 0u; with &= with - 1) {
            const int l = __ffs(with) - 1, all = __shfl_sync(0xffffffffu, w, l);
            for (int t = lane; t < all; t += 32) add(1, pages(i0 + l, t));
          }
        } else if (w > 0) {
          add(w, wp.y);
        }
      }
      n = __reduce_add_sync(0xffffffffu, n), sum = __reduce_add_sync(0xffffffffu, sum);
      most = __reduce_max_sync(0xffffffffu, most), least = __reduce_min_sync(0xffffffffu, least);
      const int rounds = (n + d.parts - 1) / d.parts;
      const float load = (sum + n * d.fixed) / d.parts + (rounds - (float)n / d.parts) * (least + d.fixed);
      return n > walks + d.cuts * d.parts ? 1e30f : fmaxf(load, most + d.fixed) + (n > walks ? d.joined : 0.f);
    };
    // the longest walk in 1, 2 .. 24, then 30, 36, 42, 48, 60 .. parts
    auto tried = [&](int k) {
      const int c = k < 24 ? k + 1 : 6 * (4 + ((k - 24) & 3)) << ((k - 24) >> 2);
      return max(1, (d.longest + c - 1) / c);
    };
    float best = 1e30f;
    int mine = 0;
    for (int k = warp; k < PW_TRIES; k += warps) {
      if (k > 0 && tried(k) == tried(k - 1)) continue;
      const float f = length(tried(k));
      if (f < best) best = f, mine = k;
    }
    __syncthreads();
    if (lane == 0) s_count[warp] = __float_as_int(best), s_size[warp] = mine;      // (not negative: the bits rise with it)
    __syncthreads();
    int at = 0;
    for (int w = 1; w < warps; ++w)
      if (s_count[w] < s_count[at] || (s_count[w] == s_count[at] && s_size[w] < s_size[at])) at = w;
    step = tried(s_size[at]);
    __syncthreads();
  }
  // a walk's pages in equal parts; the places of the sizes, counted and summed from the largest down
  auto cut = [&](int p) { return (p + step - 1) / step; };
  int shift = 0;
  while ((step - 1) >> shift >= PW_SIZES) ++shift;
  auto bucket = [&](int size) { return PW_SIZES - 1 - ((min(size, step) - 1) >> shift); };
  for (int x = threadIdx.x; x < PW_SIZES; x += blockDim.x) s_size[x] = 0;
  if (threadIdx.x == 0) s_count[0] = 0;
  __syncthreads();
  for (int i = MANY ? warp : threadIdx.x; i < v.B; i += MANY ? warps : blockDim.x) {
    const int2 wp = walk_of(i);
    const int w = wp.x;
    for (int t = MANY ? lane : 0; t < (MANY ? w : min(w, 1)); t += 32) {
      const int p = MANY ? pages(i, t) : wp.y, k = cut(p);
      atomicAdd(&s_size[bucket((p + k - 1) / k)], MANY ? k : w * k);
    }
  }
  __syncthreads();
  if (warp == 0) {
    int mine[PW_SIZES / 32], sum = 0;
#pragma unroll
    for (int x = 0; x < PW_SIZES / 32; ++x) mine[x] = s_size[lane * (PW_SIZES / 32) + x], sum += mine[x];
    int incl = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += u;
    }
    if (lane == 31) d.work[0] = min(incl, d.max_items);
    int before = incl - sum;
#pragma unroll
    for (int x = 0; x < PW_SIZES / 32; ++x) {
      s_size[lane * (PW_SIZES / 32) + x] = before;
      before += mine[x];
    }
  }
  __syncthreads();
  // (which of the parts of one size comes first is left to chance, and of no consequence: every part has its own place for its sums)
  auto store = [&](int i, int at, int tile, int part, int each, int k, int base) {
    if (at >= d.max_items) return;
    int4* o = reinterpret_cast<int4*>(d.work) + 1 + 3 * (size_t)at;
    o[0] = v.place(i);
    if constexpr (View::SHARED) o[1] = make_int4(tile, v.from(i) + part * each, v.from(i) + min((part + 1) * each, v.pages(i)), v.parts(i, k));
    else o[1] = make_int4(tile, part * each, (part + 1) * each, k);
    o[2] = make_int4(part, base, 0, 0);
  };
  auto join = [&](int i, int tile, int k, int base) {
    if constexpr (View::SHARED) return;
    const int j = atomicAdd(&s_count[0], 1);
    if (j >= d.max_joins) return;
    int4* o = const_cast<int4*>(joins_of(d.work, d.max_items)) + 2 * (size_t)j;
    o[0] = make_int4(v.place(i).y, tokens(i), tile, k);
    o[1] = make_int4(base, 0, 0, 0);
  };
  if (MANY) {
    for (int i = warp; i < v.B; i += warps) {
      const int w = walk_of(i).x;
      for (int t = lane; t < w; t += 32) {
        const int p = pages(i, t), k = cut(p), each = (p + k - 1) / k, at = atomicAdd(&s_size[bucket(each)], k);
        for (int e = 0; e < k; ++e) store(i, at + e, t, e, each, k, at);
        if (k > 1) join(i, t, k, at);
      }
    }
  } else {      // a thread a sequence; its warp helps where there are more than four parts
    // (sequences are dealt out, so that every warp has some)
    const int per = min(32, (v.B + warps - 1) / warps);
    for (int i0 = per * warp; i0 < v.B; i0 += per * warps) {
      const int i = i0 + lane;
      const int2 wp = lane < per && i < v.B ? walk_of(i) : make_int2(0, 0);
      const int w = wp.x;
      int k = 0, each = 1, at = 0;
      if (w > 0) {
        const int p = wp.y;
        k = cut(p), each = (p + k - 1) / k;
        at = atomicAdd(&s_size[bucket(each)], w * k);
        if constexpr (View::SHARED) v.note[i] = make_int2(k, at);
        if (w * k <= 4)
          for (int e = 0; e < w * k; ++e) store(i, at + e, e / k, e % k, each, k, at + e / k * k);
        if (k > 1)
          for (int t = 0; t < w; ++t) join(i, t, k, at + t * k);
      }
      for (uint32_t more = __ballot_sync(0xffffffffu, w * k > 4); more != 0u; more &= more - 1) {
        const int l = __ffs(more) - 1, ww = __shfl_sync(0xffffffffu, w, l), kk = __shfl_sync(0xffffffffu, k, l), ee = __shfl_sync(0xffffffffu, each, l),
                  aa = __shfl_sync(0xffffffffu, at, l);
        for (int e = lane; e < ww * kk; e += 32) store(i0 + l, aa + e, e / kk, e % kk, ee, kk, aa + e / kk * kk);
      }
    }
  }
  __syncthreads();
  if (threadIdx.x == 0) d.work[1] = min(s_count[0], d.max_joins);
}

// A step's pages, slots (of up to `here` tokens) and division, by one block: prefix sums over the sequences.
__global__ void __launch_bounds__(PLAN_THREADS) kv4_plan_kernel(const int32_t* __restrict__ rows, const int32_t* __restrict__ counts, int B, int T, int here,
                                                               int max_count, Kv4Pool c, Kv4Plan p, PlanWork few, PlanWork many) {
  __shared__ long long s_sum[32];
  __shared__ int s_need[32], s_size[PW_SIZES];
  __shared__ int s_row[PLAN_THREADS], s_first[PLAN_THREADS], s_pages[PLAN_THREADS], s_used[PLAN_THREADS];
  __shared__ int s_starts[PLAN_HELD + 1], s_ends[PLAN_HELD], s_request[PLAN_HELD];
  __shared__ __align__(16) int s_name[PLAN_NEAR];
  __shared__ int2 s_walk[PLAN_HELD];
  const int n_free = min(max(*c.n_free, 0), c.pages), nt = blockDim.x, lane = threadIdx.x & 31;
  const bool held = B <= PLAN_HELD;
  claim_requests(rows, counts, false, B, c);
  long long tokens = 0, wanted = 0;      // of the sequences before this round
  int given = 0;
  for (int i0 = 0; i0 < B; i0 += nt) {
    const int i = i0 + threadIdx.x;
    const int row = i < B ? rows[i] : -1, count = i < B ? counts[i] : 0, n = max(count, 0);
    const bool named = row >= 0 && row < c.requests;
    const int old = named ? c.lengths[row] : 0;
    const bool mine = claimed(i, row, named && n > 0, B, c, s_name);
    long long total;
    const long long first = tokens + block_before<long long>(n, s_sum, total);
    tokens += total;
    int status = KV4_OK;
    if (count < 0 || (n > 0 && !mine)) status = KV4_BAD_ROW;
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
      const int end = (int)min(first + n, (long long)T), request = ok && n > 0 ? row : -1;
      if (i == 0) p.starts[0] = 0;
      p.starts[i + 1] = end;
      p.status[i] = status;
      p.request[i] = request;
      if (held) {
        if (i == 0) s_starts[0] = 0;
        s_starts[i + 1] = end;
        s_request[i] = request;
      }
      if (ok && n > 0) {
        c.lengths[row] = old + n;
        p.ends[i] = old + n;
        if (held) s_ends[i] = old + n;
      } else if (!ok) {
        p.ends[i] = 0;
        if (held) s_ends[i] = 0;
      }
    }
    __syncthreads();
    // the new entries of the table, a warp a sequence
    for (int j = threadIdx.x >> 5; j < min(nt, B - i0); j += nt >> 5)
      for (int k = lane; k < s_pages[j]; k += 32) c.table[(size_t)s_row[j] * c.width + s_first[j] + k] = c.free[n_free - 1 - s_used[j] - k];
    __syncthreads();
  }
  if (threadIdx.x == 0) *c.n_free = n_free - given;
  for (int i = threadIdx.x; i < B; i += nt) {      // (when all lengths are the step's: an idle sequence may name another one's request)
    if (counts[i] != 0 || p.status[i] != KV4_OK) continue;
    const int row = rows[i], end = row >= 0 && row < c.requests ? c.lengths[row] : 0;
    p.ends[i] = end;
    if (held) s_ends[i] = end;
  }
  __syncthreads();
  const PlanView v{held ? s_starts : p.starts, held ? s_ends : p.ends, held ? s_request : p.request, B};
  for (int t = threadIdx.x; t < min(T, here); t += nt) place_token(v, c, p, t);
  if (few.work == nullptr) return;                // (kv4_share_kernel divides it)
  divide_work<false>(v, few, s_need, s_size, s_walk);
  if (many.work != nullptr) divide_work<true>(v, many, s_need, s_size, s_walk);
}

// The division of a step whose sequences may share pages, by one block: neighbours that have their first pages in common, as many as the two before, are a group.
__global__ void __launch_bounds__(PLAN_THREADS) kv4_share_kernel(Kv4Pool c, Kv4Plan p, int B, PlanWork few, PlanWork many, int32_t* records) {
  __shared__ int s_need[32], s_size[PW_SIZES], s_groups;
  __shared__ int s_starts[KV4_SHARE_MOST + 1], s_ends[KV4_SHARE_MOST], s_request[KV4_SHARE_MOST];
  __shared__ int s_link[KV4_SHARE_MOST], s_page[KV4_SHARE_MOST], s_group[KV4_SHARE_MOST], s_first[KV4_SHARE_MOST / 2], s_last[KV4_SHARE_MOST / 2];
  __shared__ int2 s_walk[PLAN_HELD], s_few[KV4_SHARE_MOST + KV4_SHARE_MOST / 2], s_many[KV4_SHARE_MOST + KV4_SHARE_MOST / 2];
  pdl_wait();
  const int nt = blockDim.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, R = few.R;
  const int32_t *starts = after_wait(p.starts), *ends = after_wait(p.ends), *request = after_wait(p.request), *table = after_wait(c.table);
  for (int i = threadIdx.x; i < B; i += nt) {
    s_starts[i + 1] = starts[i + 1];
    s_ends[i] = ends[i];
    s_request[i] = request[i];
    s_page[i] = 0;
    s_group[i] = -1;
  }
  if (threadIdx.x == 0) s_starts[0] = 0, s_groups = 0;
  __syncthreads();
  // pages that a sequence has in common with the one before it that brings tokens: tables are alike up to where they part
  for (int i = warp; i < B; i += nt >> 5) {
    int link = 0;
    if (i > 0 && s_request[i] >= 0) {
      int j = i - 1;
      while (j > 0 && s_starts[j + 1] == s_starts[j]) --j;
      const int a = s_request[j], b = s_request[i];
      if (a >= 0 && s_starts[j + 1] > s_starts[j]) {
        int hi = min(s_ends[j] - (s_starts[j + 1] - s_starts[j]), s_ends[i] - (s_starts[i + 1] - s_starts[i])) / KV4_PAGE;      // whole, and before all of the step's tokens
        const int32_t *ta = table + (size_t)a * c.width, *tb = table + (size_t)b * c.width;
        while (link < hi) {                       // (the first `link` are alike, number hi is not or is of no interest)
          const int step = (hi - link - 1) / 32 + 1, at = link + (lane + 1) * step - 1;
          const uint32_t same = __ballot_sync(0xffffffffu, at < hi && ta[at] == tb[at]);
          const int n = __popc(same & ~(same + 1u));      // (from the first lane on, without a gap)
          if (n < 32) hi = min(hi, link + (n + 1) * step - 1);
          link += n * step;
        }
        if (link < KV4_SHARE_LEAST) link = 0;
      }
    }
    if (lane == 0) s_link[i] = link;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    int before = -1, groups = 0;                 // the sequence before that brings tokens
    bool open = false;                           // whether it is in a group
    for (int i = 0; i < B; ++i) {
      if (s_starts[i + 1] == s_starts[i]) continue;
      const int link = s_request[i] >= 0 ? s_link[i] : 0;
      if (link > 0 && (!open || link == s_page[before])) {
        if (!open) s_first[groups++] = before, s_group[before] = groups - 1, s_page[before] = link;
        s_group[i] = groups - 1, s_page[i] = link, s_last[groups - 1] = i, open = true;
      } else {
        open = false;
      }
      before = i;
    }
    s_groups = groups;
  }
  __syncthreads();
  const PlanView v{s_starts, s_ends, s_request, B};
  const int n = B + s_groups;
  divide_work<false>(ShareView{v, s_page, s_first, s_last, s_few, n, R, KV4_SHARE_FEW, false}, few, s_need, s_size, s_walk);
  divide_work<false>(ShareView{v, s_page, s_first, s_last, s_many, n, R, KV4_SHARE_FEW, true}, many, s_need, s_size, s_walk);
  __syncthreads();
  // what has to be joined: a sequence's parts and its group's
  if (threadIdx.x == 0) s_need[0] = s_need[1] = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < B; i += nt) {
    const int count = v.tokens(i), g = s_group[i];
    const bool refused = s_request[i] < 0;
    if (count == 0 || (!refused && g < 0 && s_few[i].x <= 1)) continue;
    const int at = atomicAdd(&s_need[0], 1);
    int4* o = reinterpret_cast<int4*>(records) + 2 * (size_t)at;
    o[0] = make_int4(s_starts[i], count, refused ? 0 : s_few[i].x, s_few[i].y);
    if (refused) {
      o[1] = make_int4(0, 0, 0, 2);
    } else if (g < 0) {
      o[1] = make_int4(0, 0, 0, 0);
      atomicMax(&s_need[1], s_few[i].x);
    } else {
      const int column = (s_starts[i] - s_starts[s_first[g]]) * R;
      const bool large = (long long)(s_starts[s_last[g] + 1] - s_starts[s_first[g]]) * R > KV4_SHARE_FEW;
      const int2 w = large ? s_many[B + g] : s_few[B + g];
      o[1] = make_int4(w.x, w.y, column, large ? 1 : 0);
      atomicMax(&s_need[1], s_few[i].x + w.x);
    }
  }
  __syncthreads();
  if (threadIdx.x == 0) few.work[1] = s_need[0], few.work[3] = s_need[1];
}

// Positions and slots of a step's tokens from `here` on.
__global__ void __launch_bounds__(256) kv4_tokens_kernel(int B, int T, int here, Kv4Pool c, Kv4Plan p) {
  pdl_wait();
  const int t = here + blockIdx.x * blockDim.x + threadIdx.x;
  if (t < T) place_token(PlanView{after_wait(p.starts), after_wait(p.ends), after_wait(p.request), B}, c, p, t);
}

// The way back: requests are cut to `keep` tokens, the pages behind go to the stack in the order that a plan would take them in again.
__global__ void __launch_bounds__(PLAN_THREADS) kv4_truncate_kernel(const int32_t* __restrict__ rows, const int32_t* __restrict__ keep, int B, Kv4Pool c) {
  __shared__ int s_sum[32];
  __shared__ int s_row[PLAN_THREADS], s_first[PLAN_THREADS], s_pages[PLAN_THREADS], s_used[PLAN_THREADS];
  __shared__ __align__(16) int s_name[PLAN_NEAR];
  const int n_free = min(max(*c.n_free, 0), c.pages), nt = blockDim.x, lane = threadIdx.x & 31;
  claim_requests(rows, keep, true, B, c);
  int total = 0, done = 0;              // the pages of all sequences have to be known before the first goes back
  for (int round = B > nt ? 0 : 1; round < 2; ++round) {
    for (int i0 = 0; i0 < B; i0 += nt) {
      const int i = i0 + threadIdx.x, row = i < B ? rows[i] : -1, to = i < B ? keep[i] : -1;
      const bool named = row >= 0 && row < c.requests;
      const int old = named ? c.lengths[row] : 0;
      const bool cut = claimed(i, row, named, B, c, s_name) && to >= 0 && to < old;
      const int first = cut ? pages_of(to) : 0, n = cut ? pages_of(old) - first : 0;
      int all;
      const int before = done + block_before<int>(n, s_sum, all);
      if (round == 0 || B <= nt) total += all;
      if (round == 0) continue;
      done += all;
      s_row[threadIdx.x] = row;
      s_first[threadIdx.x] = first;
      s_pages[threadIdx.x] = n;
      s_used[threadIdx.x] = before;
      __syncthreads();
      if (cut) c.lengths[row] = to;
      for (int j = threadIdx.x >> 5; j < min(nt, B - i0); j += nt >> 5)
        for (int k = lane; k < s_pages[j]; k += 32) {
          int32_t* e = c.table + (size_t)s_row[j] * c.width + s_first[j] + k;
          const int at = n_free + total - 1 - s_used[j] - k;
          if (at < c.pages) c.free[at] = *e;
          *e = -1;
        }
      __syncthreads();
    }
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

// the smaller of two pairs; not a number where one of two is not
__device__ __forceinline__ __nv_bfloat162 min_pair(__nv_bfloat162 a, __nv_bfloat162 b) { return __hmin2_nan(a, b); }
__device__ __forceinline__ __half2 min_pair(__half2 a, __half2 b) { return __hmin2_nan(a, b); }
template <typename T> __device__ __forceinline__ uint32_t min_bits(uint32_t a, uint32_t b) {
  typedef typename pair_of<T>::type P;
  const P r = min_pair(*reinterpret_cast<const P*>(&a), *reinterpret_cast<const P*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}

// A vector (a head of a token's queries, keys or values) takes D / 8 lanes of eight numbers each, so that a warp has the same head of 32 / (D / 8) tokens one
// after the other: APPEND_HEADS heads of queries, whose turns' numbers are then loaded once, or one of keys or values.  Queries are bound by memory (5716
// tokens of 40 heads of 128 with 8 of keys and values: 17 of 30 us, for 117 MB; with one, two and eight heads a warp 38, 31 and 36 together).  Keys and values
// are bound by their instructions (13 us for 30 MB; both of a head by one warp 12, but 31 together, and 62 tokens 6.1 instead of 5.5): so the smallest and
// largest are found in pairs ({x, -x}: one minimum for both), a code comes from a product with 1 / s, and only where that lies so near to the middle of two
// codes that its error could matter (1e-4; its error is below 4e-6) from the quotient.
constexpr int APPEND_HEADS = 4;
template <typename T, int D, int NG, bool TURN>
__global__ void __launch_bounds__(256) kv4_append_kernel(Kv4Rows in, const float* __restrict__ rope, const int32_t* __restrict__ positions,
                                                         const int32_t* __restrict__ slots, T* __restrict__ q_out, uint8_t* __restrict__ blocks, int Tn, int H, int G) {
  constexpr int LV = D / 8, TOKENS = 32 / LV, GL = LV / NG, W = D / 32;
  const int lane = threadIdx.x & 31, l = lane % LV, t = blockIdx.x * TOKENS + lane / LV, unit = blockIdx.y * 8 + (threadIdx.x >> 5);
  const int turned = TURN ? (H + APPEND_HEADS - 1) / APPEND_HEADS : 0, vec = unit - turned;
  if (vec >= 2 * G) return;
  const bool live = t < Tn, is_q = vec < 0, is_k = vec < G;
  const int pos = live ? positions[t] : -1, slot = live && !is_q ? slots[t] : -1;
  float c[8];
  if (TURN && is_k) {
    const float4* cs = reinterpret_cast<const float4*>(rope + (size_t)max(pos, 0) * D + 8 * l);
    const float4 c0 = __ldg(cs), c1 = __ldg(cs + 1);
    c[0] = c0.x, c[1] = c0.y, c[2] = c0.z, c[3] = c0.w, c[4] = c1.x, c[5] = c1.y, c[6] = c1.z, c[7] = c1.w;
  }
  auto turn = [&](uint32_t x, int j) {
    const float2 f = bits_pair<T>(x);
    return pair_bits<T>(__fsub_rn(__fmul_rn(f.x, c[2 * j]), __fmul_rn(f.y, c[2 * j + 1])), __fadd_rn(__fmul_rn(f.y, c[2 * j]), __fmul_rn(f.x, c[2 * j + 1])));
  };
  if (TURN && is_q) {
    const int h0 = unit * APPEND_HEADS;
    const T* row = (const T*)in.q + t * in.q_row + h0 * D + 8 * l;
    T* to = q_out + ((size_t)t * H + h0) * D + 8 * l;
    uint4 u[APPEND_HEADS];
#pragma unroll
    for (int h = 0; h < APPEND_HEADS; ++h) u[h] = live && h0 + h < H ? *reinterpret_cast<const uint4*>(row + h * D) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
    for (int h = 0; h < APPEND_HEADS; ++h) {
      uint4 x = make_uint4(turn(u[h].x, 0), turn(u[h].y, 1), turn(u[h].z, 2), turn(u[h].w, 3));
      if (pos < 0) x.x = x.y = x.z = x.w = pair_bits<T>(NAN, NAN);
      if (live && h0 + h < H) *reinterpret_cast<uint4*>(to + h * D) = x;
    }
    return;
  }
  const int head = is_k ? vec : vec - G;
  const T* row = (is_k ? (const T*)in.k + t * in.k_row : (const T*)in.v + t * in.v_row) + head * D + 8 * l;
  const uint4 u = live ? *reinterpret_cast<const uint4*>(row) : make_uint4(0u, 0u, 0u, 0u);
  uint32_t w[4] = {u.x, u.y, u.z, u.w};
  if (TURN && is_k) {
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = turn(w[j], j);
  }
  // smallest and largest of a group: {lo, -hi}
  uint32_t low = min_bits<T>(min_bits<T>(w[0], w[1]), min_bits<T>(w[2], w[3]));
  uint32_t high = min_bits<T>(min_bits<T>(w[0] ^ 0x80008000u, w[1] ^ 0x80008000u), min_bits<T>(w[2] ^ 0x80008000u, w[3] ^ 0x80008000u));
  low = min_bits<T>(__byte_perm(low, high, 0x5410), __byte_perm(low, high, 0x7632));
#pragma unroll
  for (int o = GL / 2; o > 0; o >>= 1) low = min_bits<T>(low, __shfl_xor_sync(0xffffffffu, low, o));
  const float2 ends = bits_pair<T>(low);
  const float lo = ends.x, hi = -ends.y;
  uint32_t params = pair_bits<T>(__fmul_rn(__fsub_rn(hi, lo), (float)(1.0 / 15.0)), lo);
  float s = bits_pair<T>(params).x;
  if (!(s < INFINITY)) {               // a group with a number that is none, or infinite, or too wide: it stands for no numbers
    params = pair_bits<T>(NAN, NAN);
    s = 0.f;
  }
  constexpr float ROUND = 12582912.f;                                   // 1.5 2^23: its sum with a small number has that rounded in the low bits
  constexpr uint32_t BITS = 0x4b400000u;
  const float inv = s > 0.f ? __frcp_rn(s) : 0.f;
  uint32_t code[8];
  float far = 0.f;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 f = bits_pair<T>(w[j]);
    const float a = fminf(__fmul_rn(__fsub_rn(f.x, lo), inv), 15.f), b = fminf(__fmul_rn(__fsub_rn(f.y, lo), inv), 15.f);
    const float x = __fadd_rn(a, ROUND), y = __fadd_rn(b, ROUND);
    far = fmaxf(far, fmaxf(fabsf(a - (x - ROUND)), fabsf(b - (y - ROUND))));
    code[2 * j] = __float_as_uint(x), code[2 * j + 1] = __float_as_uint(y);
  }
  if (!(far < 0.4999f) || !(inv < INFINITY)) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = bits_pair<T>(w[j]);
      code[2 * j] = __float_as_uint(__fadd_rn(s > 0.f ? fminf(__fdiv_rn(__fsub_rn(f.x, lo), s), 15.f) : 0.f, ROUND));
      code[2 * j + 1] = __float_as_uint(__fadd_rn(s > 0.f ? fminf(__fdiv_rn(__fsub_rn(f.y, lo), s), 15.f) : 0.f, ROUND));
    }
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) code[j] -= BITS;
  uint8_t* blk = blocks + ((size_t)(max(slot, 0) / KV4_PAGE) * G + head) * kv4_bytes(D, NG) + max(slot, 0) % KV4_PAGE / KV4_SLICE * kv4_slice_bytes(D, NG);
  const int at = max(slot, 0) % KV4_SLICE;
  if (slot >= 0 && l % GL == 0) reinterpret_cast<uint32_t*>(blk + (is_k ? kv4_k_params(D) : kv4_v_params(D, NG)))[at * NG + l / GL] = params;
  if (is_k) {
    // the lane's dimensions 8 l .. are four codes each of two chunks; the other codes of either word lie two lanes on
    uint32_t a = code[0] | code[1] << 16 | code[2] << 4 | code[3] << 20, b = code[4] | code[5] << 16 | code[6] << 4 | code[7] << 20;
    const bool up = (l & 2) != 0;
    const uint32_t other = __shfl_xor_sync(0xffffffffu, up ? a : b, 2);
    const uint32_t word = up ? other | b << 8 : a | other << 8;
    if (slot >= 0) reinterpret_cast<uint32_t*>(blk)[at * (D / 8) + (2 * (l & 1) + (up ? 1 : 0)) * W + (l >> 2)] = word;
  } else {
    // the lane has nibble l & 3 of the eight chunks; by halves between four lanes each comes to have all four nibbles of two chunks
    const int n4 = 4 * (l & 3);
    uint32_t z[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) z[j] = (code[2 * j] | code[2 * j + 1] << 16) << n4;
    const bool odd = (l & 1) != 0, up = (l & 2) != 0;
    uint32_t x0 = __shfl_xor_sync(0xffffffffu, odd ? z[0] : z[2], 1), x1 = __shfl_xor_sync(0xffffffffu, odd ? z[1] : z[3], 1);
    x0 |= odd ? z[2] : z[0];
    x1 |= odd ? z[3] : z[1];
    uint32_t x = __shfl_xor_sync(0xffffffffu, up ? x0 : x1, 2) | (up ? x1 : x0);
    const int g = 4 * (l & 1) + (l & 2);                                // x: chunk g, and chunk g + 1 in the high half
    // the two slots of a pair, where two tokens of the warp have them, are stored together: a chunk each
    const uint32_t theirs = __shfl_xor_sync(0xffffffffu, x, LV);
    const int slot2 = __shfl_xor_sync(0xffffffffu, slot, LV);
    uint8_t* to = blk + kv4_v_codes(D) + (at / 2) * D + (l >> 2) * 4;
    if (slot >= 0 && slot2 == (slot ^ 1)) {
      const bool second = (slot & 1) != 0;
      const uint32_t word = second ? __byte_perm(theirs, x, 0x7632) : __byte_perm(x, theirs, 0x5410);
      *reinterpret_cast<uint32_t*>(to + (g + (second ? 1 : 0)) * 4 * W) = word;
    } else if (slot >= 0) {
      *reinterpret_cast<uint16_t*>(to + g * 4 * W + 2 * (at & 1)) = (uint16_t)x;
      *reinterpret_cast<uint16_t*>(to + (g + 1) * 4 * W + 2 * (at & 1)) = (uint16_t)(x >> 16);
    }
  }
}

// The values that slots stand for: a warp a head of read_slots(D) slots, keys by a word (eight numbers) a lane, values by four numbers a lane that lie
// side by side, whose codes are in four chunks: loads of two bytes (from L1) and a store of eight, instead of a load and four stores of two.  5716 slots of 8
// heads of 128 in 9.9 us for 29 MB, bound by its instructions (issue 71 %; 256 / D and 1024 / D slots a warp: 10.9 and 10.7; a warp a slot with those stores 13).
constexpr int read_slots(int D) { return 512 / D; }
// a code as a number: integers are converted at an eighth of an addition's rate
__device__ __forceinline__ float code_value(uint32_t code, float2 p) {
  return __fadd_rn(__fmul_rn(__uint_as_float(0x4b000000u | (code & 15u)) - 8388608.f, p.x), p.y);
}
template <typename T, int D, int NG>
__global__ void __launch_bounds__(256) kv4_read_kernel(const uint8_t* __restrict__ blocks, const int32_t* __restrict__ slots, T* __restrict__ k_out,
                                                       T* __restrict__ v_out, int n, int G, int pages) {
  constexpr int W = D / 32, LK = 4 * W, LV = 8 * W, SLOTS = read_slots(D), KR = SLOTS * LK / 32, VR = SLOTS * LV / 32;
  const int lane = threadIdx.x & 31;
  const long long vec = (long long)blockIdx.x * 8 + (threadIdx.x >> 5), t0 = vec / G * SLOTS;
  if (t0 >= n) return;
  const int head = (int)(vec % G), mine = lane < SLOTS && t0 + lane < n ? slots[t0 + lane] : -1;
  uint32_t kw[KR], vw[VR];
  float2 kp[KR], vp[VR];
  auto slice = [&](int slot) {
    return blocks + ((size_t)(slot / KV4_PAGE) * G + head) * kv4_bytes(D, NG) + slot % KV4_PAGE / KV4_SLICE * kv4_slice_bytes(D, NG);
  };
  auto params = [&](const uint8_t* at, bool there) { return there ? bits_pair<T>(*reinterpret_cast<const uint32_t*>(at)) : make_float2(NAN, NAN); };
  const int kl = lane % LK, ki = kl % W, kc = kl / W;              // keys: word ki of chunk kc, eight dimensions
  const int vl = lane % LV, vi = vl >> 3, vg = 4 * (vl & 1), vm = (vl >> 1) & 3;      // values: nibble vm of word vi of chunks vg .. vg + 3
#pragma unroll
  for (int r = 0; r < KR; ++r) {
    int slot = __shfl_sync(0xffffffffu, mine, r * (32 / LK) + lane / LK);
    const bool there = slot >= 0 && slot < pages * KV4_PAGE;
    slot = there ? slot : 0;
    const uint8_t* s = slice(slot);
    kw[r] = reinterpret_cast<const uint32_t*>(s)[slot % KV4_SLICE * (D / 8) + kl];
    kp[r] = params(s + kv4_k_params(D) + 4 * (slot % KV4_SLICE * NG + ki * NG / W), there);
  }
#pragma unroll
  for (int r = 0; r < VR; ++r) {
    int slot = __shfl_sync(0xffffffffu, mine, r * (32 / LV) + lane / LV);
    const bool there = slot >= 0 && slot < pages * KV4_PAGE;
    slot = there ? slot : 0;
    const uint8_t* s = slice(slot);
    const int at = slot % KV4_SLICE;
    const uint16_t* c = reinterpret_cast<const uint16_t*>(s + kv4_v_codes(D)) + (at / 2) * (D / 2) + (vg * W + vi) * 2 + (at & 1);
    vw[r] = 0;
#pragma unroll
    for (int g = 0; g < 4; ++g) vw[r] |= ((uint32_t)c[2 * g * W] >> (4 * vm) & 15u) << (8 * g);
    vp[r] = params(s + kv4_v_params(D, NG) + 4 * (at * NG + vi * NG / W), there);
  }
#pragma unroll
  for (int r = 0; r < KR; ++r) {
    const long long t = t0 + r * (32 / LK) + lane / LK;
    if (t >= n) continue;
    T* to = k_out + (t * G + head) * D + 32 * ki + 4 * kc;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t w = kw[r] >> (8 * h);
      *reinterpret_cast<uint2*>(to + 16 * h) = make_uint2(pair_bits<T>(code_value(w, kp[r]), code_value(w >> 16, kp[r])),
                                                          pair_bits<T>(code_value(w >> 4, kp[r]), code_value(w >> 20, kp[r])));
    }
  }
#pragma unroll
  for (int r = 0; r < VR; ++r) {
    const long long t = t0 + r * (32 / LV) + lane / LV;
    if (t >= n) continue;
    *reinterpret_cast<uint2*>(v_out + (t * G + head) * D + 4 * vl) = make_uint2(pair_bits<T>(code_value(vw[r], vp[r]), code_value(vw[r] >> 8, vp[r])),
                                                                               pair_bits<T>(code_value(vw[r] >> 16, vp[r]), code_value(vw[r] >> 24, vp[r])));
  }
}

}  // namespace
}  // namespace llb

using namespace llb;

extern "C" {

size_t ll_kv4_page_bytes(int head_size, int group) { return kv4_shape_ok(head_size, group) ? (size_t)kv4_bytes(head_size, head_size / group) : 0; }

static size_t work_ints(const ll_kv4_cache* cache, int B, int T, int max_count, bool share) {
  if (!kv4_step_ok(cache, B, T, max_count)) return 0;
  return Kv4Lists(B, T, max_count, cache->heads, cache->kv_heads, cache->max_length, share && kv4_shares(cache, B, T, max_count)).ints();
}
size_t ll_kv4_work_ints(const ll_kv4_cache* cache, int B, int T, int max_count) { return work_ints(cache, B, T, max_count, false); }
size_t ll_kv4_shared_work_ints(const ll_kv4_cache* cache, int B, int T, int max_count) { return work_ints(cache, B, T, max_count, true); }

static int make_plan(const ll_kv4_cache* cache, const int32_t* rows, const int32_t* counts, int B, int T, int max_count, int32_t* out, int32_t* work,
                     ll_stream stream, bool share) {
  if (int r = check_cache(cache, "kv4_plan")) return r;
  LL_CHECK_ARG(rows && counts && out && work && ((uintptr_t)work & 15) == 0 && B > 0 && T >= 0 && max_count >= 0 && (long long)T * cache->heads <= INT_MAX,
               "kv4_plan: %d sequences of %d tokens, %d at most", B, T, max_count);
  share = share && kv4_shares(cache, B, T, max_count);
  const Kv4Pool c = pool_of(cache);
  const Kv4Plan p{out, out + B + 1, out + 2 * (size_t)B + 1, out + 3 * (size_t)B + 1, out + 4 * (size_t)B + 1, out + 4 * (size_t)B + 1 + T};
  const Kv4Lists l(B, T, max_count, cache->heads, cache->kv_heads, cache->max_length, share);
  LL_CHECK_ARG(l.few_items * cache->kv_heads <= INT_MAX && l.many_items * cache->kv_heads <= INT_MAX, "kv4_plan: %d sequences of %d tokens, %d heads", B, T, cache->heads);
  const int longest = (cache->max_length + KV4_PAGE - 1) / KV4_PAGE;
  // (pages take a block of the few 0.8 us, of the many 1.4; a part's start and end 2 and 3, parts that are joined 3 and 8 more; a warp alone 3.2 and 2)
  PlanWork few{l.R, share ? INT_MAX : l.few, l.cols, longest, l.few_parts, (int)l.few_items, l.few_joins(), 2.5f, share ? 0.f : 3.5f, l.few_cut, work};
  PlanWork many{l.R, share ? INT_MAX : l.few, KV4_MANY, longest, l.many_parts, (int)l.many_items, l.many_joins(), 2.f, share ? 0.f : 5.5f, true, l.many ? work + l.few_ints() : nullptr};
  // The block itself places the tokens of a step while that takes it a few rounds; more are placed by a grid.
  const int threads = B <= 16 && T <= 2048 ? 256 : B <= 256 && T <= 4096 ? 512 : PLAN_THREADS, here = T <= 8 * threads ? T : 0;
  cudaStream_t st = (cudaStream_t)stream;
  if (share) few.cuts = many.cuts = KV4_SHARE_CUTS, few.fixed = 0.7f;
  PlanWork none = few;
  if (share) none.work = nullptr;
  kv4_plan_kernel<<<1, threads, 0, st>>>(rows, counts, B, T, here, max_count, c, p, none, many);
  LL_LAUNCH_OK("kv4_plan_kernel");
  if (here < T) {
    LL_CUDA(launch(kv4_tokens_kernel, dim3((T - here + 255) / 256), dim3(256), 0, st, true, B, T, here, c, p));
    LL_LAUNCH_OK("kv4_tokens_kernel");
  }
  if (share) {
    LL_CUDA(launch(kv4_share_kernel, dim3(1), dim3(PLAN_THREADS), 0, st, here == T, c, p, B, few, many, work + l.list_ints()));
    LL_LAUNCH_OK("kv4_share_kernel");
  }
  return LL_OK;
}
int ll_kv4_plan(const ll_kv4_cache* cache, const int32_t* rows, const int32_t* counts, int B, int T, int max_count, int32_t* out, int32_t* work,
                ll_stream stream) {
  return make_plan(cache, rows, counts, B, T, max_count, out, work, stream, false);
}
int ll_kv4_shared_plan(const ll_kv4_cache* cache, const int32_t* rows, const int32_t* counts, int B, int T, int max_count, int32_t* out, int32_t* work,
                       ll_stream stream) {
  return make_plan(cache, rows, counts, B, T, max_count, out, work, stream, true);
}

int ll_kv4_truncate(const ll_kv4_cache* cache, const int32_t* rows, const int32_t* keep, int B, ll_stream stream) {
  if (int r = check_cache(cache, "kv4_truncate")) return r;
  LL_CHECK_ARG(rows && keep && B > 0, "kv4_truncate: %d sequences", B);
  kv4_truncate_kernel<<<1, B <= 32 ? 256 : PLAN_THREADS, 0, (cudaStream_t)stream>>>(rows, keep, B, pool_of(cache));
  LL_LAUNCH_OK("kv4_truncate_kernel");
  return LL_OK;
}

int ll_kv4_append(const ll_kv4_cache* cache, void* blocks, const void* q, long long q_row, const void* k, long long k_row, const void* v, long long v_row,
                  const float* rope, const int32_t* positions, const int32_t* slots, void* q_out, int T, ll_stream stream) {
  if (int r = check_cache(cache, "kv4_append")) return r;
  const int H = cache->heads, G = cache->kv_heads;
  LL_CHECK_ARG(k && v && positions && slots && blocks && (!rope || (q && q_out)) && T > 0, "kv4_append: %d tokens of %d heads, %d cached", T, H, G);
  const uintptr_t a = (uintptr_t)(rope ? q : nullptr) | (uintptr_t)k | (uintptr_t)v | (uintptr_t)rope | (uintptr_t)(rope ? q_out : nullptr) | (uintptr_t)blocks;
  LL_CHECK_ARG((a & 15) == 0 && ((rope ? q_row : 0) | k_row | v_row) % 8 == 0, "kv4_append: rows have to start on 16-byte boundaries");
  const Kv4Rows in{q, k, v, q_row, k_row, v_row};
  const int tokens = 256 / cache->head_size, vecs = ((rope ? (H + APPEND_HEADS - 1) / APPEND_HEADS : 0) + 2 * G + 7) / 8;
  LL_CHECK_ARG(vecs <= 65535, "kv4_append: %d heads, %d cached", H, G);
  cudaStream_t st = (cudaStream_t)stream;
  const dim3 grid((T + tokens - 1) / tokens, vecs);
#define APPEND_AS(TT, DD, NG, TURN) kv4_append_kernel<TT, DD, NG, TURN><<<grid, 256, 0, st>>>(in, rope, positions, slots, (TT*)q_out, (uint8_t*)blocks, T, H, G);
#define APPEND(DD, NG)                                                                \
  if (cache->dtype == LL_BF16 && rope) { APPEND_AS(__nv_bfloat16, DD, NG, true) }     \
  else if (cache->dtype == LL_BF16) { APPEND_AS(__nv_bfloat16, DD, NG, false) }       \
  else if (rope) { APPEND_AS(__half, DD, NG, true) }                                  \
  else { APPEND_AS(__half, DD, NG, false) }
  KV4_SHAPES(cache->head_size, cache->group, APPEND)
#undef APPEND
#undef APPEND_AS
  LL_LAUNCH_OK("kv4_append_kernel");
  return LL_OK;
}

int ll_kv4_read(const ll_kv4_cache* cache, const void* blocks, const int32_t* slots, void* k, void* v, int n, ll_stream stream) {
  if (int r = check_cache(cache, "kv4_read")) return r;
  LL_CHECK_ARG(blocks && slots && k && v && n > 0, "kv4_read: %d slots", n);
  const int at_once = read_slots(cache->head_size);
  const long long grid = (((long long)n + at_once - 1) / at_once * cache->kv_heads + 7) / 8;
  LL_CHECK_ARG(grid <= INT_MAX, "kv4_read: %d slots of %d heads", n, cache->kv_heads);
  cudaStream_t st = (cudaStream_t)stream;
#define READ_AS(TT, DD, NG) \
  kv4_read_kernel<TT, DD, NG><<<(unsigned)grid, 256, 0, st>>>((const uint8_t*)blocks, slots, (TT*)k, (TT*)v, n, cache->kv_heads, cache->pages);
#define READ(DD, NG)                                              \
  if (cache->dtype == LL_BF16) { READ_AS(__nv_bfloat16, DD, NG) } \
  else { READ_AS(__half, DD, NG) }
  KV4_SHAPES(cache->head_size, cache->group, READ)
#undef READ
#undef READ_AS
  LL_LAUNCH_OK("kv4_read_kernel");
  return LL_OK;
}

}  // extern "C"
