// The division of a paged step's attention among blocks: which parts of which walks there are, and where a part's sums go.
#pragma once
#include <algorithm>
#include <climits>

#include "kv4.cuh"

namespace llb {

struct Kv4Attn {
  const void* q;
  long long q_row;
  const uint8_t* blocks;
  const int32_t *table, *work;
  void* y;
  float* part;         // [kept][G][columns] of D sums, then [kept][G][columns] of (reference, sum of weights)
  int H, G, width, pages;
  int items, kept, cols;      // items there is room for, parts whose sums there is room for, columns of a tile that may be in use
  float scale;
  int* word;           // wait_word()
  int* odd;            // [items][G] of the tcgen05 kernel: bit 0, 1: its tile 0, 1 is left to the kernel of few columns
};

namespace {

// A list of parts of walks: four numbers (parts, walks that are in more than one part), the parts, then those walks.
// One part of a walk: a range of one request's pages for one tile of columns (a column: one query of one of the heads that share a key head, the
// heads of a token next to one another).  The largest parts come first.
struct __align__(16) Kv4Item {
  int row, first, count, pos0;         // request (-1: its tokens are refused), first row and number of its tokens, position of the first one
  int tile, page0, page1;              // tile of columns; pages of the part
  int parts;                           // parts of the walk
  int part, base;                      // which of them this is; index of the walk's first part among all parts
  int pad[2];
};
static_assert(sizeof(Kv4Item) == 48, "three loads of 16 bytes");
__device__ __forceinline__ Kv4Item load_item(const int32_t* work, int i) {
  Kv4Item it;
  const int4* p = reinterpret_cast<const int4*>(work) + 1 + 3 * (size_t)i;
  const int4 a = p[0], b = p[1], c = p[2];
  it.row = a.x, it.first = a.y, it.count = a.z, it.pos0 = a.w, it.tile = b.x, it.page0 = b.y, it.page1 = b.z, it.parts = b.w, it.part = c.x, it.base = c.y;
  return it;
}
// A walk whose parts have to be joined.
struct __align__(16) Kv4Join {
  int first, count, tile, parts;       // first row and number of the request's tokens, tile of columns, parts
  int base, pad[3];                    // index of the first part
};
__host__ __device__ __forceinline__ const int4* joins_of(const int32_t* work, int max_items) { return reinterpret_cast<const int4*>(work) + 1 + 3 * (size_t)max_items; }

// For a role that gives up: copies and products that it has issued end (a millisecond and more) before the block lets go of its memory.
__device__ __forceinline__ void kv4_let_end() {
  for (const long long from = clock64(); clock64() - from < 2000000;) __nanosleep(512);
}

// column -> token and head: a shift where the heads of a key head are 1, 2, 4 .., else a division
__device__ __forceinline__ int column_token(int c, int R) { return (R & (R - 1)) == 0 ? c >> (31 - __clz(R)) : c / R; }
__device__ __forceinline__ int column_head(int c, int R) { return (R & (R - 1)) == 0 ? c & (R - 1) : c % R; }

constexpr float KV4_NONE = -1e37f;      // the reference of a column that has seen no key

// Sequences that bring up to KV4_FEW_MOST columns a key head go to the kernel of few columns (in tiles of KV4_FEW_BESIDE beside the others), others to the
// tcgen05 kernel in tiles of KV4_MANY.
// us, few / tcgen05, heads of 128, 2000 keys: 32 heads over 32, one request of 16, 32, 48 tokens 16.1 / 21.9, 19.9 / 22.3, 23.5 / 22.7, eight requests 43 / 77,
// 57 / 77, 118 / 78; 32 heads over 8, one of 8, 16 tokens 15.8 / 22.3, 16.0 / 22.9, eight 28 / 31, 42 / 32.
// Where no request of the cache has more than KV4_WHOLE pages, walks are not cut, and the launch that joins parts falls away (30 to 500 keys of 32 heads, whole /
// cut: one request 3.7 - 6.1 / 4.7 - 6.3, 64 requests 13.8 - 34.8 / 14.8 - 36.1).
constexpr int KV4_FEW_MOST = 32, KV4_FEW_BESIDE = 8, KV4_MANY = 256, KV4_WHOLE = 8;
// Walks for KV4_ROUNDS rounds of blocks stay whole; fewer are cut into at most KV4_CUTS rounds more of parts.
constexpr int KV4_ROUNDS = 3, KV4_CUTS = 2;

inline bool kv4_many(int max_count, int R) { return (long long)max_count * R > KV4_FEW_MOST; }
inline int kv4_sms() { return sm_count() > 0 ? sm_count() : 148; }

// whether a step's lists have a size
inline bool kv4_step_ok(const ll_kv4_cache* c, int B, int T, int max_count) {
  return c != nullptr && c->kv_heads > 0 && c->heads > 0 && c->heads % c->kv_heads == 0 && c->max_length > 0 && B > 0 && T >= 0 && max_count >= 0 &&
         (long long)T * c->heads <= INT_MAX;
}

// A step's two lists: sequences of few columns and, where one may bring more, of many.  Sizes as the host knows them.
struct Kv4Lists {
  int R, cols, few, few_parts, many_parts;
  long long few_items, many_items;      // at most
  bool many, few_cut;
  Kv4Lists(int B, int T, int max_count, int H, int G, int max_length) {
    R = H / G;
    many = kv4_many(max_count, R);
    const long long c = (long long)max_count * R;
    cols = many ? KV4_FEW_BESIDE : c <= 4 ? 4 : c <= 8 ? 8 : 16;
    few = many ? KV4_FEW_MOST : INT_MAX;
    few_parts = std::max(1, 4 * kv4_sms() / G);
    many_parts = std::max(1, kv4_sms() / G);
    // Where no request has more than KV4_WHOLE pages, walks are not cut, and there is nothing to join.
    few_cut = max_length > KV4_WHOLE * KV4_PAGE;
    // tiles: of n columns n / cols, and one more a sequence that is not a whole number of them; sequences of the few have KV4_FEW_MOST columns at most
    // where the others go to the many (and refused ones, whose tokens count here too, may have any)
    const long long seqs = std::min(B, std::max(T, 1)), tiles = (long long)T * R / cols + seqs;
    few_items = (many ? std::min(tiles, seqs * ((KV4_FEW_MOST + cols - 1) / cols)) : tiles) + KV4_CUTS * few_parts;
    many_items = many ? (long long)T * R / KV4_MANY + std::min(seqs, (long long)T * R / KV4_FEW_MOST) + KV4_CUTS * many_parts : 0;
  }
  // walks in more than one part: every one has a part more than it would have whole
  int few_joins() const { return KV4_CUTS * few_parts; }
  int many_joins() const { return KV4_CUTS * many_parts; }
  size_t few_ints() const { return 4 + sizeof(Kv4Item) / 4 * (size_t)few_items + sizeof(Kv4Join) / 4 * (size_t)few_joins(); }
  size_t ints() const { return few_ints() + (many ? 4 + sizeof(Kv4Item) / 4 * (size_t)many_items + sizeof(Kv4Join) / 4 * (size_t)many_joins() : 0); }
  // sums are kept of parts that have to be joined, and none are where there are walks for KV4_ROUNDS rounds
  int few_kept() const { return (int)std::min(few_items, (long long)(KV4_ROUNDS + KV4_CUTS) * few_parts); }
  int many_kept() const { return (int)std::min(many_items, (long long)(KV4_ROUNDS + KV4_CUTS) * many_parts); }
  size_t few_floats(int G, int D) const { return ((size_t)few_kept() * G * cols * (D + 2) + 3) / 4 * 4; }
  size_t many_floats(int G, int D) const { return (size_t)many_kept() * G * KV4_MANY * (D + 2); }
  // sums of both lists, and a word for every block of the many
  size_t bytes(int G, int D) const { return sizeof(float) * (few_floats(G, D) + many_floats(G, D)) + sizeof(int) * (size_t)many_items * G; }
};

}  // namespace
int kv4_prompt_launch(const Kv4Attn& a, int dtype, int head_size, int group, cudaStream_t st);      // paged_prompt.cu
}  // namespace llb
