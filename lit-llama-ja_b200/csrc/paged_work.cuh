// The division of a paged step's attention among blocks: which parts of which walks there are, and where a part's sums go.
#pragma once
#include "kv4.cuh"

namespace llb {

struct Kv4Attn {
  const void* q;
  long long q_row;
  const uint8_t* blocks;
  const int32_t *table, *work;
  void* y;
  float* part;         // [items][G][columns] of D sums, then [items][G][columns] of (reference, sum of weights)
  int H, G, width, pages, max_items;
  float scale;
  int* word;           // wait_word()
};

namespace {

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

constexpr float KV4_NONE = -1e37f;      // the reference of a column that has seen no key

// Sequences that bring up to this many columns a key head go to the kernel of few columns, others to the tcgen05 kernel in tiles of KV4_MANY.
constexpr int KV4_FEW_MOST = 32, KV4_MANY = 256;

inline bool kv4_many(int max_count, int R, int head_size) { return head_size >= 64 && (long long)max_count * R > KV4_FEW_MOST; }
inline int kv4_sms() { return sm_count() > 0 ? sm_count() : 148; }

}  // namespace
int kv4_prompt_launch(const Kv4Attn& a, int dtype, int head_size, int group, cudaStream_t st);      // paged_prompt.cu
}  // namespace llb
