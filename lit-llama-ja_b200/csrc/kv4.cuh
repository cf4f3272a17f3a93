// Layout of the paged key/value cache in 4 bits (paged_kv4.cu writes it, paged_attn.cu reads it).
//
// A page holds 64 slots.  Of every page each key/value head has one run of bytes: four slices of 16 slots, so that a warp that walks a head's keys
// copies its slice of a page at once.  A slice:
//   key codes    [16 slots][D / 2 bytes]      4 chunks (t) of W = D / 32 words a slot
//   value codes  [8 pairs of slots][D bytes]  8 chunks (g) of W words a pair
//   key parameters, then value parameters: [16 slots][D / group][scale, lowest value], in the cache's type
// The codes lie as the operands of a 16 x 16 product want them (mma.sync m16n8k16, A by rows): one load gives a lane the words of all its tiles, and a
// word's codes become pairs of numbers by masks alone:
//   keys:   rows are slots.  Word i of chunk t holds the dimensions 32 i + 16 (n >> 1) + 4 t + 2 (n & 1) + e, the code of nibble n, half e at bit 16 e + 4 n
//   values: rows are dimensions, pairs run along the slots.  Word i of chunk g holds the dimensions 32 i + 8 n + g of slot 2 pair + e at bit 16 e + 4 n
// A word belongs to one group of 32 dimensions.  A nibble under a mask is a subnormal number of fp16: nibble 0 is its code times 2^-24, nibble 1 its
// code times 2^-20, exactly; nibbles 2 and 3 are so after one shift by eight.
#pragma once
#include "common.cuh"

namespace llb {
namespace {

constexpr int KV4_PAGE = 64, KV4_SLICE = 16;

__host__ __device__ constexpr int kv4_v_codes(int D) { return KV4_SLICE * D / 2; }
__host__ __device__ constexpr int kv4_k_params(int D) { return KV4_SLICE * D; }
__host__ __device__ constexpr int kv4_v_params(int D, int groups) { return KV4_SLICE * (D + 4 * groups); }
__host__ __device__ constexpr int kv4_slice_bytes(int D, int groups) { return KV4_SLICE * (D + 8 * groups); }
__host__ __device__ constexpr int kv4_bytes(int D, int groups) { return KV4_PAGE / KV4_SLICE * kv4_slice_bytes(D, groups); }

template <typename T> struct pair_of;
template <> struct pair_of<__nv_bfloat16> { typedef __nv_bfloat162 type; };
template <> struct pair_of<__half> { typedef __half2 type; };
__device__ __forceinline__ float2 to_float2(__nv_bfloat162 v) { return __bfloat1622float2(v); }
__device__ __forceinline__ float2 to_float2(__half2 v) { return __half22float2(v); }
template <typename T> __device__ __forceinline__ typename pair_of<T>::type to_pair(float a, float b);
template <> __device__ __forceinline__ __nv_bfloat162 to_pair<__nv_bfloat16>(float a, float b) { return __floats2bfloat162_rn(a, b); }
template <> __device__ __forceinline__ __half2 to_pair<__half>(float a, float b) { return __floats2half2_rn(a, b); }
template <typename T> __device__ __forceinline__ uint32_t pair_bits(float a, float b) {
  const typename pair_of<T>::type v = to_pair<T>(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <typename T> __device__ __forceinline__ float2 bits_pair(uint32_t u) { return to_float2(*reinterpret_cast<const typename pair_of<T>::type*>(&u)); }

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

// head sizes and groups that there are kernels for
inline bool kv4_shape_ok(int D, int group) { return (D == 32 || D == 64 || D == 128) && (group == 32 || group == 64 || group == 128) && group <= D; }

}  // namespace
}  // namespace llb

// CALL(D, groups) for the head size and group at hand
#define KV4_SHAPES(head_size, group, CALL)                                 \
  if (head_size == 32) { CALL(32, 1) }                                     \
  else if (head_size == 64 && group == 64) { CALL(64, 1) }                 \
  else if (head_size == 64) { CALL(64, 2) }                                \
  else if (group == 128) { CALL(128, 1) }                                  \
  else if (group == 64) { CALL(128, 2) }                                   \
  else { CALL(128, 4) }
