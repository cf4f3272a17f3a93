// Rows of logits by vectors of 16 bytes on the address's own grid, wherever a row begins; places outside of the row are -inf.
#pragma once
#include <type_traits>

#include "common.cuh"

namespace llb {
namespace {

template <typename T> struct row_vec;      // numbers of a vector
template <> struct row_vec<float> { static constexpr int n = 4; };
template <> struct row_vec<__nv_bfloat16> { static constexpr int n = 8; };
template <> struct row_vec<__half> { static constexpr int n = 8; };

template <typename T>
__device__ __forceinline__ void vec_values(const uint4& r, float (&x)[4]) {
  x[0] = __uint_as_float(r.x), x[1] = __uint_as_float(r.y), x[2] = __uint_as_float(r.z), x[3] = __uint_as_float(r.w);
}
template <typename T>
__device__ __forceinline__ void vec_values(const uint4& r, float (&x)[8]) {
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float2 f;
    if constexpr (std::is_same<T, __half>::value) f = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
    else f = make_float2(__uint_as_float(w[j] << 16), __uint_as_float(w[j] & 0xffff0000u));
    x[2 * j] = f.x, x[2 * j + 1] = f.y;
  }
}
// The largest of a vector, of pairs at once; a number that is none is passed over.
template <typename T>
__device__ __forceinline__ float vec_max(const uint4& r) {
  if constexpr (std::is_same<T, float>::value) {
    return fmaxf(fmaxf(__uint_as_float(r.x), __uint_as_float(r.y)), fmaxf(__uint_as_float(r.z), __uint_as_float(r.w)));
  } else if constexpr (std::is_same<T, __half>::value) {
    auto h = [](const uint32_t& u) { return *reinterpret_cast<const __half2*>(&u); };
    const float2 f = __half22float2(__hmax2(__hmax2(h(r.x), h(r.y)), __hmax2(h(r.z), h(r.w))));
    return fmaxf(f.x, f.y);
  } else {
    auto h = [](const uint32_t& u) { return *reinterpret_cast<const __nv_bfloat162*>(&u); };
    const float2 f = __bfloat1622float2(__hmax2(__hmax2(h(r.x), h(r.y)), __hmax2(h(r.z), h(r.w))));
    return fmaxf(f.x, f.y);
  }
}
// A vector of -inf.
template <typename T>
__device__ __forceinline__ uint4 none_vector() {
  constexpr uint32_t NONE = std::is_same<T, float>::value ? 0xff800000u : std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;
  return make_uint4(NONE, NONE, NONE, NONE);
}
// How many numbers the row begins behind a 16-byte boundary.
template <typename T>
__device__ __forceinline__ int row_offset(const T* row) { return (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T)); }
// The vector that begins with number i of the row (a boundary of the address; i may be negative), as it is in memory.
template <typename T>
__device__ __forceinline__ uint4 load_vector(const T* row, int i, int V) {
  constexpr int N = row_vec<T>::n;
  if (i >= 0 && i + N <= V) return __ldg(reinterpret_cast<const uint4*>(row + i));
  constexpr uint32_t NONE = std::is_same<T, float>::value ? 0xff800000u : std::is_same<T, __half>::value ? 0xfc00u : 0xff80u;      // -inf
  uint32_t w[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if constexpr (N == 4) {
      w[j] = i + j >= 0 && i + j < V ? __float_as_uint(row[i + j]) : NONE;
    } else {
      const uint16_t* h = reinterpret_cast<const uint16_t*>(row);
      const int k = i + 2 * j;
      w[j] = (k >= 0 && k < V ? (uint32_t)h[k] : NONE) | (k + 1 >= 0 && k + 1 < V ? (uint32_t)h[k + 1] : NONE) << 16;
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
template <typename T>
__device__ __forceinline__ void load_values(const T* row, int i, int V, float (&x)[row_vec<T>::n]) {
  vec_values<T>(load_vector(row, i, V), x);
}

}  // namespace
}  // namespace llb
