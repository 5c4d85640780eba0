// na_chunk.h — 16-byte chunks of a row at any alignment of its elements, with a
// bounded last chunk, and sums over a group of lanes: the kernels that stream rows of
// any width (na_norm.hip, na_rotary.hip, na_norm_rotary.hip).
#pragma once

#include "na_common.h"

namespace na {
namespace {

// Rows and channels have any alignment of their type: the hardware takes
// 16-byte accesses at element alignment.
template <int A>
struct Mem16;
template <>
struct Mem16<2> {
  typedef uint32_t t __attribute__((ext_vector_type(4), aligned(2)));
};
template <>
struct Mem16<4> {
  typedef uint32_t t __attribute__((ext_vector_type(4), aligned(4)));
};

template <typename T>
struct Chunk {
  static constexpr int N = 16 / (int)sizeof(T);
  typedef uint32_t raw __attribute__((ext_vector_type(4)));
  typedef typename Mem16<sizeof(T)>::t mem;
  static __device__ __forceinline__ raw load(const T *p, int n) {  // n: elements of the row left
    if (n >= N) return *reinterpret_cast<const mem *>(p);
    raw r = {0, 0, 0, 0};
    if (sizeof(T) == 4) {
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (e < n) r[e % 4] = reinterpret_cast<const uint32_t *>(p)[e];
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (e < n) r[e / 2 % 4] |= (uint32_t)reinterpret_cast<const uint16_t *>(p)[e] << (16 * (e & 1));
    }
    return r;
  }
  static __device__ __forceinline__ float get(const raw &r, int e);
  static __device__ __forceinline__ void store(T *p, const float *x, int n);
};
template <>
__device__ __forceinline__ float Chunk<float>::get(const raw &r, int e) {
  return __uint_as_float(r[e]);
}
template <>
__device__ __forceinline__ float Chunk<bf16_t>::get(const raw &r, int e) {
  return __uint_as_float(e & 1 ? r[e / 2] & 0xffff0000u : r[e / 2] << 16);
}
template <>
__device__ __forceinline__ float Chunk<f16_t>::get(const raw &r, int e) {
  return (float)__builtin_bit_cast(f16_t, (uint16_t)(r[e / 2] >> (16 * (e & 1))));
}

template <typename T>
struct Hw {  // the type the compiler converts floats to
  typedef T t;
};
template <>
struct Hw<bf16_t> {
  typedef __bf16 t;
};

template <typename T>
__device__ __forceinline__ void Chunk<T>::store(T *p, const float *x, int n) {
  typedef typename Hw<T>::t H;
  if (n >= N) {
    H h[N];
#pragma unroll
    for (int e = 0; e < N; ++e) h[e] = (H)x[e];
    raw r;
    __builtin_memcpy(&r, h, 16);
    *reinterpret_cast<mem *>(p) = r;
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (e < n) reinterpret_cast<H *>(p)[e] = (H)x[e];
  }
}

template <int CTRL>
__device__ __forceinline__ float dpp_add(float x) {
  return x + __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), CTRL, 0xf, 0xf, true));
}

// Sum over an aligned group of 2^lg lanes (wave-uniform lg), in every lane.
__device__ __forceinline__ float lanes_sum(float x, int lg) {
  if (lg > 0) x = dpp_add<0xB1>(x);   // lane ^ 1
  if (lg > 1) x = dpp_add<0x4E>(x);   // lane ^ 2
  if (lg > 2) x = dpp_add<0x141>(x);  // mirror within 8 lanes
  if (lg > 3) x = dpp_add<0x140>(x);  // mirror within 16 lanes
  if (lg > 4) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  }
  if (lg > 5) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  }
  return x;
}

}  // namespace
}  // namespace na
