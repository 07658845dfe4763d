// Sums and maxima over groups of lanes, and rows of 8 elements, for the kernels
// that keep a head's row in the lanes of one wave.
#pragma once
#include "common.h"

namespace dmad {

// The value of lane l ^ m inside groups that already agree on the lanes below:
// quad permutations for 1 and 2, mirrors of 8 and 16 lanes for 4 and 8.
template <int CTRL>
__device__ __forceinline__ float dpp_move(float x) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xf, 0xf, false));
}

struct LaneAdd {
  __device__ __forceinline__ static float op(float a, float b) { return a + b; }
};
struct LaneMax {
  __device__ __forceinline__ static float op(float a, float b) { return fmaxf(a, b); }
};

// permlane16_swap(x, x) gives every lane the values of both 16-lane rows of its
// pair, permlane32_swap(x, x) those of both halves of the wave.
template <typename OP>
__device__ __forceinline__ float across16(float x) {
  const uint32_t u = __float_as_uint(x);
  const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  return OP::op(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
template <typename OP>
__device__ __forceinline__ float across32(float x) {
  const uint32_t u = __float_as_uint(x);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return OP::op(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// Reduction over aligned groups of W lanes; every lane gets the result.
template <int W, typename OP>
__device__ __forceinline__ float group_reduce(float x) {
  if constexpr (W >= 2) x = OP::op(x, dpp_move<0xB1>(x));    // quad_perm 1,0,3,2
  if constexpr (W >= 4) x = OP::op(x, dpp_move<0x4E>(x));    // quad_perm 2,3,0,1
  if constexpr (W >= 8) x = OP::op(x, dpp_move<0x141>(x));   // mirror of 8 lanes
  if constexpr (W >= 16) x = OP::op(x, dpp_move<0x140>(x));  // mirror of 16 lanes
  if constexpr (W >= 32) x = across16<OP>(x);
  if constexpr (W >= 64) x = across32<OP>(x);
  return x;
}
template <int W>
__device__ __forceinline__ float group_sum(float x) {
  return group_reduce<W, LaneAdd>(x);
}

// A vector load or store; NT: not to be kept in the caches.
template <bool NT, typename V>
__device__ __forceinline__ V load_vec(const void* p) {
  if constexpr (NT) return __builtin_nontemporal_load((const V*)p);
  else return *(const V*)p;
}
template <bool NT, typename V>
__device__ __forceinline__ void store_vec(void* p, V v) {
  if constexpr (NT) __builtin_nontemporal_store(v, (V*)p);
  else *(V*)p = v;
}

// 8 consecutive elements of a row, as loaded (16 bytes, or 32 in fp32).
template <typename T>
struct Row8 {
  i32x4_t v;
  template <bool NT = false>
  __device__ __forceinline__ void load(const T* p) { v = load_vec<NT, i32x4_t>(p); }
  __device__ __forceinline__ void zero() { v = i32x4_t{0, 0, 0, 0}; }
  __device__ __forceinline__ float get(int e) const {
    return Elem<T>::to_f32((uint16_t)(((uint32_t)v[e >> 1] >> ((e & 1) * 16)) & 0xffff));
  }
  template <bool NT = false>
  __device__ __forceinline__ static void store(T* p, const float (&x)[8]) {
    i32x4_t o;
#pragma unroll
    for (int k = 0; k < 4; ++k) o[k] = (int)Elem<T>::pack2(x[2 * k], x[2 * k + 1]);
    store_vec<NT>(p, o);
  }
};
template <>
struct Row8<float> {
  f32x4_t lo, hi;
  template <bool NT = false>
  __device__ __forceinline__ void load(const float* p) {
    lo = load_vec<NT, f32x4_t>(p);
    hi = load_vec<NT, f32x4_t>(p + 4);
  }
  __device__ __forceinline__ void zero() { lo = hi = f32x4_t{0.f, 0.f, 0.f, 0.f}; }
  __device__ __forceinline__ float get(int e) const { return e < 4 ? lo[e & 3] : hi[e & 3]; }
  template <bool NT = false>
  __device__ __forceinline__ static void store(float* p, const float (&x)[8]) {
    store_vec<NT>(p, f32x4_t{x[0], x[1], x[2], x[3]});
    store_vec<NT>(p + 4, f32x4_t{x[4], x[5], x[6], x[7]});
  }
};

}  // namespace dmad
