// 16-byte vectors at any element's address, and the last, partial one of a row (gfx950).
#pragma once
#include "common.h"

namespace {

// (global memory takes 16-byte accesses at any address; the type only tells the compiler not to assume more)
typedef u32x4 u32x4_any __attribute__((aligned(2)));

// elements 0...min(n, E) - 1 of a 16-byte vector, zeros behind them.  WHOLE: n is at least E or at most 0.
template <bool WHOLE, typename T> __device__ __forceinline__ Vec16<T> load_part(const T* p, int n) {
  constexpr int E = Vec16<T>::N;
  Vec16<T> v = zero16<T>();
  if (n >= E) {
    v = __builtin_bit_cast(Vec16<T>, (u32x4)*reinterpret_cast<const u32x4_any*>(p));
  } else if (!WHOLE) {
#pragma unroll
    for (int e = 0; e < E - 1; ++e)
      if (e < n) v.v[e] = p[e];
  }
  return v;
}
template <bool WHOLE, typename T> __device__ __forceinline__ void store_part(T* p, const Vec16<T>& v, int n) {
  constexpr int E = Vec16<T>::N;
  if (n >= E) {
    *reinterpret_cast<u32x4_any*>(p) = __builtin_bit_cast(u32x4, v);
  } else if (!WHOLE) {
#pragma unroll
    for (int e = 0; e < E - 1; ++e)
      if (e < n) p[e] = v.v[e];
  }
}

}  // namespace
