// Vector loads and stores that convert between a stored type (fp32, bf16, fp16) and fp32 registers.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace grace {

using bf16_t = __bf16;    // gfx950 converts with v_cvt_pk_bf16_f32 (round to nearest even, NaN kept)
using half_t = _Float16;

// element types as the host passes them to a launcher
enum class ElType : int { kF32 = 0, kBF16 = 1, kF16 = 2 };

inline int el_bytes(ElType t) { return t == ElType::kF32 ? 4 : 2; }

// V consecutive elements, aligned as one element only: gfx950 takes wide global accesses at any
// element's address, so rows of odd width and odd views need no narrower kernels.
template <typename T, int V>
struct __attribute__((packed, aligned(sizeof(T)))) Pack {
  T v[V];
};

// the first n of V elements at p, widened to fp32; the others are zero
template <int V, typename T>
__device__ __forceinline__ void load_vec(const T* __restrict__ p, float (&o)[V], int n = V) {
  if (n >= V) {
    const Pack<T, V> r = *reinterpret_cast<const Pack<T, V>*>(p);
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] = (float)r.v[i];
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] = i < n ? (float)p[i] : 0.f;
  }
}

// one rounding to nearest even (none for fp32) of the first n of V elements
template <int V, typename T>
__device__ __forceinline__ void store_vec(T* __restrict__ p, const float (&x)[V], int n = V) {
  if (n >= V) {
    Pack<T, V> r;
#pragma unroll
    for (int i = 0; i < V; ++i) r.v[i] = (T)x[i];
    *reinterpret_cast<Pack<T, V>*>(p) = r;
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (i < n) p[i] = (T)x[i];
  }
}

}  // namespace grace
