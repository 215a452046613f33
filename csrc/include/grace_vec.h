// Vector loads and stores that convert between a stored type (fp32, bf16, fp16) and fp32 registers.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

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

// The same address, as a value of its own.  The element-wise branch of a partial vector works on it: seeing
// one address in both branches, the compiler takes the elements they share out of the wide access, which then
// falls apart into a halfword, two dwords and so on.  It names global memory, which the compiler no longer
// sees: a generic access in one branch would make every wait behind it one for all loads.
template <typename T>
using GlobalPtr = __attribute__((address_space(1))) T*;
template <typename T>
__device__ __forceinline__ GlobalPtr<T> apart(T* p) {
  GlobalPtr<T> q = (GlobalPtr<T>)p;
  asm("" : "+v"(q));
  return q;
}

// V elements as stored, in whole registers (two 16-bit values to a register: a struct of elements that
// lives across a loop gets a register for each)
template <typename T, int V>
struct Bits {
  static constexpr int W = (V * (int)sizeof(T) + 3) / 4;
  uint32_t w[W];
};
template <int W, int A>
struct __attribute__((packed, aligned(A))) Words {
  uint32_t w[W];
};

// The first n (1 or more) of V elements at p; the others are zero.  ONCE: data that passes the caches by (nontemporal)
template <bool ONCE = false, typename T, int V>
__device__ __forceinline__ void load_bits(const T* __restrict__ p, Bits<T, V>& o, int n = V) {
  constexpr int W = Bits<T, V>::W;
  if constexpr (V == 1 && sizeof(T) == 2) {
    o.w[0] = *reinterpret_cast<const uint16_t*>(p);
  } else if (n >= V) {
    if constexpr (ONCE) {
      typedef uint32_t word __attribute__((aligned(2)));
#pragma unroll
      for (int i = 0; i < W; ++i) o.w[i] = __builtin_nontemporal_load(reinterpret_cast<const word*>(p) + i);
      return;
    }
    const Words<W, sizeof(T)> r = *reinterpret_cast<const Words<W, sizeof(T)>*>(p);
#pragma unroll
    for (int i = 0; i < W; ++i) o.w[i] = r.w[i];
  } else {
#pragma unroll
    for (int i = 0; i < W; ++i) o.w[i] = 0;
    const GlobalPtr<const T> q = apart(p);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if (i >= n) continue;
      if constexpr (sizeof(T) == 4) o.w[i] = ((GlobalPtr<const uint32_t>)q)[i];
      else o.w[i / 2] |= (uint32_t)((GlobalPtr<const uint16_t>)q)[i] << (16 * (i & 1));
    }
  }
}

template <typename T, int V>
__device__ __forceinline__ float bits_at(const Bits<T, V>& b, int i) {
  if constexpr (sizeof(T) == 4) return __uint_as_float(b.w[i]);
  else if constexpr (std::is_same<T, bf16_t>::value)
    return __uint_as_float(i & 1 ? b.w[i / 2] & 0xffff0000u : b.w[i / 2] << 16);
  else return (float)__builtin_bit_cast(half_t, (uint16_t)(b.w[i / 2] >> (16 * (i & 1))));
}

// the first n of V elements at p, widened to fp32; the others are zero
template <int V, typename T>
__device__ __forceinline__ void load_vec(const T* __restrict__ p, float (&o)[V], int n = V) {
  if (n >= V) {
    const Pack<T, V> r = *reinterpret_cast<const Pack<T, V>*>(p);
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] = (float)r.v[i];
  } else {
    const GlobalPtr<const T> q = apart(p);
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] = i < n ? (float)q[i] : 0.f;
  }
}

// one rounding to nearest even (none for fp32) of the first n of V elements
template <bool ONCE = false, int V, typename T>
__device__ __forceinline__ void store_vec(T* __restrict__ p, const float (&x)[V], int n = V) {
  if (n >= V) {
    Pack<T, V> r;
#pragma unroll
    for (int i = 0; i < V; ++i) r.v[i] = (T)x[i];
    if constexpr (ONCE) {
      typedef uint32_t word __attribute__((aligned(2)));
      const Words<V * sizeof(T) / 4, 4> w = __builtin_bit_cast(Words<V * sizeof(T) / 4, 4>, r);
#pragma unroll
      for (int i = 0; i < V * (int)sizeof(T) / 4; ++i)
        __builtin_nontemporal_store(w.w[i], reinterpret_cast<word*>(p) + i);
      return;
    }
    *reinterpret_cast<Pack<T, V>*>(p) = r;
  } else {
    const GlobalPtr<T> q = apart(p);
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (i < n) q[i] = (T)x[i];
  }
}

}  // namespace grace
