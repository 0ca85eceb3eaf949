// Rotary positions: what the kernels that rotate share.
//
// Pair i of a row at position t is turned by the angle t * f_i. f_i is held as a whole
// number of 2^-64 turns, so that the product modulo one turn is a 64-bit integer multiplication,
// exact at every position; its upper 32 bits, rounded, go to sincospif as a float of half turns
// (at most 2^-33 turns, 7.4e-10 radians, from the rounding, and 2^-24 relative from the float).
#pragma once

#include <stdint.h>

#include "common.cuh"

namespace mlora {

struct RotaryAngles {
  const int64_t* turns;      // [pairs], null: nothing is rotated
  const int32_t* positions;  // [tokens]
  int pairs;                 // half of the dimensions that are rotated
  int interleaved;           // pairs (2i, 2i + 1), or (i, i + pairs)
  float factor;              // of both outputs
};

// {cos, sin} * factor
__device__ __forceinline__ float2 rotary_turn(int64_t turns, int position, float factor) {
  const uint64_t angle = (uint64_t)turns * (uint64_t)(int64_t)position;
  const float half_turns = (float)(int32_t)(uint32_t)((angle + 0x80000000ull) >> 32) * 0x1p-31f;
  float s, c;
  sincospif(half_turns, &s, &c);
  return make_float2(c * factor, s * factor);
}

// V elements of T as they lie in memory.
template <int BYTES>
struct RawBytes;
template <>
struct RawBytes<16> {
  using type = uint4;
};
template <>
struct RawBytes<8> {
  using type = uint2;
};
template <>
struct RawBytes<4> {
  using type = uint32_t;
};
template <>
struct RawBytes<1> {
  using type = unsigned char;
};
template <>
struct RawBytes<2> {
  using type = unsigned short;
};

template <typename T, int V>
struct Vec {
  using Raw = typename RawBytes<V * (int)sizeof(T)>::type;
  union {
    Raw raw;
    T at[V];
  };
  __device__ __forceinline__ Vec() : raw() {}
  __device__ __forceinline__ void load(const T* p) { raw = __ldcg(reinterpret_cast<const Raw*>(p)); }
  __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<Raw*>(p) = raw; }
  __device__ __forceinline__ void to_f(float (&f)[V]) const {
    if constexpr (sizeof(T) == 2 && V > 1) {
      uint32_t w[V / 2];
      memcpy(w, &raw, sizeof(raw));
#pragma unroll
      for (int i = 0; i < V; i += 2) {
        f[i] = Pack2<T>::lo(w[i / 2]);
        f[i + 1] = Pack2<T>::hi(w[i / 2]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) f[i] = Num<T>::to_f(at[i]);
    }
  }
  __device__ __forceinline__ void from_f(const float (&f)[V]) {
    if constexpr (sizeof(T) == 2 && V > 1) {  // two roundings an instruction
      uint32_t w[V / 2];
#pragma unroll
      for (int i = 0; i < V; i += 2) w[i / 2] = pack_round2<T>(f[i], f[i + 1]);
      memcpy(&raw, w, sizeof(raw));
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) at[i] = Num<T>::from_f(f[i]);
    }
  }
};

// A row of `dim` elements is worked on in units of two vectors of V: those of V pairs (V divides
// their number), or 2 V elements that are not rotated. Where unit u lies: its vectors' first elements
// (the second one may lie past the row: dim behind the pairs is a multiple of V only), the first pair.
struct RotaryUnit {
  int e0, e1, pair;
  bool turned, both;
};
__device__ __forceinline__ RotaryUnit rotary_unit(const RotaryAngles& a, bool rotated, int dim, int V, int u) {
  RotaryUnit r;
  r.pair = u * V;
  r.turned = rotated && r.pair < a.pairs;
  if (r.turned && !a.interleaved) {
    r.e0 = r.pair;
    r.e1 = r.pair + a.pairs;
  } else {
    r.e0 = 2 * r.pair;
    r.e1 = r.e0 + V;
  }
  r.both = r.e1 < dim;
  return r;
}

// A unit's two vectors where they lie side by side and 32 bytes allow it: whole sectors at once.
template <typename T, int V>
__device__ __forceinline__ void load_both(Vec<T, V> (&x)[2], const T* p) {
  static_assert(V * sizeof(T) == 16, "32 bytes");
  uint4 a, b;
  asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(a.x), "=r"(a.y), "=r"(a.z), "=r"(a.w), "=r"(b.x), "=r"(b.y), "=r"(b.z), "=r"(b.w)
               : "l"(p)
               : "memory");
  x[0].raw = a;
  x[1].raw = b;
}
template <typename T, int V>
__device__ __forceinline__ void store_both(T* p, const Vec<T, V> (&x)[2]) {
  static_assert(V * sizeof(T) == 16, "32 bytes");
  const uint4 a = x[0].raw, b = x[1].raw;
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w),
               "r"(b.x), "r"(b.y), "r"(b.z), "r"(b.w)
               : "memory");
}

// One pair; the same roundings in every kernel and width.
__device__ __forceinline__ void rotary_pair(float2 t, float& a, float& b) {
  const float x = __fmaf_rn(a, t.x, -__fmul_rn(b, t.y));
  b = __fmaf_rn(b, t.x, __fmul_rn(a, t.y));
  a = x;
}

// The two vectors of a rotated unit, `t` the {cos, sin} of its pairs.
template <int V>
__device__ __forceinline__ void rotary_apply(bool interleaved, const float2 (&t)[V], float (&a)[V], float (&b)[V]) {
  if constexpr (V > 1) {
    if (interleaved) {
#pragma unroll
      for (int i = 0; i < V; i += 2) {
        rotary_pair(t[i / 2], a[i], a[i + 1]);
        rotary_pair(t[V / 2 + i / 2], b[i], b[i + 1]);
      }
      return;
    }
  }
#pragma unroll
  for (int i = 0; i < V; ++i) rotary_pair(t[i], a[i], b[i]);
}

}  // namespace mlora
