// Rows that are rotated on the way from the projections to `out` and into a cache of their own type: what
// csrc/paged_append.cu launches, and csrc/paged_append_codes.cu beside its own work.
#pragma once

#include "common.cuh"
#include "device.h"
#include "paged.h"

namespace mlora {

constexpr int kRotNT = 256, kRotUnits = 4;

// {cos, sin} of `rows` tokens from t0 on, [rows][pairs].
__device__ __forceinline__ void rotary_table(const RotaryAngles& a, int t0, int rows, float2* table) {
  for (int e = threadIdx.x; e < rows * a.pairs; e += kRotNT) {
    const int t = e / a.pairs;
    table[e] = rotary_turn(__ldg(a.turns + (e - t * a.pairs)), __ldcg(a.positions + t0 + t), a.factor);
  }
}

// What CTA `cta` of those that rotate does: `per_cta` tokens, their q_heads query heads and, where `kv_heads` is not 0,
// their rows of K and V.
template <typename T, int V>
__device__ __forceinline__ void append_rows(const PagedAppendArgs& p, int kv_heads, int cta, int per_cta, int units, float2* s_turn) {
  const int tid = threadIdx.x;
  const int t0 = cta * per_cta, tokens = min(per_cta, p.tokens - t0);
  const int heads = p.q_heads + 2 * kv_heads;
  const int all = tokens * heads * units;  // below 2^31: checked on the host
  bool made = p.angles.turns == nullptr;
  for (int first = 0; first < all; first += kRotNT * kRotUnits) {
    Vec<T, V> x[kRotUnits][2];
    RotaryUnit un[kRotUnits];
    T* dst[kRotUnits];
    int turn_at[kRotUnits];
#pragma unroll
    for (int k = 0; k < kRotUnits; ++k) {
      const int at = first + k * kRotNT + tid;
      dst[k] = nullptr;
      if (at >= all) continue;
      const int row = at / units, u = at - row * units, t = row / heads, h = row - t * heads;
      const int64_t token = t0 + t;
      const bool query = h < p.q_heads;
      const int side = !query && h >= p.q_heads + kv_heads, hk = h - p.q_heads - side * kv_heads;
      un[k] = rotary_unit(p.angles, side == 0 && p.angles.turns != nullptr, p.dim, V, u);
      turn_at[k] = t * p.angles.pairs + un[k].pair;
      const T* src;
      if (query) {
        src = static_cast<const T*>(p.q) + token * p.q_token + h * p.q_head;
        dst[k] = static_cast<T*>(p.out) + token * p.out_token + h * p.out_head;
      } else {
        const PagedSide& s = p.side[side];
        src = static_cast<const T*>(s.src) + token * s.src_token + hk * s.src_head;
        const int slot = __ldcg(p.slot_map + token);
        if (slot >= 0) {
          const int block = slot / p.block_size, off = slot - block * p.block_size;
          if (block < p.num_blocks) dst[k] = static_cast<T*>(s.dst) + block * s.block + off * s.slot + hk * s.head;
          else if (u == 0 && hk == 0) flag_error(p.status, kErrKvRange);
        }
      }
      x[k][0].load(src + un[k].e0);
      if (un[k].both) x[k][1].load(src + un[k].e1);
    }
    if (!made) {
      rotary_table(p.angles, t0, tokens, s_turn);
      __syncthreads();
      made = true;
    }
#pragma unroll
    for (int k = 0; k < kRotUnits; ++k) {
      if (dst[k] == nullptr) continue;
      if (un[k].turned) {
        float a[V], b[V];
        x[k][0].to_f(a);
        x[k][1].to_f(b);
        rotary_apply<V>(p.angles.interleaved != 0, s_turn + turn_at[k], a, b);
        x[k][0].from_f(a);
        x[k][1].from_f(b);
      }
      x[k][0].store(dst[k] + un[k].e0);
      if (un[k].both) x[k][1].store(dst[k] + un[k].e1);
    }
  }
}

// Tokens a CTA that rotates takes: as many as fill its threads once, and no more than leave every SM two CTAs.
inline int tokens_per_cta(const PagedAppendArgs& a, int heads, int units) {
  const int64_t fill = kRotNT * kRotUnits / ((int64_t)heads * units), even = a.tokens / (2 * device_sm_count()) + 1;
  const int64_t n = fill < even ? fill : even;
  return n < 1 ? 1 : n > 16 ? 16 : (int)n;
}

}  // namespace mlora
