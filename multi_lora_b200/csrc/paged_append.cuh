// Rows that are rotated on the way from the projections to `out` and into a cache of their own type: what
// csrc/paged_append.cu launches, and csrc/paged_append_codes.cu beside its own work.
#pragma once

#include "common.cuh"
#include "device.h"
#include "paged.h"

namespace mlora {

constexpr int kRotNT = 256;

// {cos, sin} of `rows` tokens from t0 on, [rows][pairs], a row as [V / 2][unit][2]: what threads with neighbouring
// units read at once, 16 bytes each, lies side by side in the banks.
template <int V>
__device__ __forceinline__ void rotary_table(const RotaryAngles& a, int t0, int rows, float2* table) {
  const int units = a.pairs / V;
  for (int e = threadIdx.x; e < rows * a.pairs; e += kRotNT) {
    const int t = e / a.pairs, pair = e - t * a.pairs, u = pair / V, i = pair % V;
    table[t * a.pairs + (V == 1 ? u : ((i >> 1) * units + u) * 2 + (i & 1))] =
        rotary_turn(__ldg(a.turns + pair), __ldcg(a.positions + t0 + t), a.factor);
  }
}
// Those of the unit that begins with `pair`; `row`: the token's.
template <int V>
__device__ __forceinline__ void rotary_row(const RotaryAngles& a, const float2* row, int pair, float2 (&turn)[V]) {
  if constexpr (V == 1) {
    turn[0] = row[pair];
  } else {
#pragma unroll
    for (int j = 0; j < V / 2; ++j) {
      const float4 q = reinterpret_cast<const float4*>(row)[j * (a.pairs / V) + pair / V];
      turn[2 * j] = make_float2(q.x, q.y);
      turn[2 * j + 1] = make_float2(q.z, q.w);
    }
  }
}

// What CTA `cta` of those that rotate does: `per_cta` tokens, their q_heads query heads and, where `kv_heads` is not 0,
// their rows of K and V. A thread has one token and one unit of its rows, whose {cos, sin} it keeps, and goes through
// every so many heads: a unit then costs little besides its loads, its arithmetic and its stores (with a token, head
// and unit of its own at every turn it took 300 instructions, and 4340 tokens of 32 heads 17.5 us where they take 15.3).
template <typename T, int V>
__device__ __forceinline__ void append_rows(const PagedAppendArgs& p, int kv_heads, int cta, int per_cta, int units, float2* s_turn) {
  const int t0 = cta * per_cta, tokens = min(per_cta, p.tokens - t0);
  const int heads = p.q_heads + 2 * kv_heads, step = kRotNT / units / per_cta;  // heads of a token at once
  const int row = threadIdx.x / units, u = threadIdx.x - row * units, t = row / step;
  const bool rotates = p.angles.turns != nullptr;
  int h = t < tokens ? row - t * step : heads;
  const int64_t token = t0 + min(t, tokens - 1);
  const RotaryUnit un = rotary_unit(p.angles, rotates, p.dim, V, u);
  const T *from_q = nullptr, *from_k = nullptr, *from_v = nullptr;
  T *to_q = nullptr, *to_k = nullptr, *to_v = nullptr;
  if (p.q_heads > 0) {
    from_q = static_cast<const T*>(p.q) + token * p.q_token;
    to_q = static_cast<T*>(p.out) + token * p.out_token;
  }
  if (kv_heads > 0) {
    from_k = static_cast<const T*>(p.side[0].src) + token * p.side[0].src_token;
    from_v = static_cast<const T*>(p.side[1].src) + token * p.side[1].src_token;
    const int slot = __ldcg(p.slot_map + token);
    if (slot >= 0) {
      const int block = slot / p.block_size, off = slot - block * p.block_size;
      if (block < p.num_blocks) {
        to_k = static_cast<T*>(p.side[0].dst) + block * p.side[0].block + off * p.side[0].slot;
        to_v = static_cast<T*>(p.side[1].dst) + block * p.side[1].block + off * p.side[1].slot;
      } else if (u == 0 && h == 0) {
        flag_error(p.status, kErrKvRange);
      }
    }
  }
  // a row's two pieces: those of the unit's pairs, or side by side where it is not rotated
  auto load = [&](int h, Vec<T, V> (&x)[2], T*& dst, bool& turned) {
    const int side = h - p.q_heads >= kv_heads, hk = h - p.q_heads - side * kv_heads;
    const T* src;
    if (h < p.q_heads) {
      src = from_q + h * p.q_head;
      dst = to_q + h * p.out_head;
    } else if (side == 0) {
      src = from_k + hk * p.side[0].src_head;
      dst = to_k == nullptr ? nullptr : to_k + hk * p.side[0].head;
    } else {
      src = from_v + hk * p.side[1].src_head;
      dst = to_v == nullptr ? nullptr : to_v + hk * p.side[1].head;
    }
    turned = un.turned && (h < p.q_heads || side == 0);
    const int e0 = turned ? un.e0 : 2 * V * u, e1 = turned ? un.e1 : e0 + V;
    if constexpr (V * sizeof(T) == 16) {
      if (p.wide && e1 == e0 + V && e1 < p.dim) {
        load_both<T, V>(x, src + e0);
        return;
      }
    }
    x[0].load(src + e0);
    if (e1 < p.dim) x[1].load(src + e1);
  };
  Vec<T, V> x[2];
  T* dst = nullptr;
  bool turned = false;
  if (h < heads) load(h, x, dst, turned);
  float2 turn[V];
  if (rotates) {  // while the first rows are on their way
    rotary_table<V>(p.angles, t0, tokens, s_turn);
    __syncthreads();
    if (un.turned) rotary_row<V>(p.angles, s_turn + (token - t0) * p.angles.pairs, un.pair, turn);
  }
  while (h < heads) {
    if (dst != nullptr) {
      if (turned) {
        float a[V], b[V];
        x[0].to_f(a);
        x[1].to_f(b);
        rotary_apply<V>(p.angles.interleaved != 0, turn, a, b);
        x[0].from_f(a);
        x[1].from_f(b);
      }
      const int e0 = turned ? un.e0 : 2 * V * u, e1 = turned ? un.e1 : e0 + V;
      bool wide = false;
      if constexpr (V * sizeof(T) == 16) {
        wide = p.wide && e1 == e0 + V && e1 < p.dim;
        if (wide) store_both<T, V>(dst + e0, x);
      }
      if (!wide) {
        x[0].store(dst + e0);
        if (e1 < p.dim) x[1].store(dst + e1);
      }
    }
    h += step;
    if (h < heads) load(h, x, dst, turned);
  }
}

// Tokens a CTA that rotates takes: as many as leave every SM three CTAs, and its threads a row of every token, at most
// eight (prompts of 4340 tokens, 32 and 48 heads of 128: 15.3 and 22.4 us; five tokens 17.0 and 24.5, two 18.3 and 25.6).
inline int tokens_per_cta(const PagedAppendArgs& a, int units) {
  const int room = kRotNT / units, even = a.tokens / (3 * device_sm_count()) + 1;
  const int n = even < room ? even : room;
  return n > 8 ? 8 : n;
}

}  // namespace mlora
