// Tiles of e4m3 codes under the warp-level tensor cores.
//
// A code is exact in f16, so codes enter the products as they are and their scales stay outside, in
// fp32: a key's multiplies its score, a value's the probability that goes to the second product.
//   * Q is taken in f16. f16 queries are; a bf16 row is multiplied by the power of two that brings its largest
//     element to 2^14 .. 2^15 (undone on the score), which keeps its 8 bits down to 2^-29 of that
//     element and anything below to 2^-40 of it.
//   * P times the value's scale is taken in f16 relative to the largest scale so far (per warp) and times 2^15:
//     11 bits of it (of f16 queries, whose result has as many, two terms: 21 bits), and
//     nothing coarser than 2^-40 of the largest scale.
// Four codes of a register are two operands of the product as they lie: of a row of K the dimension may be taken in any order
// (Q in the same), and of V, transposed in pairs of columns, the even columns make one tile of eight and
// the odd ones another, so that a thread ends up with four columns side by side.
#pragma once

#include "mma.cuh"
#include "paged_sched.cuh"

namespace mlora {

constexpr int kCodeTile = 128;  // keys a stage: 32 of them a warp
constexpr float kCodeUp = 15.f; // P is taken times 2^15
constexpr float kCodeLeast = 0x1p-126f;  // what scales of V are taken relative to is no less: its reciprocal is finite

// Codes 0 and 1 (2 and 3) of a word as a pair of f16.
__device__ __forceinline__ uint32_t codes_lo(uint32_t x) {
  uint32_t y;
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\t}" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ uint32_t codes_hi(uint32_t x) {
  uint32_t y;
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, h;\n\t}" : "=r"(y) : "r"(x));
  return y;
}
// 0x80 in every byte that is a NaN.
__device__ __forceinline__ uint32_t codes_nan(uint32_t x) { return ((x & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }

// Byte offset of 16 codes of a key in a tile of rows of D bytes, swizzled by D bytes as TMA writes them.
template <int D>
__device__ __forceinline__ uint32_t code_at(int key, int chunk) {
  return (uint32_t)(key * D + ((chunk ^ (D == 128 ? key & 7 : (key >> 1) & 3)) << 4));
}

// The power of two that a bf16 row is multiplied by, from its largest magnitude's bits; zeros, infinities and NaN stay.
__device__ __forceinline__ int code_query_shift(uint32_t most) {
  const int exponent = (int)(most >> 7);
  return exponent == 0 || exponent == 255 ? 0 : min(14 - (exponent - 127), 100);
}

// The rows lane / 4 and + 8 of Q as f16 operands: of 16 dimensions the lane's are (lane % 4) * 4 + {0, 1} and {2, 3}. unscale:
// what a row's products have to be multiplied by.
template <typename T, int D, typename Row>
__device__ __forceinline__ void code_queries(int dim, Row row, uint32_t (&qf)[D / 16][4], float (&unscale)[2]) {
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const T* src = row(e);  // null: no such row
    uint2 u[D / 16];
#pragma unroll
    for (int c = 0; c < D / 16; ++c)
      u[c] = src != nullptr && c * 16 + (threadIdx.x & 3) * 4 < dim ? __ldcg(reinterpret_cast<const uint2*>(src + c * 16 + (threadIdx.x & 3) * 4))
                                                                    : make_uint2(0u, 0u);
    unscale[e] = 1.f;
    if constexpr (Num<T>::is_bf16) {
      uint32_t most = 0u;  // magnitudes as whole numbers
#pragma unroll
      for (int c = 0; c < D / 16; ++c) {
        most = max(max(most, u[c].x & 0x7fffu), max(u[c].x >> 16 & 0x7fffu, max(u[c].y & 0x7fffu, u[c].y >> 16 & 0x7fffu)));
      }
      most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
      most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
      const int up = code_query_shift(most);
      const float f = __uint_as_float((uint32_t)(up + 127) << 23);
      unscale[e] = __uint_as_float((uint32_t)(127 - up) << 23);
#pragma unroll
      for (int c = 0; c < D / 16; ++c) {
        u[c].x = pack_round2<__half>(Pack2<T>::lo(u[c].x) * f, Pack2<T>::hi(u[c].x) * f);
        u[c].y = pack_round2<__half>(Pack2<T>::lo(u[c].y) * f, Pack2<T>::hi(u[c].y) * f);
      }
    }
#pragma unroll
    for (int c = 0; c < D / 16; ++c) {
      qf[c][e] = u[c].x;
      qf[c][2 + e] = u[c].y;
    }
  }
}

// What a warp has of an item so far: 16 rows.
template <int D>
struct CodeSums {
  float o[D / 8][4];     // tiles 2c and 2c + 1: even and odd columns of 16 c .. 16 c + 15
  float m[2], l[2];      // maximum and sum, the latter times 2^kCodeUp
  float most, inv_most;  // o is in units of the largest scale of V so far, times 2^kCodeUp
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int n = 0; n < D / 8; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
    m[0] = m[1] = -INFINITY;
    l[0] = l[1] = 0.f;
    most = inv_most = 0.f;
  }
  // In units of one, without the power of two; `weight`: of row e besides.
  __device__ __forceinline__ void settle(int e, float weight) {
    const float f = weight * 0x1p-15f;  // not times `most`: it may be as small as a normal number can
#pragma unroll
    for (int n = 0; n < D / 8; ++n) {
      o[n][2 * e] = o[n][2 * e] * f * most;
      o[n][2 * e + 1] = o[n][2 * e + 1] * f * most;
    }
  }
};

// The keys of one item and what its rows see of them.
struct CodeSpan {
  int kv, first;           // keys that some row sees
  int all_first, all_end;  // those that every row sees
  int limit[2], floor_[2]; // those of the lane's rows
  bool several;            // tokens
};

// 32 keys from j0 on, at row k0 of a tile of K at `ks` and of V at `vs`; key_f, value_f: the scales of each eight of them;
// row_f: what a row's products are multiplied by besides.
template <typename T, int D>
__device__ __forceinline__ void code_tile(CodeSums<D>& z, const uint32_t (&qf)[D / 16][4], const CodeSpan& it, uint32_t ks,
                                          uint32_t vs, int k0, int j0, const float4& key_f, const float4& value_f,
                                          const float (&row_f)[2]) {
  constexpr bool TWO = !Num<T>::is_bf16;  // terms of P
  const int lane = threadIdx.x & 31;
  float s[4][4];
#pragma unroll
  for (int n = 0; n < 4; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
  for (int c0 = 0; c0 < D / 16; c0 += 4) {  // 64 dimensions
    uint32_t kf[4][4];
#pragma unroll
    for (int n = 0; n < 4; ++n)
      ldsm_x4(ks + code_at<D>(k0 + n * 8 + (lane & 7), c0 + (lane >> 3)), kf[n][0], kf[n][1], kf[n][2], kf[n][3]);
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
      for (int n = 0; n < 4; ++n)
        mma_16816<__half>(s[n], qf[c0 + c][0], qf[c0 + c][1], qf[c0 + c][2], qf[c0 + c][3], codes_lo(kf[n][c]), codes_hi(kf[n][c]));
  }
  const float kf4[4] = {key_f.x, key_f.y, key_f.z, key_f.w};
  float vf4[4] = {value_f.x, value_f.y, value_f.z, value_f.w};
  const bool edge = j0 + 32 > it.all_end || j0 < it.all_first;
#pragma unroll
  for (int n = 0; n < 4; ++n) {
    const float f0 = kf4[n] * row_f[0], f1 = kf4[n] * row_f[1];
    s[n][0] *= f0;
    s[n][1] *= f0;
    s[n][2] *= f1;
    s[n][3] *= f1;
  }
  if (edge) {
#pragma unroll
    for (int n = 0; n < 4; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int j = j0 + n * 8 + (lane & 3) * 2 + (e & 1);
        if (j >= it.limit[e >> 1] || j < it.floor_[e >> 1]) s[n][e] = -INFINITY;
      }
  }
  // the scales of V relative to the largest so far
  const float most = fmaxf(fmaxf(fmaxf(vf4[0], vf4[1]), fmaxf(vf4[2], vf4[3])), kCodeLeast);
  if (most > z.most) {  // the whole warp
    const float f = z.most / most;
#pragma unroll
    for (int n = 0; n < D / 8; ++n) {
      z.o[n][0] *= f;
      z.o[n][1] *= f;
      z.o[n][2] *= f;
      z.o[n][3] *= f;
    }
    z.most = most;
    z.inv_most = 1.f / most;
  }
#pragma unroll
  for (int n = 0; n < 4; ++n) vf4[n] *= z.inv_most;
  uint32_t pf[2][4], pr[2][4];
  float fix[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    float top = fmaxf(fmaxf(fmaxf(s[0][2 * e], s[0][2 * e + 1]), fmaxf(s[1][2 * e], s[1][2 * e + 1])),
                      fmaxf(fmaxf(s[2][2 * e], s[2][2 * e + 1]), fmaxf(s[3][2 * e], s[3][2 * e + 1])));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const float m_new = fmaxf(z.m[e], top), ref = m_new == -INFINITY ? 0.f : m_new;
    fix[e] = exp2_fast(z.m[e] - ref);
    z.m[e] = m_new;
    const float base = ref - kCodeUp;
    float sum[4];
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const float p0 = exp2_fast(s[n][2 * e] - base), p1 = exp2_fast(s[n][2 * e + 1] - base);
      sum[n] = p0 + p1;
      const float w0 = p0 * vf4[n], w1 = p1 * vf4[n];
      uint32_t& hi = pf[n >> 1][(n & 1) * 2 + e];
      hi = pack_round2<__half>(w0, w1);
      if (TWO) pr[n >> 1][(n & 1) * 2 + e] = pack_round2<__half>(w0 - Pack2<__half>::lo(hi), w1 - Pack2<__half>::hi(hi));
    }
    z.l[e] = z.l[e] * fix[e] + ((sum[0] + sum[1]) + (sum[2] + sum[3]));
  }
  if (__any_sync(0xffffffffu, fix[0] != 1.f || fix[1] != 1.f)) {
#pragma unroll
    for (int n = 0; n < D / 8; ++n) {
      z.o[n][0] *= fix[0];
      z.o[n][1] *= fix[0];
      z.o[n][2] *= fix[1];
      z.o[n][3] *= fix[1];
    }
  }
  const bool clear = j0 + 32 > it.kv || j0 < it.first, mixed = edge && it.several;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    // V's fragments of 16 keys: the lane's are (lane % 4) * 2 + {0, 1} and + 8
    uint32_t vf[D / 16][2];
#pragma unroll
    for (int c = 0; c < D / 16; c += 2)
      ldsm_x4_trans(vs + code_at<D>(k0 + h * 16 + (lane & 15), c + (lane >> 4)), vf[c][0], vf[c][1], vf[c + 1][0], vf[c + 1][1]);
    if (clear) {  // codes of keys that no row sees may be NaN: 0 * NaN is
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int j = j0 + h * 16 + i * 8 + (lane & 3) * 2;
        const uint32_t keep = (j < it.kv && j >= it.first ? 0xffffu : 0u) | (j + 1 < it.kv && j + 1 >= it.first ? 0xffff0000u : 0u);
#pragma unroll
        for (int c = 0; c < D / 16; ++c) vf[c][i] &= keep;
      }
    }
    if (mixed) {  // and NaN of keys that only some rows see goes to these rows by itself
      uint32_t any = 0u;
#pragma unroll
      for (int c = 0; c < D / 16; ++c) any |= codes_nan(vf[c][0]) | codes_nan(vf[c][1]);
      if (__builtin_expect(__any_sync(0xffffffffu, any != 0u), 0)) {
        const float nan = __uint_as_float(0x7fc00000u);
#pragma unroll 1
        for (int i = 0; i < 16; ++i) {
          const int j = j0 + h * 16 + i;
          if (j < it.first || j >= it.kv) continue;
#pragma unroll
          for (int c = 0; c < D / 16; ++c) {
            uint32_t x;
            asm volatile("ld.shared.b32 %0, [%1];" : "=r"(x) : "r"(vs + code_at<D>(k0 + h * 16 + i, c) + (lane & 3) * 4));
            x = codes_nan(x);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              if (j >= it.limit[e] || j < it.floor_[e]) continue;
              if (x & 0x80u) z.o[2 * c][2 * e] = nan;
              if (x & 0x8000u) z.o[2 * c + 1][2 * e] = nan;
              if (x & 0x800000u) z.o[2 * c][2 * e + 1] = nan;
              if (x & 0x80000000u) z.o[2 * c + 1][2 * e + 1] = nan;
            }
          }
        }
#pragma unroll
        for (int c = 0; c < D / 16; ++c)
#pragma unroll
          for (int i = 0; i < 2; ++i) vf[c][i] &= ~((codes_nan(vf[c][i]) >> 7) * 0xffu);
      }
    }
#pragma unroll
    for (int c = 0; c < D / 16; ++c) {
      // {even, odd} columns of two keys -> even columns of both, odd columns of both
      const uint32_t x = __byte_perm(vf[c][0], 0u, 0x3120), y = __byte_perm(vf[c][1], 0u, 0x3120);
      const uint32_t x0 = codes_lo(x), y0 = codes_lo(y), x1 = codes_hi(x), y1 = codes_hi(y);
      mma_16816<__half>(z.o[2 * c], pf[h][0], pf[h][1], pf[h][2], pf[h][3], x0, y0);
      mma_16816<__half>(z.o[2 * c + 1], pf[h][0], pf[h][1], pf[h][2], pf[h][3], x1, y1);
      if (TWO) {
        mma_16816<__half>(z.o[2 * c], pr[h][0], pr[h][1], pr[h][2], pr[h][3], x0, y0);
        mma_16816<__half>(z.o[2 * c + 1], pr[h][0], pr[h][1], pr[h][2], pr[h][3], x1, y1);
      }
    }
  }
}

// ---- up to eight rows: keys and columns take the sixteen rows of a product, queries its eight columns, so that it
// takes half as many of them, and half the registers for Q, scores and sums ----

__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// Row lane / 4 of Q as code_queries has it. unscale: of the rows (lane % 4) * 2 and + 1.
template <typename T, int D>
__device__ __forceinline__ void code_queries_few(int dim, const T* src, uint32_t (&qf)[D / 16][2], float (&unscale)[2]) {
  const int lane = threadIdx.x & 31;
  uint2 u[D / 16];
#pragma unroll
  for (int c = 0; c < D / 16; ++c)
    u[c] = src != nullptr && c * 16 + (lane & 3) * 4 < dim ? __ldcg(reinterpret_cast<const uint2*>(src + c * 16 + (lane & 3) * 4))
                                                           : make_uint2(0u, 0u);
  float back = 1.f;
  if constexpr (Num<T>::is_bf16) {
    uint32_t most = 0u;
#pragma unroll
    for (int c = 0; c < D / 16; ++c)
      most = max(max(most, u[c].x & 0x7fffu), max(u[c].x >> 16 & 0x7fffu, max(u[c].y & 0x7fffu, u[c].y >> 16 & 0x7fffu)));
    most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
    most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
    const int up = code_query_shift(most);
    const float f = __uint_as_float((uint32_t)(up + 127) << 23);
    back = __uint_as_float((uint32_t)(127 - up) << 23);
#pragma unroll
    for (int c = 0; c < D / 16; ++c) {
      u[c].x = pack_round2<__half>(Pack2<T>::lo(u[c].x) * f, Pack2<T>::hi(u[c].x) * f);
      u[c].y = pack_round2<__half>(Pack2<T>::lo(u[c].y) * f, Pack2<T>::hi(u[c].y) * f);
    }
  }
#pragma unroll
  for (int c = 0; c < D / 16; ++c) {
    qf[c][0] = u[c].x;
    qf[c][1] = u[c].y;
  }
#pragma unroll
  for (int e = 0; e < 2; ++e) unscale[e] = __shfl_sync(0xffffffffu, back, ((lane & 3) * 2 + e) * 4);
}

template <int D>
struct CodeSumsFew {
  float o[D / 16][4];    // columns 16 c + (lane / 4) * 2 and + 1 of the two rows: {first, second} of the even one, of the odd one
  float m[2], l[2];      // as in CodeSums, of rows (lane % 4) * 2 and + 1; l of the lane's keys
  float most, inv_most;
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int c = 0; c < D / 16; ++c) o[c][0] = o[c][1] = o[c][2] = o[c][3] = 0.f;
    m[0] = m[1] = -INFINITY;
    l[0] = l[1] = 0.f;
    most = inv_most = 0.f;
  }
  __device__ __forceinline__ void scale(float a, float b) {
#pragma unroll
    for (int c = 0; c < D / 16; ++c) {
      o[c][0] *= a;
      o[c][1] *= b;
      o[c][2] *= a;
      o[c][3] *= b;
    }
  }
  __device__ __forceinline__ void settle(int e, float weight) {
    const float f = weight * 0x1p-15f;
#pragma unroll
    for (int c = 0; c < D / 16; ++c) {
      o[c][e] = o[c][e] * f * most;
      o[c][2 + e] = o[c][2 + e] * f * most;
    }
  }
};

// As code_tile.
template <typename T, int D>
__device__ __forceinline__ void code_tile_few(CodeSumsFew<D>& z, const uint32_t (&qf)[D / 16][2], const CodeSpan& it, uint32_t ks,
                                              uint32_t vs, int k0, int j0, const float4& key_f, const float4& value_f,
                                              const float (&row_f)[2]) {
  constexpr bool TWO = !Num<T>::is_bf16;
  const int lane = threadIdx.x & 31;
  // scores of keys lane / 4 (+ 8 n) for rows (lane % 4) * 2 and + 1; two chains a tile of 16 keys
  float s[2][2][4];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) s[i][0][e] = s[i][1][e] = 0.f;
#pragma unroll
  for (int c0 = 0; c0 < D / 16; c0 += 4) {  // 64 dimensions
    uint32_t kf[4][4];
#pragma unroll
    for (int n = 0; n < 4; ++n)
      ldsm_x4(ks + code_at<D>(k0 + n * 8 + (lane & 7), c0 + (lane >> 3)), kf[n][0], kf[n][1], kf[n][2], kf[n][3]);
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
      for (int i = 0; i < 2; ++i)
        mma_16816<__half>(s[i][c & 1], codes_lo(kf[2 * i][c]), codes_lo(kf[2 * i + 1][c]), codes_hi(kf[2 * i][c]),
                          codes_hi(kf[2 * i + 1][c]), qf[c0 + c][0], qf[c0 + c][1]);
  }
  // V's fragments of the first 16 keys, in flight during the softmax
  uint32_t vf[D / 16][2];
  auto load_v = [&](int h) {
#pragma unroll
    for (int c = 0; c < D / 16; c += 2)
      ldsm_x4_trans(vs + code_at<D>(k0 + h * 16 + (lane & 15), c + (lane >> 4)), vf[c][0], vf[c][1], vf[c + 1][0], vf[c + 1][1]);
  };
  load_v(0);
  const float kf4[4] = {key_f.x, key_f.y, key_f.z, key_f.w};
  float vf4[4] = {value_f.x, value_f.y, value_f.z, value_f.w};
  const bool edge = j0 + 32 > it.all_end || j0 < it.all_first;
  float x[4][2];  // eight keys a step, rows
#pragma unroll
  for (int n = 0; n < 4; ++n)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      x[n][e] = (s[n >> 1][0][(n & 1) * 2 + e] + s[n >> 1][1][(n & 1) * 2 + e]) * (kf4[n] * row_f[e]);
      if (edge) {
        const int j = j0 + n * 8 + (lane >> 2);
        if (j >= it.limit[e] || j < it.floor_[e]) x[n][e] = -INFINITY;
      }
    }
  const float most = fmaxf(fmaxf(fmaxf(vf4[0], vf4[1]), fmaxf(vf4[2], vf4[3])), kCodeLeast);
  if (most > z.most) {  // the whole warp
    const float f = z.most / most;
    z.scale(f, f);
    z.most = most;
    z.inv_most = 1.f / most;
  }
#pragma unroll
  for (int n = 0; n < 4; ++n) vf4[n] *= z.inv_most;
  float fix[2], base[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    float top = fmaxf(fmaxf(x[0][e], x[1][e]), fmaxf(x[2][e], x[3][e]));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
    const float m_new = fmaxf(z.m[e], top), ref = m_new == -INFINITY ? 0.f : m_new;
    fix[e] = exp2_fast(z.m[e] - ref);
    z.m[e] = m_new;
    base[e] = ref - kCodeUp;
  }
  if (__any_sync(0xffffffffu, fix[0] != 1.f || fix[1] != 1.f)) z.scale(fix[0], fix[1]);
  uint32_t pf[4], pr[4];  // of eight keys each, transposed: the lane's keys are (lane % 4) * 2 and + 1, its row lane / 4
  float sum[2] = {0.f, 0.f};
#pragma unroll
  for (int n = 0; n < 4; ++n) {
    const float p0 = exp2_fast(x[n][0] - base[0]), p1 = exp2_fast(x[n][1] - base[1]);
    sum[0] += p0;
    sum[1] += p1;
    const float w0 = p0 * vf4[n], w1 = p1 * vf4[n];
    const uint32_t hi = pack_round2<__half>(w0, w1);
    pf[n] = transpose_8x8(hi);
    if (TWO) pr[n] = transpose_8x8(pack_round2<__half>(w0 - Pack2<__half>::lo(hi), w1 - Pack2<__half>::hi(hi)));
  }
  z.l[0] = z.l[0] * fix[0] + sum[0];
  z.l[1] = z.l[1] * fix[1] + sum[1];
  const bool clear = j0 + 32 > it.kv || j0 < it.first, mixed = edge && it.several;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    if (h == 1) load_v(1);
    if (clear) {  // codes of keys that no row sees may be NaN: 0 * NaN is
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int j = j0 + h * 16 + i * 8 + (lane & 3) * 2;
        const uint32_t keep = (j < it.kv && j >= it.first ? 0xffffu : 0u) | (j + 1 < it.kv && j + 1 >= it.first ? 0xffff0000u : 0u);
#pragma unroll
        for (int c = 0; c < D / 16; ++c) vf[c][i] &= keep;
      }
    }
    if (mixed) {  // and NaN of keys that only some rows see goes to these rows by itself
      uint32_t any = 0u;
#pragma unroll
      for (int c = 0; c < D / 16; ++c) any |= codes_nan(vf[c][0]) | codes_nan(vf[c][1]);
      if (__builtin_expect(__any_sync(0xffffffffu, any != 0u), 0)) {
        const float nan = __uint_as_float(0x7fc00000u);
#pragma unroll 1
        for (int i = 0; i < 16; ++i) {
          const int j = j0 + h * 16 + i;
          if (j < it.first || j >= it.kv) continue;
#pragma unroll
          for (int c = 0; c < D / 16; ++c) {
            unsigned short w;
            asm volatile("ld.shared.u16 %0, [%1];" : "=h"(w) : "r"(vs + code_at<D>(k0 + h * 16 + i, c) + (lane >> 2) * 2));
            const uint32_t two = codes_nan(w);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              if (j >= it.limit[e] || j < it.floor_[e]) continue;
              if (two & 0x80u) z.o[c][e] = nan;
              if (two & 0x8000u) z.o[c][2 + e] = nan;
            }
          }
        }
#pragma unroll
        for (int c = 0; c < D / 16; ++c)
#pragma unroll
          for (int i = 0; i < 2; ++i) vf[c][i] &= ~((codes_nan(vf[c][i]) >> 7) * 0xffu);
      }
    }
#pragma unroll
    for (int c = 0; c < D / 16; ++c) {
      // {even, odd} columns of two keys -> even columns of both, odd columns of both: rows 0 - 7 and 8 - 15 of the product
      const uint32_t a = __byte_perm(vf[c][0], 0u, 0x3120), b = __byte_perm(vf[c][1], 0u, 0x3120);
      const uint32_t a0 = codes_lo(a), a1 = codes_hi(a), a2 = codes_lo(b), a3 = codes_hi(b);
      mma_16816<__half>(z.o[c], a0, a1, a2, a3, pf[2 * h], pf[2 * h + 1]);
      if (TWO) mma_16816<__half>(z.o[c], a0, a1, a2, a3, pr[2 * h], pr[2 * h + 1]);
    }
  }
}

}  // namespace mlora
