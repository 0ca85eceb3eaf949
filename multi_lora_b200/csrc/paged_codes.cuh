// Tiles of e4m3 codes under the warp-level tensor cores.
//
// A code is exact in f16, so codes enter the products as they are and their scales stay outside, in
// fp32: a key's multiplies its score, a value's the probability that goes to the second product.
//   * Q is taken in f16. f16 queries are; a bf16 row is multiplied by the power of two that brings its largest
//     element to 2^14 .. 2^15 (undone on the score), which keeps its 8 bits down to 2^-29 of that
//     element and anything below to 2^-40 of it.
//   * P times the value's scale is taken in f16 in a unit of the row's own, in which the largest such product
//     that the row has met is 2^11 or more: 11 bits of it (of f16 queries, whose result has as many, two
//     terms: 21 bits), and nothing coarser than 2^-36 of the row's largest. (In units of the largest scale of a tile,
//     values behind or beside a block of much larger ones lost their bits, for rows that do not see that block too.)
// Four codes of a register are two operands of the product as they lie: of a row of K the dimension may be taken in any order
// (Q in the same), and of V, transposed in pairs of columns, the even columns make one tile of eight and
// the odd ones another, so that a thread ends up with four columns side by side.
#pragma once

#include "float2.cuh"
#include "mma.cuh"
#include "paged_sched.cuh"

namespace mlora {

constexpr int kCodeTile = 128;  // keys a stage: 32 of them a warp

// What enters the second product for a score x and the scale f of its value is w = exp2(x - m) f up, with a running maximum m
// and a unit 1 / up of the row's own. `up` makes the largest exp2(x - m) f of the tile that it was chosen for a small power of
// two (with nothing of it lost), and stays until a w would pass 2^kCodeTop or a score is kCodeRaise above m: then both
// are chosen again. So sums seldom have to be multiplied, and w is in f16's range. What a row goes by hangs on nothing
// but scores and scales of keys that it sees. up is at most 2^126, whose reciprocal is a normal number.
constexpr float kCodeTop = 15.75f, kCodeRaise = 24.f;
constexpr float kCodeNone = -0x1.fffffep127f;  // the maximum of a row that has met nothing: finite, differences are no NaN
constexpr float kCodeMostUp = 0x1p126f;
constexpr float kCodeWide = 0x1p18f;  // a larger maximum is chosen again at every tile: sums with it are too coarse

// log2 f, taken as linear between powers of two: too small by at most 0.09. f >= 0; -127 of zero and minus zero.
__device__ __forceinline__ float code_log(float f) { return fmaf((float)(__float_as_uint(f) & 0x7fffffffu), 0x1p-23f, -127.f); }
// What a score and code_log of its value's scale may have as their sum: w is below 2^(kCodeTop + 0.14) then (0.05 are
// lost to rounding), and f16 ends at 2^15.99.
__device__ __forceinline__ float code_limit(float m, float up) {
  return fabsf(m) < kCodeWide ? m + (kCodeTop - __log2f(up)) : -INFINITY;
}
// f up, finite: a probability that it meets may be zero.
__device__ __forceinline__ float code_weight(float f, float up) { return fminf(f * up, 0x1.fffffep127f); }
__device__ __forceinline__ float code_inverse(float x) {  // two units off at most; infinity below 2^-128
  float y;
  asm("rcp.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// The unit in which `largest` is `as`, where the maximum was raised by `raised`: sums so far are not made larger.
__device__ __forceinline__ float code_new_up(float as, float up, float raised, float largest) {
  return fminf(fminf(as * code_inverse(largest), up * exp2_fast(raised)), kCodeMostUp);
}
// What sums in the old unit are multiplied by; `fix`: exp2(-raised).
__device__ __forceinline__ float code_rescale(float fix, float up, float next) {
  return fix * fminf(next * code_inverse(up), 0x1.fffffep127f);
}

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
  float m[2], l[2];      // maximum and sum
  float up[2];           // o is in units of 1 / up
  float limit[2];        // code_limit
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int n = 0; n < D / 8; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
    m[0] = m[1] = kCodeNone;
    l[0] = l[1] = 0.f;
    up[0] = up[1] = kCodeMostUp;
    limit[0] = limit[1] = -INFINITY;
  }
  __device__ __forceinline__ void scale(float a, float b) {
#pragma unroll
    for (int n = 0; n < D / 8; ++n) {
      o[n][0] *= a;
      o[n][1] *= a;
      o[n][2] *= b;
      o[n][3] *= b;
    }
  }
  // Row e in units of one, and times `weight`. (Where that product is subnormal, another part of the row is 2^-24 or more.)
  __device__ __forceinline__ void settle(int e, float weight) {
    const float f = weight * code_inverse(up[e]);
#pragma unroll
    for (int n = 0; n < D / 8; ++n) {
      o[n][2 * e] *= f;
      o[n][2 * e + 1] *= f;
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

// New maxima and units of those of a warp's rows that need them, from 32 keys: `top`, a score or the larger of two of eight keys
// each, and the scales of their values; lanes A, B (and C) apart have the other keys of a row.
// What a row goes by hangs on its own scores alone: others' may be of keys that it does not see.
template <int A, int B, int C = 0, typename Sums>
__device__ __forceinline__ void code_raise(Sums& z, const float (&top)[4][2], const float (&f)[4], const bool (&need)[2]) {
  auto over_lanes = [](float x) {
    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, A));
    x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, B));
    return C > 0 ? fmaxf(x, __shfl_xor_sync(0xffffffffu, x, C)) : x;
  };
  const int lane = threadIdx.x & 31;
  const uint32_t row = C > 0 ? 0x11111111u << (lane & 3) : 0xfu << (lane & 28);  // its lanes
  float fix[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const bool again = (__ballot_sync(0xffffffffu, need[e]) & row) != 0u;
    const float most = over_lanes(fmaxf(fmaxf(top[0][e], top[1][e]), fmaxf(top[2][e], top[3][e])));
    const float raised = again && most > z.m[e] ? most - z.m[e] : 0.f, back = exp2_fast(-raised);
    if (again) z.m[e] = fmaxf(z.m[e], most);
    float largest = 0.f;
#pragma unroll
    for (int n = 0; n < 4; ++n) largest = fmaxf(largest, f[n] * exp2_fast(top[n][e] - z.m[e]));
    largest = over_lanes(largest);
    const float up = again ? code_new_up(0x1p11f, z.up[e], raised, largest) : z.up[e];
    z.l[e] *= back;
    fix[e] = again ? code_rescale(back, z.up[e], up) : 1.f;
    z.up[e] = up;
    z.limit[e] = code_limit(z.m[e], up);
  }
  z.scale(fix[0], fix[1]);
}

// 32 keys from j0 on, at row k0 of a tile of K at `ks` and of V at `vs`; key_f, value_f: the scales of each eight of them,
// value_log: code_log of the latter; row_f: what a row's products are multiplied by besides.
template <typename T, int D>
__device__ __forceinline__ void code_tile(CodeSums<D>& z, const uint32_t (&qf)[D / 16][4], const CodeSpan& it, uint32_t ks,
                                          uint32_t vs, int k0, int j0, const float4& key_f, const float4& value_f,
                                          const float4& value_log, const float (&row_f)[2]) {
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
  const float vf4[4] = {value_f.x, value_f.y, value_f.z, value_f.w};
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
  float top[4][2];  // the larger of the lane's scores of eight keys
  bool need[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
#pragma unroll
    for (int n = 0; n < 4; ++n) top[n][e] = fmaxf(s[n][2 * e], s[n][2 * e + 1]);
    need[e] = fmaxf(max3(top[0][e], top[1][e], top[2][e]), top[3][e]) > z.m[e] + kCodeRaise ||
              fmaxf(max3(top[0][e] + value_log.x, top[1][e] + value_log.y, top[2][e] + value_log.z), top[3][e] + value_log.w) >
                  z.limit[e];
  }
  if (__any_sync(0xffffffffu, need[0] || need[1])) code_raise<1, 2>(z, top, vf4, need);
  uint32_t pf[2][4], pr[2][4];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const uint64_t m2 = pack2(-z.m[e], -z.m[e]), up2 = pack2(z.up[e], z.up[e]);
    uint64_t sum = 0;
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const uint64_t x = add2(pack2(s[n][2 * e], s[n][2 * e + 1]), m2), p = pack2(exp2_fast(lo_of(x)), exp2_fast(hi_of(x)));
      sum = add2(sum, p);
      // f first: it and the unit may be far apart, with a probability of zero between them
      const uint64_t w = mul2(mul2(p, pack2(vf4[n], vf4[n])), up2);
      uint32_t& hi = pf[n >> 1][(n & 1) * 2 + e];
      hi = pack_round2<__half>(lo_of(w), hi_of(w));
      if (TWO) pr[n >> 1][(n & 1) * 2 + e] = pack_round2<__half>(lo_of(w) - Pack2<__half>::lo(hi), hi_of(w) - Pack2<__half>::hi(hi));
    }
    z.l[e] += lo_of(sum) + hi_of(sum);
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
  float up[2], limit[2];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int c = 0; c < D / 16; ++c) o[c][0] = o[c][1] = o[c][2] = o[c][3] = 0.f;
    m[0] = m[1] = kCodeNone;
    l[0] = l[1] = 0.f;
    up[0] = up[1] = kCodeMostUp;
    limit[0] = limit[1] = -INFINITY;
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
    const float f = weight * code_inverse(up[e]);
#pragma unroll
    for (int c = 0; c < D / 16; ++c) {
      o[c][e] *= f;
      o[c][2 + e] *= f;
    }
  }
};

// As code_tile.
template <typename T, int D>
__device__ __forceinline__ void code_tile_few(CodeSumsFew<D>& z, const uint32_t (&qf)[D / 16][2], const CodeSpan& it, uint32_t ks,
                                              uint32_t vs, int k0, int j0, const float4& key_f, const float4& value_f,
                                              const float4& value_log, const float (&row_f)[2]) {
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
  const float vf4[4] = {value_f.x, value_f.y, value_f.z, value_f.w};
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
  uint64_t size[4];
#pragma unroll
  for (int n = 0; n < 4; ++n) {
    const float f = n == 0 ? value_log.x : n == 1 ? value_log.y : n == 2 ? value_log.z : value_log.w;
    size[n] = add2(pack2(x[n][0], x[n][1]), pack2(f, f));
  }
  const bool need[2] = {fmaxf(max3(x[0][0], x[1][0], x[2][0]), x[3][0]) > z.m[0] + kCodeRaise ||
                            fmaxf(max3(lo_of(size[0]), lo_of(size[1]), lo_of(size[2])), lo_of(size[3])) > z.limit[0],
                        fmaxf(max3(x[0][1], x[1][1], x[2][1]), x[3][1]) > z.m[1] + kCodeRaise ||
                            fmaxf(max3(hi_of(size[0]), hi_of(size[1]), hi_of(size[2])), hi_of(size[3])) > z.limit[1]};
  if (__any_sync(0xffffffffu, need[0] || need[1])) code_raise<4, 8, 16>(z, x, vf4, need);
  const uint64_t m2 = pack2(-z.m[0], -z.m[1]), up2 = pack2(z.up[0], z.up[1]);
  uint32_t pf[4], pr[4];  // of eight keys each, transposed: the lane's keys are (lane % 4) * 2 and + 1, its row lane / 4
  uint64_t sum = 0;
#pragma unroll
  for (int n = 0; n < 4; ++n) {
    const uint64_t d = add2(pack2(x[n][0], x[n][1]), m2), p = pack2(exp2_fast(lo_of(d)), exp2_fast(hi_of(d)));
    sum = add2(sum, p);
    const uint64_t w = mul2(mul2(p, pack2(vf4[n], vf4[n])), up2);
    const uint32_t hi = pack_round2<__half>(lo_of(w), hi_of(w));
    pf[n] = transpose_8x8(hi);
    if (TWO) pr[n] = transpose_8x8(pack_round2<__half>(lo_of(w) - Pack2<__half>::lo(hi), hi_of(w) - Pack2<__half>::hi(hi)));
  }
  z.l[0] += lo_of(sum);
  z.l[1] += hi_of(sum);
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
