// New keys (rotated) and values into a paged cache of e4m3 codes with a scale for each
// block and head, and the step's queries rotated, in one launch.
//
// A value x is held as a code c with x ~ c * f, f the scale of its block and head. Scales are powers of
// two: f = 2^k with the smallest k for which the largest finite |x| of the rows that a call
// brings to the block is at most 448 * 2^k, and not less than the block's own scale where it holds
// rows before them. So a row costs what e4m3 costs and no more (a floating-point code loses
// nothing by a power of two), and where a scale grows the older rows' codes follow without an error, but for those
// that fall among e4m3's subnormals, which are rounded to nearest even. Infinities are held as +-448 f, NaN as NaN.
// The rotated key is quantised from fp32: it is rounded once.
//
// New rows of a block are a run: consecutive tokens with consecutive slots, which begins where the slot is not the
// one behind its predecessor's or begins a block. A CTA takes the runs that begin in a window of tokens, whole,
// with some of the heads, K and V: it has every row that a scale depends on, so nothing
// is agreed on between CTAs. Four units a thread (two vectors each) wait in registers between the maximum and the
// codes; more are read again. Memory bounds it, with few rows the latency of
// slots, rows and scales, one after the other.
#include <cuda_fp8.h>

#include <climits>

#include "device.h"
#include "kernels.h"
#include "paged.h"
#include "paged_append.cuh"

namespace mlora {

constexpr int kCodeUnits = 4, kCodeWindow = 32;

// What the host decides about a launch.
struct CodeShape {
  int q_ctas, q_per_cta;   // CTAs that rotate queries, tokens each
  int units;               // of a row
  int window, parts, part_heads;
  int max_rows, turn_rows; // rows that runs of a window can have; of those with {cos, sin} in shared memory
};

// The scale of rows whose largest magnitude is `most`: 448 = 1.75 * 2^8.
__device__ __forceinline__ float code_scale(float most) {
  const int k = (int)((__float_as_uint(most) + 0x1fffffu) >> 23) - 127 - 8;
  return most > 0.f ? __uint_as_float((uint32_t)(max(k, -100) + 127) << 23) : 0x1p-100f;
}

// V values over the scale, rounded to codes at dst.
template <int V>
__device__ __forceinline__ void store_codes(unsigned char* dst, const float (&x)[V], float scale) {
  float y[V];
  if ((__float_as_uint(scale) & 0x7fffffu) == 0) {  // a power of two: its reciprocal is exact
    const float inv = 1.f / scale;
#pragma unroll
    for (int i = 0; i < V; ++i) y[i] = x[i] * inv;
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) y[i] = x[i] / scale;
  }
  if constexpr (V == 1) {
    *dst = (unsigned char)__nv_cvt_float_to_fp8(y[0], __NV_SATFINITE, __NV_E4M3);
  } else {
    union {
      typename RawBytes<V>::type raw;
      unsigned short pair[V / 2];
    } u;
#pragma unroll
    for (int i = 0; i < V; i += 2)
      u.pair[i / 2] = __nv_cvt_float2_to_fp8x2(make_float2(y[i], y[i + 1]), __NV_SATFINITE, __NV_E4M3);
    *reinterpret_cast<typename RawBytes<V>::type*>(dst) = u.raw;
  }
}

template <typename T, int V>
__global__ void __launch_bounds__(kRotNT) paged_append_codes_kernel(const PagedAppendArgs p, const CodeShape g) {
  extern __shared__ __align__(16) unsigned char s_dyn[];
  float2* s_turn = reinterpret_cast<float2*>(s_dyn);
  pdl_wait();
  pdl_trigger();
  if ((int)blockIdx.x < g.q_ctas) {
    append_rows<T, V>(p, 0, blockIdx.x, g.q_per_cta, g.units, s_turn);
    return;
  }
  __shared__ int s_rows, s_runs, s_grown;
  __shared__ int s_first[kCodeWindow];  // row that a run begins with
  int* s_slot = reinterpret_cast<int*>(s_turn + g.turn_rows * p.angles.pairs);  // [max_rows], -1: not of a run that begins here
  short* s_run = reinterpret_cast<short*>(s_slot + g.max_rows);                // [max_rows]
  uint32_t* s_most = reinterpret_cast<uint32_t*>(s_run + (g.max_rows + 1) / 2 * 2);  // [window][2 part_heads]
  float* s_scale = reinterpret_cast<float*>(s_most + g.window * 2 * g.part_heads);
  float* s_ratio = s_scale + g.window * 2 * g.part_heads;
  const int tid = threadIdx.x, lane = tid & 31;
  const int cta = blockIdx.x - g.q_ctas, part = cta % g.parts, t0 = cta / g.parts * g.window;
  const int head0 = part * g.part_heads, heads = min(g.part_heads, p.kv_heads - head0), items = 2 * heads;

  // ---- the runs that begin in the window ----
  if (tid < 32) {
    auto slot_at = [&](int t) { return t >= 0 && t < p.tokens ? __ldcg(p.slot_map + t) : -1; };
    const int t = t0 + lane, before = lane < g.window ? slot_at(t - 1) : -1;
    int slot = lane < g.window ? slot_at(t) : -1;
    bool begins = slot >= 0 && (before < 0 || before + 1 != slot || slot % p.block_size == 0);
    if (slot >= 0 && slot / p.block_size >= p.num_blocks) {
      if (part == 0) flag_error(p.status, kErrKvRange);
      slot = -1;
      begins = false;
    }
    const unsigned mask = __ballot_sync(0xffffffffu, begins);
    const int run = __popc(mask & (0xffffffffu >> (31 - lane))) - 1;
    int rows = 0;
    if (mask != 0u) {
      if (lane < g.window) {
        s_slot[lane] = run >= 0 ? slot : -1;
        s_run[lane] = (short)run;
      }
      if (begins) s_first[run] = lane;
      const int last = __shfl_sync(0xffffffffu, slot, g.window - 1), last_run = __shfl_sync(0xffffffffu, run, 31);
      rows = min(g.window, p.tokens - t0);
      // the last run behind the window's end: at most the rest of its block
      for (int most = last >= 0 ? p.block_size - 1 - last % p.block_size : 0; most > 0; most -= 32) {
        const int r = rows + lane;
        const int want = last + 1 + r - g.window;
        const bool goes = lane < most && slot_at(t0 + r) == want;
        const unsigned more = __ballot_sync(0xffffffffu, goes);
        const int n = more == 0xffffffffu ? 32 : __ffs(~more) - 1;
        if (lane < n) {
          s_slot[r] = want;
          s_run[r] = (short)last_run;
        }
        rows += n;
        if (n < 32) break;
      }
    }
    if (lane == 0) {
      s_rows = rows;
      s_runs = __popc(mask);
      s_grown = 0;
    }
  }
  __syncthreads();
  const int rows = s_rows, runs = s_runs;
  if (rows == 0) return;
  for (int i = tid; i < runs * items; i += kRotNT) s_most[i] = 0u;
  const bool rotated = p.angles.turns != nullptr;
  const int all = rows * items * g.units, chunks = (all + kRotNT * kCodeUnits - 1) / (kRotNT * kCodeUnits);

  struct Unit {
    Vec<T, V> x[2];
    RotaryUnit un;
    int row, item;  // row < 0: none
  };
  Unit w[kCodeUnits];
  auto load = [&](int chunk) {
#pragma unroll
    for (int k = 0; k < kCodeUnits; ++k) {
      const int at = (chunk * kCodeUnits + k) * kRotNT + tid;
      w[k].row = -1;
      if (at >= all) continue;
      const int piece = at / g.units, u = at - piece * g.units, row = piece / items;
      w[k].item = piece - row * items;
      if (s_slot[row] < 0) continue;
      w[k].row = row;
      const int side = w[k].item >= heads, h = head0 + w[k].item - side * heads;
      const PagedSide& s = p.side[side];
      w[k].un = rotary_unit(p.angles, side == 0 && rotated, p.dim, V, u);
      const T* src = static_cast<const T*>(s.src) + (int64_t)(t0 + row) * s.src_token + h * s.src_head;
      w[k].x[0].load(src + w[k].un.e0);
      if (w[k].un.both) w[k].x[1].load(src + w[k].un.e1);
    }
  };
  auto values = [&](const Unit& w, float (&a)[V], float (&b)[V]) {
    w.x[0].to_f(a);
    w.x[1].to_f(b);
    if (!w.un.turned) return;
    if (w.row < g.turn_rows) {
      rotary_apply<V>(p.angles.interleaved != 0, s_turn + w.row * p.angles.pairs + w.un.pair, a, b);
    } else {
      float2 cs[V];
      const int position = __ldcg(p.angles.positions + t0 + w.row);
#pragma unroll
      for (int i = 0; i < V; ++i) cs[i] = rotary_turn(__ldg(p.angles.turns + w.un.pair + i), position, p.angles.factor);
      rotary_apply<V>(p.angles.interleaved != 0, cs, a, b);
    }
  };

  load(0);
  if (rotated) rotary_table(p.angles, t0, min(rows, g.turn_rows), s_turn);
  __syncthreads();
  // ---- the largest magnitudes ----
  const bool lanes_share = (g.units & (g.units - 1)) == 0 && g.units <= 32;  // a row's units lie in aligned lanes
  for (int c = 0; c < chunks; ++c) {
    if (c > 0) load(c);
#pragma unroll
    for (int k = 0; k < kCodeUnits; ++k) {
      uint32_t most = 0u;  // of magnitudes as whole numbers, in the same order
      if (w[k].row >= 0) {
        float a[V], b[V];
        values(w[k], a, b);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const uint32_t ua = __float_as_uint(a[i]) & 0x7fffffffu, ub = __float_as_uint(b[i]) & 0x7fffffffu;
          if (ua < 0x7f800000u) most = max(most, ua);
          if (ub < 0x7f800000u && w[k].un.both) most = max(most, ub);
        }
      }
      if (lanes_share)
        for (int o = g.units >> 1; o > 0; o >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
      if (w[k].row >= 0 && most != 0u && (!lanes_share || (lane & (g.units - 1)) == 0))
        atomicMax(s_most + s_run[w[k].row] * items + w[k].item, most);
    }
  }
  __syncthreads();
  // ---- the scales ----
  for (int i = tid; i < runs * items; i += kRotNT) {
    const int run = i / items, item = i - run * items, side = item >= heads, h = head0 + item - side * heads;
    const int slot = s_slot[s_first[run]], block = slot / p.block_size;
    float* at = p.scale[side] + block * p.scale_block[side] + h * p.scale_head[side];
    float scale = code_scale(__uint_as_float(s_most[i])), ratio = 1.f;
    if (slot - block * p.block_size > 0) {
      const float old = __ldcg(at);
      if (old < scale) ratio = old / scale;
      scale = fmaxf(scale, old);
    }
    *at = scale;
    s_scale[i] = scale;
    s_ratio[i] = ratio;
    if (ratio != 1.f) s_grown = 1;
  }
  __syncthreads();
  // ---- the codes ----
  for (int c = chunks - 1; c >= 0; --c) {
    if (c < chunks - 1) load(c);
#pragma unroll
    for (int k = 0; k < kCodeUnits; ++k) {
      if (w[k].row < 0) continue;
      float a[V], b[V];
      values(w[k], a, b);
      const int slot = s_slot[w[k].row], block = slot / p.block_size, off = slot - block * p.block_size;
      const int side = w[k].item >= heads, h = head0 + w[k].item - side * heads;
      const PagedSide& s = p.side[side];
      unsigned char* dst = static_cast<unsigned char*>(s.dst) + block * s.block + off * s.slot + h * s.head;
      const float scale = s_scale[s_run[w[k].row] * items + w[k].item];
      store_codes<V>(dst + w[k].un.e0, a, scale);
      if (w[k].un.both) store_codes<V>(dst + w[k].un.e1, b, scale);
    }
  }
  if (s_grown == 0) return;
  // ---- older rows of blocks whose scales have grown ----
  for (int i = 0; i < runs * items; ++i) {
    const float ratio = s_ratio[i];
    if (ratio == 1.f) continue;
    const int run = i / items, item = i - run * items, side = item >= heads, h = head0 + item - side * heads;
    const int slot = s_slot[s_first[run]], block = slot / p.block_size, off = slot - block * p.block_size;
    const PagedSide& s = p.side[side];
    unsigned char* base = static_cast<unsigned char*>(s.dst) + block * s.block + h * s.head;
    const int pieces = p.dim / V;
    for (int e = tid; e < off * pieces; e += kRotNT) {
      const int row = e / pieces;
      unsigned char* at = base + row * s.slot + (e - row * pieces) * V;
      union {
        typename RawBytes<V>::type raw;
        unsigned char code[V];
      } u;
      u.raw = *reinterpret_cast<const typename RawBytes<V>::type*>(at);
      float x[V];
#pragma unroll
      for (int j = 0; j < V; ++j) x[j] = __half2float(__half(__nv_cvt_fp8_to_halfraw(u.code[j], __NV_E4M3))) * ratio;
      store_codes<V>(at, x, 1.f);
    }
  }
}

namespace {

template <typename T, int V>
cudaError_t codes_v(const PagedAppendArgs& a, cudaStream_t st, bool pdl) {
  CodeShape g{};
  g.units = (a.dim + 2 * V - 1) / (2 * V);
  g.q_per_cta = a.q_heads > 0 ? tokens_per_cta(a, a.q_heads, g.units) : 1;
  g.q_ctas = a.q_heads > 0 ? (a.tokens + g.q_per_cta - 1) / g.q_per_cta : 0;
  // heads for which a whole block's rows wait in registers; windows that leave every SM about eight CTAs
  const int block = a.block_size < a.tokens ? a.block_size : a.tokens;
  const int64_t per_head = 2ll * block * g.units, room = (int64_t)kRotNT * kCodeUnits / per_head;
  g.part_heads = room < 1 ? 1 : room > a.kv_heads ? a.kv_heads : (int)room;
  g.parts = (a.kv_heads + g.part_heads - 1) / g.part_heads;
  const int64_t want = (int64_t)a.tokens * g.parts / (8 * device_sm_count());
  g.window = want < 1 ? 1 : want > kCodeWindow ? kCodeWindow : (int)want;
  g.max_rows = g.window + a.block_size;
  if (a.angles.turns != nullptr) {
    const int most = 48 * 1024 / (a.angles.pairs * (int)sizeof(float2));
    g.turn_rows = g.max_rows < most ? g.max_rows : most;
    if (g.q_per_cta > g.turn_rows && g.q_ctas > 0) g.turn_rows = g.q_per_cta;
  }
  const size_t smem = (size_t)g.turn_rows * a.angles.pairs * sizeof(float2) + g.max_rows * sizeof(int) +
                      (g.max_rows + 1) / 2 * 2 * sizeof(short) + (size_t)g.window * 2 * g.part_heads * 3 * sizeof(float);
  const int64_t ctas = ((int64_t)a.tokens + g.window - 1) / g.window * g.parts + g.q_ctas;
  if (a.block_size > kAppendMaxBlock || ctas > INT_MAX || smem > 160 * 1024 ||
      (int64_t)g.max_rows * 2 * g.part_heads * g.units > INT_MAX)
    return cudaErrorInvalidValue;
  auto kern = paged_append_codes_kernel<T, V>;
  static SmemLimit limit;
  if (const cudaError_t e = limit.raise(kern, 160 * 1024); e != cudaSuccess) return e;
  return launch_kernel(kern, dim3((unsigned)ctas), dim3(kRotNT), smem, st, pdl, a, g);
}

template <typename T>
cudaError_t codes_t(const PagedAppendArgs& a, int vec, cudaStream_t st, bool pdl) {
  if (vec * sizeof(T) == 16) return codes_v<T, 16 / (int)sizeof(T)>(a, st, pdl);
  if (vec * sizeof(T) == 8) return codes_v<T, 8 / (int)sizeof(T)>(a, st, pdl);
  return codes_v<T, 1>(a, st, pdl);
}

}  // namespace

cudaError_t launch_paged_append_codes(const PagedAppendArgs& a, int dtype, int vec, cudaStream_t st, bool pdl) {
  switch (dtype) {
    case kBF16: return codes_t<__nv_bfloat16>(a, vec, st, pdl);
    case kF16: return codes_t<__half>(a, vec, st, pdl);
    case kF32: return codes_t<float>(a, vec, st, pdl);
  }
  return cudaErrorInvalidValue;
}

}  // namespace mlora
