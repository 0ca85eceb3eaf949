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
// with some of the heads of K or V: it has every row that a scale depends on, so nothing
// is agreed on between CTAs. A thread goes through every so many rows of one head with one unit of them (two
// vectors), once for the largest magnitude and again for the codes: the first two wait in registers, others come
// out of L2 again. A window's {cos, sin} are made once, for all of the CTA's heads.
//
// Measured over sets of inputs larger than L2, bf16 heads of 128, queries rotated beside: 512 tokens of 64 and 8 heads
// 7.6 us (20 MB, 2.6 TB/s), prompts of 4340 tokens, 32 and 8 heads, 32.3 us (98 MB, 3.0 TB/s): about 240 instructions a
// unit and turn bound it, as the latency of slots, rows and scales, one after the other, does with few rows. Calls that find the
// scales which they leave behind, as these do from the second on, round no older rows again. With the scales put back
// before every call (less 2 us for that; inputs partly in L2): 512 tokens whose scales do not grow 6.3 us, a third of them do
// 13.0, all 16.9; the prompts, whose blocks are new, 32.4. fp32 rows of the same prompts: 49.8.
#include <cuda_fp8.h>

#include <climits>

#include "device.h"
#include "kernels.h"
#include "paged.h"
#include "paged_append.cuh"

namespace mlora {

constexpr int kCodeWindow = 32;
// Rows of a thread that wait in registers between the two turns. (Four, and the three CTAs an SM that this leaves: prompts of
// 4340 tokens 40 us, 512 single tokens 11.2, where two and four CTAs take 32.8 and 9.4; one row, forth and back, 33.0 and 9.9.)
constexpr int kKept = 2;

// What the host decides about a launch.
struct CodeShape {
  int code_ctas, q_per_cta;       // CTAs of codes come first; tokens of each that rotates queries
  int units;                      // of a row
  int window, parts, part_items;  // an item: a head of K, or of V
  int step;                       // rows of an item at once
  int max_rows, turn_rows;        // rows that runs of a window can have; of those with {cos, sin} in shared memory
  int scale_at;                   // of shared memory
};

// The scale of rows whose largest magnitude is `most`: 448 = 1.75 * 2^8.
__device__ __forceinline__ float code_scale(float most) {
  const int k = (int)((__float_as_uint(most) + 0x1fffffu) >> 23) - 127 - 8;
  return most > 0.f ? __uint_as_float((uint32_t)(max(k, -100) + 127) << 23) : 0x1p-100f;
}

// V values over the scale, rounded to codes at dst; `inv`: its reciprocal where that is exact, otherwise 0.
template <int V>
__device__ __forceinline__ void store_codes(unsigned char* dst, float (&x)[V], float scale, float inv) {
  if (inv != 0.f) {
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] *= inv;
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] /= scale;
  }
  if constexpr (V == 1) {
    *dst = (unsigned char)__nv_cvt_float_to_fp8(x[0], __NV_SATFINITE, __NV_E4M3);
  } else {
    union {
      typename RawBytes<V>::type raw;
      unsigned short pair[V / 2];
    } u;
#pragma unroll
    for (int i = 0; i < V; i += 2)
      u.pair[i / 2] = __nv_cvt_float2_to_fp8x2(make_float2(x[i], x[i + 1]), __NV_SATFINITE, __NV_E4M3);
    *reinterpret_cast<typename RawBytes<V>::type*>(dst) = u.raw;
  }
}

template <typename T, int V>
__global__ void __launch_bounds__(kRotNT, 4) paged_append_codes_kernel(const PagedAppendArgs p, const CodeShape g) {
  extern __shared__ __align__(16) unsigned char s_dyn[];
  float2* s_turn = reinterpret_cast<float2*>(s_dyn);
  pdl_wait();
  pdl_trigger();
  if ((int)blockIdx.x >= g.code_ctas) {
    append_rows<T, V>(p, 0, blockIdx.x - g.code_ctas, g.q_per_cta, g.units, s_turn);
    return;
  }
  __shared__ int s_rows, s_runs, s_grown;
  __shared__ int s_first[kCodeWindow];  // row that a run begins with
  int2* s_place = reinterpret_cast<int2*>(s_turn + g.turn_rows * p.angles.pairs);  // [max_rows] block and slot; block -1: not of a run that begins here
  short* s_run = reinterpret_cast<short*>(s_place + g.max_rows);                   // [max_rows]
  uint32_t* s_most = reinterpret_cast<uint32_t*>(s_run + (g.max_rows + 1) / 2 * 2);  // [window][part_items]
  float2* s_scale = reinterpret_cast<float2*>(s_dyn + g.scale_at);                 // and its reciprocal, if that is exact
  const int tid = threadIdx.x, lane = tid & 31;
  const int part = blockIdx.x % g.parts, t0 = blockIdx.x / g.parts * g.window;
  const int item0 = part * g.part_items, items = min(g.part_items, 2 * p.kv_heads - item0);

  // ---- the runs that begin in the window ----
  if (tid < 32) {
    auto slot_at = [&](int t) { return t >= 0 && t < p.tokens ? __ldcg(p.slot_map + t) : -1; };
    const int t = t0 + lane, before = lane < g.window ? slot_at(t - 1) : -1;
    const int slot = lane < g.window ? slot_at(t) : -1;
    int block = slot >= 0 ? slot / p.block_size : -1;
    const int off = slot - block * p.block_size;
    bool begins = slot >= 0 && (before < 0 || before + 1 != slot || off == 0);
    if (block >= p.num_blocks) {
      if (part == 0) flag_error(p.status, kErrKvRange);
      block = -1;
      begins = false;
    }
    const unsigned mask = __ballot_sync(0xffffffffu, begins);
    const int run = __popc(mask & (0xffffffffu >> (31 - lane))) - 1;
    int rows = 0;
    if (mask != 0u) {
      if (lane < g.window) {
        s_place[lane] = make_int2(run >= 0 ? block : -1, off);
        s_run[lane] = (short)run;
      }
      if (begins) s_first[run] = lane;
      const int last = __shfl_sync(0xffffffffu, slot, g.window - 1), last_block = __shfl_sync(0xffffffffu, block, g.window - 1),
                last_off = __shfl_sync(0xffffffffu, off, g.window - 1), last_run = __shfl_sync(0xffffffffu, run, 31);
      rows = min(g.window, p.tokens - t0);
      // the last run behind the window's end: at most the rest of its block
      for (int most = last_block >= 0 ? p.block_size - 1 - last_off : 0; most > 0; most -= 32) {
        const int r = rows + lane, behind = 1 + r - g.window;
        const bool goes = lane < most && slot_at(t0 + r) == last + behind;
        const unsigned more = __ballot_sync(0xffffffffu, goes);
        const int n = more == 0xffffffffu ? 32 : __ffs(~more) - 1;
        if (lane < n) {
          s_place[r] = make_int2(last_block, last_off + behind);
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

  // the scales that the blocks have, on their way meanwhile
  auto scale_at = [&](int i, bool& begun) {
    const int run = i / items, item = item0 + i - run * items, side = item >= p.kv_heads, h = item - side * p.kv_heads;
    const int2 place = s_place[s_first[run]];
    begun = place.y > 0;
    return p.scale[side] + place.x * p.scale_block[side] + h * p.scale_head[side];
  };
  float held_scale = 0.f;
  if (tid < runs * items) {
    bool begun;
    const float* at = scale_at(tid, begun);
    if (begun) held_scale = __ldcg(at);
  }

  // A thread has one item, one unit of its rows, and every step-th row.
  const int lane_row = tid / (g.units * items), mine = lane_row < g.step ? tid - lane_row * g.units * items : -1;
  const int own = mine >= 0 ? mine / g.units : 0, u = mine - own * g.units;
  const int side = item0 + own >= p.kv_heads, h = item0 + own - side * p.kv_heads;
  const bool rotated = p.angles.turns != nullptr && item0 < p.kv_heads;
  const RotaryUnit un = rotary_unit(p.angles, side == 0 && rotated, p.dim, V, u);
  const PagedSide& s = p.side[side];
  const T* from = static_cast<const T*>(s.src) + t0 * s.src_token + h * s.src_head;
  unsigned char* to = static_cast<unsigned char*>(s.dst) + h * s.head;
  auto there = [&](int row) { return mine >= 0 && row < rows && s_place[row].x >= 0; };
  auto load = [&](int row, Vec<T, V> (&x)[2]) {
    const T* src = from + row * s.src_token;
    x[0].load(src + un.e0);
    if (un.both) x[1].load(src + un.e1);
  };
  auto values = [&](int row, const Vec<T, V> (&x)[2], float (&a)[V], float (&b)[V]) {
    x[0].to_f(a);
    x[1].to_f(b);
    if (!un.turned) return;
    float2 turn[V];
    if (row < g.turn_rows) {
      rotary_row<V>(p.angles, s_turn + row * p.angles.pairs, un.pair, turn);
    } else {
      const int position = __ldcg(p.angles.positions + t0 + row);
#pragma unroll
      for (int i = 0; i < V; ++i) turn[i] = rotary_turn(__ldg(p.angles.turns + un.pair + i), position, p.angles.factor);
    }
    rotary_apply<V>(p.angles.interleaved != 0, turn, a, b);
  };
  // The first rows stay in registers, those behind them come out of L2 again.
  Vec<T, V> x[kKept][2];
#pragma unroll
  for (int i = 0; i < kKept; ++i)
    if (there(lane_row + i * g.step)) load(lane_row + i * g.step, x[i]);
  if (rotated) rotary_table<V>(p.angles, t0, min(rows, g.turn_rows), s_turn);
  __syncthreads();
  // ---- the largest magnitudes, as whole numbers in the same order ----
  uint32_t most = 0u;
  int most_run = -1;
  auto count = [&](int row, const Vec<T, V> (&x)[2]) {
    float a[V], b[V];
    values(row, x, a, b);
    const int run = s_run[row];
    if (run != most_run) {
      if (most != 0u) atomicMax(s_most + most_run * items + own, most);
      most = 0u;
      most_run = run;
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const uint32_t ua = __float_as_uint(a[i]) & 0x7fffffffu, ub = __float_as_uint(b[i]) & 0x7fffffffu;
      if (ua < 0x7f800000u) most = max(most, ua);
      if (ub < 0x7f800000u && un.both) most = max(most, ub);
    }
  };
#pragma unroll
  for (int i = 0; i < kKept; ++i)
    if (there(lane_row + i * g.step)) count(lane_row + i * g.step, x[i]);
#pragma unroll 1
  for (int row = lane_row + kKept * g.step; row < rows; row += g.step) {
    if (!there(row)) continue;
    Vec<T, V> y[2];
    load(row, y);
    count(row, y);
  }
  if (most != 0u) atomicMax(s_most + most_run * items + own, most);
  __syncthreads();
  // ---- the scales ----
  for (int i = tid; i < runs * items; i += kRotNT) {
    bool begun;
    float* at = scale_at(i, begun);
    float scale = code_scale(__uint_as_float(s_most[i])), ratio = 1.f;
    if (begun) {
      const float old = i == tid ? held_scale : __ldcg(at);
      if (old < scale) ratio = old / scale;
      scale = fmaxf(scale, old);
    }
    *at = scale;
    s_scale[i] = make_float2(scale, (__float_as_uint(scale) & 0x7fffffu) == 0 ? 1.f / scale : 0.f);
    s_most[i] = __float_as_uint(ratio);
    if (ratio != 1.f) s_grown = 1;
  }
  __syncthreads();
  // ---- the codes ----
  auto put = [&](int row, const Vec<T, V> (&x)[2]) {
    float a[V], b[V];
    values(row, x, a, b);
    const int2 place = s_place[row];
    unsigned char* dst = to + place.x * s.block + place.y * s.slot;
    const float2 scale = s_scale[s_run[row] * items + own];
    store_codes<V>(dst + un.e0, a, scale.x, scale.y);
    if (un.both) store_codes<V>(dst + un.e1, b, scale.x, scale.y);
  };
#pragma unroll
  for (int i = 0; i < kKept; ++i)
    if (there(lane_row + i * g.step)) put(lane_row + i * g.step, x[i]);
#pragma unroll 1
  for (int row = lane_row + kKept * g.step; row < rows; row += g.step) {
    if (!there(row)) continue;
    Vec<T, V> y[2];
    load(row, y);
    put(row, y);
  }
  if (s_grown == 0) return;
  // ---- older rows of blocks whose scales have grown: a warp a block and head, four pieces a lane on their way ----
  const int pieces = p.dim / V;
  for (int i = tid >> 5; i < runs * items; i += kRotNT / 32) {
    const float ratio = __uint_as_float(s_most[i]);
    if (ratio == 1.f) continue;
    const int run = i / items, item = item0 + i - run * items, side = item >= p.kv_heads, h = item - side * p.kv_heads;
    const int2 place = s_place[s_first[run]];
    const PagedSide& s = p.side[side];
    unsigned char* base = static_cast<unsigned char*>(s.dst) + place.x * s.block + h * s.head;
    const int all = place.y * pieces;
    constexpr int AT_ONCE = 4;
    for (int e0 = lane; e0 < all; e0 += 32 * AT_ONCE) {
      union {
        typename RawBytes<V>::type raw;
        unsigned char code[V];
      } u[AT_ONCE];
      auto at = [&](int k) {
        const int e = e0 + 32 * k, row = e / pieces;
        return base + row * s.slot + (e - row * pieces) * V;
      };
#pragma unroll
      for (int k = 0; k < AT_ONCE; ++k)
        if (e0 + 32 * k < all) u[k].raw = *reinterpret_cast<const typename RawBytes<V>::type*>(at(k));
#pragma unroll
      for (int k = 0; k < AT_ONCE; ++k) {
        if (e0 + 32 * k >= all) continue;
        float x[V];
#pragma unroll
        for (int j = 0; j < V; ++j) x[j] = __half2float(__half(__nv_cvt_fp8_to_halfraw(u[k].code[j], __NV_E4M3))) * ratio;
        store_codes<V>(at(k), x, 1.f, 1.f);
      }
    }
  }
}

namespace {

template <typename T, int V>
cudaError_t codes_v(const PagedAppendArgs& a, cudaStream_t st, bool pdl) {
  CodeShape g{};
  g.units = (a.dim + 2 * V - 1) / (2 * V);
  g.q_per_cta = a.q_heads > 0 ? tokens_per_cta(a, g.units) : 1;
  const int q_ctas = a.q_heads > 0 ? (a.tokens + g.q_per_cta - 1) / g.q_per_cta : 0;
  // Items for which a whole block's rows are four units a thread, and windows of as many tokens (a window's
  // runs have as many rows as it has tokens, more or less), but no more than leave every SM two CTAs. (Prompts of 4340
  // tokens 32.3 us; three units a thread 37.9, six 36.3; four CTAs an SM for 512 single tokens 14.6 and not 9.3.)
  // Then, as long as its rows go through the threads in one turn, a window takes more tokens until all CTAs are at work
  // at once, those of the queries among them (512 single tokens 7.6 us, 9.3 without; 400 5.6 and 7.2, 256 5.6 and 6.5).
  const int block = a.block_size < a.tokens ? a.block_size : a.tokens, all_items = 2 * a.kv_heads;
  const int64_t full = 4 * kRotNT / g.units, room = full / block;
  g.part_items = room < 1 ? 1 : room > all_items ? all_items : (int)room;
  if (g.part_items > kRotNT / g.units) g.part_items = kRotNT / g.units;
  g.step = kRotNT / (g.units * g.part_items);
  g.parts = (all_items + g.part_items - 1) / g.part_items;
  const int64_t even = (int64_t)a.tokens * g.parts / (2 * device_sm_count()), rows = full / g.part_items;
  int64_t window = even < rows ? even : rows;
  if (window < 1) window = 1;
  while (window < g.step && window < rows && (a.tokens + window - 1) / window * g.parts + q_ctas > 4 * device_sm_count()) ++window;
  g.window = window > kCodeWindow ? kCodeWindow : (int)window;
  g.max_rows = g.window + a.block_size;
  if (a.angles.turns != nullptr) {
    const int most = 48 * 1024 / (a.angles.pairs * (int)sizeof(float2));
    g.turn_rows = g.max_rows < most ? g.max_rows : most;
    if (g.q_per_cta > g.turn_rows) g.turn_rows = g.q_per_cta;
  }
  const size_t most_at = (size_t)g.turn_rows * a.angles.pairs * sizeof(float2) + g.max_rows * sizeof(int2) +
                         (g.max_rows + 1) / 2 * 2 * sizeof(short);
  g.scale_at = (int)((most_at + (size_t)g.window * g.part_items * sizeof(uint32_t) + 7) / 8 * 8);
  const size_t smem = g.scale_at + (size_t)g.window * g.part_items * sizeof(float2);
  const int64_t code_ctas = ((int64_t)a.tokens + g.window - 1) / g.window * g.parts, ctas = code_ctas + q_ctas;
  g.code_ctas = (int)code_ctas;
  if (a.block_size > kAppendMaxBlock || ctas > INT_MAX || smem > 160 * 1024 ||
      (int64_t)g.max_rows * g.part_items * g.units > INT_MAX)
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
