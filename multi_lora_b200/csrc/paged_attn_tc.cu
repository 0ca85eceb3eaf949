// Attention over the paged cache for chunks of new tokens, on the fifth-
// generation tensor cores.
//
// The rows of a (request, key head) are its new tokens times the G query heads
// of the key head (row r: token r / G, head r % G), so that one pass over K and
// V serves the whole group. A CTA takes 256 of them, as two tiles of 128, over
// a run of 128-key tiles (the even split of paged_sched.cuh):
//   S = Q K^T   (tcgen05.mma, both operands from shared memory, S in TMEM)
//   P = exp2(scale' S - m)  by one warpgroup a tile of rows, a thread a row: a
//               row's 64 scores in registers, P written over S in TMEM
//   O += P V    (tcgen05.mma, P from TMEM, V from shared memory as it lies, with
//               the columns as the contiguous dimension; O in TMEM, 2 x 128 fp32 columns)
// A key tile is worked on in two halves of 64 keys, and each tile of rows has two
// buffers of 64 TMEM columns that hold a half's S and then its P (2 x 2 x 64 of
// them and 2 x D for O fill the 512). So the tensor cores are a half ahead: they
// compute S of the next half while the warpgroups work on this one, and neither
// waits for the other's latency.
//
// The running maximum that P is taken against is raised only when a row's
// scores exceed it by 2^8 (O is rescaled in TMEM then, rarely after the first
// tiles); P stays below 2^8 and everything is normalised at the end by the sum of P
// in fp32. f16 has few exponents: P and its sum are taken times 2^11 there and the
// maximum is raised from 2^4 on, so that P stays below 2^15 and what is subnormal lies
// below 2^-25 of the largest: tens of thousands of small ones would be lost together.
//
// P goes in as two terms, its upper 8 bits (f16: 11) and the rest (16 bits of it; 21):
// one term would add as much error as the result's own rounding. The second term is one
// more product of the same size. In f16, one term and two: 2048 tokens over 16384 keys
// 542 and 662 us, eight prompts 69 and 76, 1 to 6 drafts 98 and 109, the error 2.5e-4 and
// 2.1e-4 of the result's norm, the latter the rounding of the result alone.
//
// Head_dims below 64 and between 64 and 128 run as these, with columns of zeros that
// TMA fills in.
//
// What bounds it: the exponentials (16 a cycle and SM: 2048 cycles for two
// 128 x 128 tiles) and the tensor cores (4096 multiply-adds a cycle: 3072
// cycles with the second term, at D = 128), and over a
// long launch the power that these draw. Measured, bf16 and f16: 2048 tokens x 32 heads over 16384 keys in
// 720 us back to back (810 TFLOP/s; 640 before the power cap is reached, the tensor pipe 69 % busy at
// 1.6 GHz); 8 prompts of 128 to 1024 tokens 69 and 76 us: 4.3 items a CTA whose beginnings and ends
// (8000 cycles each) are a third of the work beside 14.5 tiles of 4300; 32 requests of 1 to 6 drafts
// over up to 8192 keys 105 and 109 us, 68 % of the measured copy bandwidth, where the second term keeps
// V's slots longer in a ring of 2.5 tiles; 512 tokens over 8192 keys with a window of 1000 33 us.
//
// Keys that a row does not see may hold anything: their scores are replaced, and
// since 0 * NaN is NaN their V is not multiplied by them. Rows of V that no row of
// the item sees are cleared in shared memory; infinities and NaN in those that some
// rows see are taken out there and added to these rows' outputs at the end. Both are done by
// the warp that fetches Q, while the softmax works. Where the products made NaN of an infinity that a
// row does see, its output is settled after it was stored (paged_settle).
#include <climits>

#include "device.h"
#include "kernels.h"
#include "paged_sched.cuh"
#include "paged_tma.h"
#include "tc.cuh"

namespace mlora {

constexpr int kChunkKeys = 128;   // keys a tile
constexpr int kHalfKeys = 64;     // keys a step of the tensor cores and the softmax
constexpr int kChunkRows = 256;   // query rows an item: two tiles of 128
constexpr int kChunkThreads = 384;
constexpr int kChunkJoin = 3;     // joining a piece costs about three key tiles
constexpr int kChunkItem = 2;     // an item costs about two besides its tiles (3 and 4: prompts 5 % slower)
using ChunkSplit = PagedSplit<kChunkJoin, kChunkItem>;

struct ChunkArgs {
  CUtensorMap k_map, v_map, q_map;
  PagedAttnArgs a;
  int box;
  int q_tma;   // Q tiles are boxes of q_map (group divides 128)
  int out32;   // rows of the output allow 32-byte stores
};

template <int D>
struct ChunkCfg {
  static constexpr int kSlot = kChunkKeys * D * 2;       // K or V of a tile
  static constexpr int kQ = 128 * D * 2;                 // one tile of Q
  static constexpr int kSlots = 160 * 1024 / kSlot;
  static constexpr int kSmem = 2 * kQ + kSlots * kSlot + 1024;
  static constexpr int kPart = 128 * (D + 2);            // floats of a tile's piece
};

struct ChunkItem {
  int req, head, rt, q0, qn, kv, rows;  // rows: of the whole request
  int first, end;                       // keys that some row of the item sees
  int tile0, n;
};

__device__ __forceinline__ void chunk_span(const PagedAttnArgs& p, ChunkItem& it) {
  const int r0 = it.rt * kChunkRows, r1 = min(it.rows, r0 + kChunkRows);
  const int base = it.kv - it.qn;
  it.first = paged_first_key(p, base + paged_token(p, r0));
  it.end = max(0, base + paged_token(p, r1 - 1) + 1);
  it.tile0 = it.first / kChunkKeys;
  it.n = max(1, (it.end + kChunkKeys - 1) / kChunkKeys - it.tile0);
}

// Keys [lo, hi) that every row of the item sees (none when lo >= hi).
__device__ __forceinline__ void chunk_seen(const PagedAttnArgs& p, const ChunkItem& it, int& lo, int& hi) {
  const int r0 = it.rt * kChunkRows, r1 = min(it.rows, r0 + kChunkRows);
  const int base = it.kv - it.qn;
  lo = paged_first_key(p, base + paged_token(p, r1 - 1));
  hi = max(0, base + paged_token(p, r0) + 1);
}

// One tile of rows only: the warps of both tiles work on it, each on every other half of the keys.
__device__ __forceinline__ bool chunk_solo(const ChunkItem& it) { return it.rows - it.rt * kChunkRows <= 128; }

__device__ __forceinline__ void chunk_request(const PagedAttnArgs& p, ChunkItem& it, int req, const PagedRequest& r) {
  it.req = req;
  it.q0 = r.q0;
  it.qn = r.qn;
  it.kv = r.kv;
  it.rows = r.qn * p.group;
}

// Whether the second half of the CTA's last tile of the item lies behind every row's keys.
template <typename Cursor>
__device__ __forceinline__ bool chunk_odd(const ChunkItem& it, const Cursor& cur) {
  return (it.tile0 + cur.tile + cur.len - 1) * kChunkKeys + kHalfKeys >= it.end;
}

__device__ __forceinline__ void tmem_ld32_async(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
// Ties registers of an asynchronous load to this point: nothing that uses them moves before it.
__device__ __forceinline__ void tie32(uint32_t (&r)[32]) {
  asm volatile(""
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                 "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]),
                 "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]),
                 "+r"(r[30]), "+r"(r[31]));
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
// Shared-memory descriptors by their halves: the upper one is a constant, the lower
// one an address in 16-byte units (plus the leading offset), so that stepping
// through a tile is one 32-bit addition and the tensor cores are not kept waiting
// for 64-bit address arithmetic.
constexpr uint32_t kDescHi = (1024u >> 4)       // 8 rows of 128 bytes to the next 8 (stride offset)
                             | (1u << 14)       // descriptor version of sm_100
                             | (2u << 29);      // 128-byte swizzle
// D[tmem] (+)= A[smem] * B[smem]^T, rows of 64 columns (128 bytes) in both.
__device__ __forceinline__ void umma_ss(uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\t"
      "mov.b64 a, {%1, %5};\n\tmov.b64 b, {%2, %5};\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_lo), "r"(b_lo), "r"(idesc), "r"((uint32_t)accumulate), "n"(kDescHi)
      : "memory");
}
// D[tmem] (+)= A[tmem] * B[smem]: A's row in its lane, two 16-bit elements a
// column; B as V lies: rows of 64 columns, the next 64 columns the leading offset on.
__device__ __forceinline__ void umma_ts(uint32_t d_tmem, uint32_t a_tmem, uint32_t b_lo, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\t"
      "mov.b64 b, {%2, %5};\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "r"(b_lo), "r"(idesc), "r"((uint32_t)accumulate), "n"(kDescHi)
      : "memory");
}

// One lane of the (converged) warp, always the same; unlike a comparison of the lane
// number it lets the compiler keep descriptors in uniform registers.
__device__ __forceinline__ bool elect_one() {
  uint32_t is;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(is));
  return is != 0;
}

// Two fp32 values in one register pair, and arithmetic on both at once.
__device__ __forceinline__ uint64_t pack2u(uint32_t lo, uint32_t hi) {
  uint64_t v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "r"(lo), "r"(hi));
  return v;
}
__device__ __forceinline__ uint64_t pack2(float lo, float hi) { return pack2u(__float_as_uint(lo), __float_as_uint(hi)); }
__device__ __forceinline__ float lo_of(uint64_t v) { return __uint_as_float((uint32_t)v); }
__device__ __forceinline__ float hi_of(uint64_t v) { return __uint_as_float((uint32_t)(v >> 32)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// What was taken out of V, added in TMEM to the outputs of row r, if it sees it: the
// item's keys of [from, to) that not every row sees, those of every
// tile's half `half` if that is not negative. Seldom run, so kept out of the kernel's registers.
template <typename T, int D>
__device__ __noinline__ void chunk_give_back(const PagedAttnArgs& p, uint32_t o_addr, int req, int head, int rt, int qn, int kv,
                                             int r, int from, int to, int half) {
  ChunkItem it;
  it.qn = qn;
  it.kv = kv;
  it.rt = rt;
  it.rows = qn * p.group;
  int seen_lo, seen_hi;
  chunk_seen(p, it, seen_lo, seen_hi);
  const int pos = kv - qn + paged_token(p, r);
  if (r < it.rows) {
    from = max(from, paged_first_key(p, pos));
    to = min(to, pos + 1);
  } else {
    to = from;
  }
#pragma unroll 1
  for (int c = 0; c < D / 32; ++c) {
    uint32_t o[32];
    tmem_ld32_async(o_addr + c * 32, o);
    tmem_wait_ld();
    tie32(o);
#pragma unroll 1
    for (int j = from; j < to; ++j) {
      if ((j >= seen_lo && j < seen_hi) || (half >= 0 && ((j / kHalfKeys) & 1) != half)) continue;
      const int block = __ldcg(p.tables + req * p.table_stride + j / p.block_size);
      if (block < 0 || block >= p.num_blocks) continue;
      const uint32_t* src = reinterpret_cast<const uint32_t*>(static_cast<const T*>(p.v) + block * p.v_block +
                                                              (j % p.block_size) * p.v_slot + head * p.v_head + c * 32);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const uint32_t w = c * 32 + 2 * i < p.dim ? __ldcg(src + i) : 0u;
        const float a = Pack2<T>::lo(w), b = Pack2<T>::hi(w);
        if (!isfinite(a)) o[2 * i] = __float_as_uint(__uint_as_float(o[2 * i]) + a);
        if (!isfinite(b)) o[2 * i + 1] = __float_as_uint(__uint_as_float(o[2 * i + 1]) + b);
      }
    }
    __syncwarp();
    tmem_st32(o_addr + c * 32, o);
  }
  tmem_wait_st();
}

// What the lanes of a softmax warp wrote of an item: one, two or four threads a row (`share`), 32 columns in turn.
struct ChunkPlace {
  PagedPlace item;
  int q0, row0, share;
};
// The outputs of the marked lanes, settled; the marks are taken back.
template <typename T>
__device__ __noinline__ void chunk_settle(const PagedAttnArgs& p, const ChunkPlace* at, uint32_t* marks) {
  const int thread = threadIdx.x & 127, per = 128 / at->share, row = at->row0 + (thread & (per - 1));
  const bool mine = (*marks >> (thread & 31) & 1u) != 0u;
  const int t = paged_token(p, row);
  T* dst = static_cast<T*>(p.out) + (int64_t)(at->q0 + t) * p.out_token +
           (int64_t)(at->item.head * p.group + row - t * p.group) * p.out_head;
#pragma unroll 1
  for (int c0 = thread / per * 32; c0 < p.dim; c0 += at->share * 32)
#pragma unroll 1
    for (int c = c0; c < min(c0 + 32, p.dim); c += 8) paged_settle<T, 4>(p, &at->item, row, c, dst + c, mine);
  __syncwarp();
  if ((thread & 31) == 0) *marks = 0u;
  __syncwarp();
}

template <int N>
__device__ __forceinline__ void regs_down() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void regs_up() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}

template <typename T, int D>
__global__ void __launch_bounds__(kChunkThreads, 1)
paged_attention_chunk_kernel(const __grid_constant__ ChunkArgs args) {
  using C = ChunkCfg<D>;
  constexpr int NS = C::kSlots, HALF = kChunkKeys * 128;
  constexpr uint32_t kKeep = Num<T>::is_bf16 ? 0xffff0000u : 0xffffe000u;  // bits of fp32 that the type holds
  constexpr float kRaise = Num<T>::is_bf16 ? 8.f : 4.f, kUp = Num<T>::is_bf16 ? 0.f : 11.f;  // in powers of two
  constexpr uint32_t S_COL = 0, O_COL = 256;
  extern __shared__ __align__(1024) unsigned char s_raw[];
  __shared__ __align__(8) uint64_t full[NS], empty[NS], q_ready[2], q_free[2], s_full[2][2], p_ready[2][2], pv_done[2][2];
  __shared__ uint32_t s_tmem;
  __shared__ int s_last[2];
  __shared__ bool s_skipped;
  __shared__ float2 s_mate[128];
  __shared__ uint32_t s_odd[8];    // lanes of a softmax warp that stored what is not finite though the row's sum is
  __shared__ ChunkPlace s_place[8];  // of the item whose output each softmax warp writes
  __shared__ uint32_t s_clean;  // V tiles that have been cleaned
  __shared__ uint32_t s_taken;           // a value that is not finite was taken out of one of them
  const PagedAttnArgs& p = args.a;
  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = same_in_warp(tid >> 5);
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(s_raw) + 1023) & ~uintptr_t(1023));
  unsigned char* ring = smem + 2 * C::kQ;

  if (tid == 0) {
    for (int s = 0; s < NS; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 3);  // both warps of the tensor cores, and the one that cleans V
    }
    for (int q = 0; q < 2; ++q) {
      mbar_init(&q_ready[q], 1);
      mbar_init(&q_free[q], 2);
      for (int b = 0; b < 2; ++b) {
        mbar_init(&s_full[q][b], 1);
        mbar_init(&p_ready[q][b], 4);
        mbar_init(&pv_done[q][b], 1);
      }
    }
    fence_barrier_init();
    s_clean = s_taken = 0u;
    for (int w = 0; w < 8; ++w) s_odd[w] = 0u;
    tma_prefetch_map(&args.k_map);
    tma_prefetch_map(&args.v_map);
    if (args.q_tma) tma_prefetch_map(&args.q_map);
  }
  if (warp == 1) tmem_alloc(&s_tmem, 512);
  tc_fence_before();
  pdl_wait();
  pdl_trigger();

  ChunkSplit split;
  ChunkItem it;
  int before, in_req;
  int req;
  PagedRequest found;
  bool skipped = false;  // a request that is not computed
  paged_find<kChunkThreads, 32>(
      p.requests,
      [&](int i, int part, int parts, PagedRequest& r) {
        r = paged_request(p, i, part == 0 && blockIdx.x == 0);
        skipped |= r.odd;
        ChunkItem x;
        chunk_request(p, x, i, r);
        int n = 0;
        for (x.rt = part; x.rt * kChunkRows < x.rows; x.rt += parts) {
          chunk_span(p, x);
          n += x.n + kChunkItem;
        }
        return n * p.kv_heads;
      },
      split, req, found, before, in_req);
  skipped = __syncthreads_or(skipped);  // and the barriers are initialised, and s_tmem is there
  if (tid == 96) s_skipped = skipped;   // for its own warp, at the end: no register holds it until then
  tc_fence_after();
  const uint32_t tmem = s_tmem;
  PagedCursor<ChunkSplit> cur(split);
  auto item_of_request = [&](int rel) {  // the item that holds unit `rel` of request it.req: a lane a tile of rows
    const int per_head = in_req / p.kv_heads;
    it.head = rel / per_head;
    rel -= it.head * per_head;
    it.rt = 0;
    for (int rt0 = 0; rt0 * kChunkRows < it.rows; rt0 += 32) {
      ChunkItem x = it;
      x.rt = rt0 + lane;
      int units = 0;
      if (x.rt * kChunkRows < x.rows) {
        chunk_span(p, x);
        units = x.n + kChunkItem;
      }
      int upto = units;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += u;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, rel < upto);
      if (hit != 0u) {
        const int src = __ffs(hit) - 1;
        it.rt = rt0 + src;
        cur.unit = rel - __shfl_sync(0xffffffffu, upto - units, src);
        break;
      }
      rel -= __shfl_sync(0xffffffffu, upto, 31);
    }
    chunk_span(p, it);
  };
  auto next_item = [&]() {
    if (++it.rt * kChunkRows >= it.rows) {
      it.rt = 0;
      if (++it.head == p.kv_heads) {
        it.head = 0;
        PagedRequest r;
        const int i = paged_next(p, it.req, INT_MAX, r);
        if (i < p.requests) {
          r.q0 = same_in_warp(r.q0);
          r.qn = same_in_warp(r.qn);
          r.kv = same_in_warp(r.kv);
          chunk_request(p, it, i, r);
        }
      }
    }
    chunk_span(p, it);
  };
  if (cur.pos < cur.end) {
    chunk_request(p, it, req, found);
    item_of_request(cur.pos - before);
    if (cur.begin(it.n)) next_item();
  }
  bool ok = true;

  // Registers: 384 threads are launched with 168 each (64512); the four warps of
  // the producer and the tensor cores keep 72, the softmax warps take 216: 128 * 72
  // + 256 * 216 = 64512.
  if (warp < 4) {
    regs_down<72>();
    if (warp == 0) {  // ---- producer: K and V of each tile, a box of a page a lane ----
      const int boxes = kChunkKeys / args.box, jobs = boxes * (D / 64);
      const int b = lane % boxes, half = lane / boxes;
      int slot = 0, round = 0;
      while (cur.take(it.n)) {
        const int32_t* table = p.tables + it.req * p.table_stride;
        for (int k = 0; k < cur.len; ++k) {
          const int j = (it.tile0 + cur.tile + k) * kChunkKeys + b * args.box;
          int block = (int)p.num_blocks, off = 0;  // out of range: zeros
          if (lane < jobs && j < it.end && j + args.box > it.first) {
            const int e = __ldcg(table + j / p.block_size);
            off = j % p.block_size;
            if (e >= 0 && e < p.num_blocks) block = e;
            else flag_error(p.status, kErrKvRange);
          }
#pragma unroll
          for (int side = 0; side < 2; ++side) {
            if (round > 0) ok = __all_sync(0xffffffffu, ok && mbar_poll(&empty[slot], (round - 1) & 1, p.status));
            if (ok) {
              if (lane == 0) mbar_arrive_expect_tx(&full[slot], C::kSlot);
              __syncwarp();
              if (lane < jobs)
                tma_load_4d(ring + slot * C::kSlot + half * HALF + b * args.box * 128,
                            side == 0 ? &args.k_map : &args.v_map, half * 64, off, it.head, block, &full[slot]);
            }
            if (++slot == NS) {
              slot = 0;
              ++round;
            }
          }
        }
        if (cur.advance()) next_item();
      }
    } else if (warp < 3) {  // ---- tensor cores, a warp a tile of rows: S of a half, then O of the half before ----
      // A wait costs its warp over 100 cycles even when it need not wait, and the tensor
      // cores hold no more than two instructions: with one issuing warp they
      // idled for half the time. While one of these two waits the other one issues.
      const int q = warp - 1;
      constexpr uint32_t idesc_s = umma_idesc_f16(Num<T>::is_bf16, 128, kHalfKeys);
      constexpr uint32_t idesc_o = umma_idesc_f16(Num<T>::is_bf16, 128, D) | (1u << 16);  // B: columns contiguous
      constexpr uint32_t kStep = kHalfKeys * 128 >> 4;  // a half of a K or V tile
      const uint32_t ring_lo = smem_addr(ring) >> 4;
      const uint32_t s_col = tmem + S_COL + q * 128, o_col = tmem + O_COL + q * D;
      int kslot = 0, k_phase = 0, vslot = 1, v_phase = 0;
      int n = 0;                 // halves begun
      int items = 0, pairs = 0;  // items, and those of two tiles of rows
      auto wait = [&](uint64_t* bar, int parity) { ok = ok && mbar_poll(bar, parity & 1, p.status); };
      bool held = false, held_first = false, held_last = false;  // the half whose product with V is to come
      uint32_t held_lo = 0;
      int held_slot = 0;
      uint32_t dirty = 0, held_dirty = 0;  // V tiles to be cleaned so far; those that the held half waits for
      auto values = [&]() {  // half n - 1 of this tile of rows is the newest, half `number` the held one
        const int number = n - 1, b = number & 1;
        if (held_dirty != 0u) ok = ok && count_poll(&s_clean, held_dirty, p.status);
        wait(&p_ready[q][b], number >> 1);
        tc_fence_after();
        if (elect_one()) {
          const uint32_t a = s_col + b * 64;
#pragma unroll
          for (int i = 0; i < kHalfKeys / 16; ++i) umma_ts(o_col, a + i * 8, held_lo + i * 128, idesc_o, !held_first || i > 0);
#pragma unroll
          for (int i = 0; i < kHalfKeys / 16; ++i) umma_ts(o_col, a + 32 + i * 8, held_lo + i * 128, idesc_o, true);
          umma_commit(&pv_done[q][b]);
          if (held_last) umma_commit(&empty[held_slot]);
        }
        held = false;
      };
      while (cur.take(it.n)) {
        const bool solo = chunk_solo(it);  // this warp then has every other half of the one tile
        const int qs = solo ? 0 : q, h0 = solo ? q : 0;
        const bool odd = !solo && chunk_odd(it, cur);
        const uint32_t q_lo = smem_addr(smem + qs * C::kQ) >> 4;
        int seen_lo, seen_hi;
        chunk_seen(p, it, seen_lo, seen_hi);
        bool tile_dirty = false;
        if (held) values();  // nothing of the item before waits for this one's Q, or keeps its V from the ring
#pragma unroll 1
        for (int k = 0; k < cur.len; ++k) {
          wait(&full[kslot], k_phase);
          const int h1 = solo ? q + 1 : odd && k == cur.len - 1 ? 1 : 2;
#pragma unroll 1
          for (int h = h0; h < h1; ++h) {
            const bool first = k == 0 && h == h0, last = h == h1 - 1;
            if (first) wait(&q_ready[qs], qs == 0 ? items : pairs);
            const int b = n & 1;
            if (n > 1) wait(&pv_done[q][b], (n >> 1) - 1);  // P in this buffer has been read
            tc_fence_after();
            if (elect_one()) {
              const uint32_t kl = ring_lo + kslot * (C::kSlot >> 4) + h * kStep;
#pragma unroll
              for (int i = 0; i < D / 16; ++i)
                umma_ss(s_col + b * 64, q_lo + (i >> 2) * (HALF >> 4) + 2 * (i & 3), kl + (i >> 2) * (HALF >> 4) + 2 * (i & 3),
                        idesc_s, i > 0);
              umma_commit(&s_full[q][b]);
              if (last) umma_commit(&empty[kslot]);
              if (last && k == cur.len - 1) {  // two arrivals free a tile of Q
                umma_commit(&q_free[qs]);
                if (!solo) umma_commit(&q_free[qs]);
              }
            }
            if (held) values();
            ++n;
            if (h == h0) {
              wait(&full[vslot], v_phase);
              const int j0 = (it.tile0 + cur.tile + k) * kChunkKeys;
              tile_dirty = j0 + kChunkKeys > seen_hi || j0 < seen_lo;
              if (tile_dirty) ++dirty;
            }
            held_dirty = tile_dirty ? dirty : 0u;
            held = true;
            held_first = first;
            held_last = last;
            held_lo = ring_lo + vslot * (C::kSlot >> 4) + h * kStep + ((HALF >> 4) << 16);
            held_slot = vslot;
          }
          kslot += 2;
          if (kslot >= NS) {
            kslot -= NS;
            k_phase ^= 1;
          }
          vslot += 2;
          if (vslot >= NS) {
            vslot -= NS;
            v_phase ^= 1;
          }
        }
        ++items;
        pairs += solo ? 0 : 1;
        if (cur.advance()) next_item();
      }
      if (held) values();
    } else {  // ---- Q of each item, as soon as the scores of the item before are done; V's tiles cleaned ----
      int items[2] = {0, 0};
      int slot = 0, phase = 0;
      uint32_t dirty = 0;
      while (cur.take(it.n)) {
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const int r0 = it.rt * kChunkRows + q * 128;
          if (r0 >= it.rows) continue;
          if (items[q] > 0) ok = __all_sync(0xffffffffu, ok && mbar_poll(&q_free[q], (items[q] - 1) & 1, p.status));
          ++items[q];
          if (args.q_tma) {  // rows behind the request's are others', or zeros: no score of theirs is used
            if (ok && lane == 0) {
              mbar_arrive_expect_tx(&q_ready[q], C::kQ);
              for (int c = 0; c < D / 64; ++c)
                tma_load_3d(smem + q * C::kQ + c * HALF, &args.q_map, c * 64, it.head * p.group, it.q0 + paged_token(p, r0),
                            &q_ready[q]);
            }
            __syncwarp();
          } else {
            constexpr int PIECES = D / 8, AT_ONCE = 8;  // 16-byte pieces, swizzled as TMA would
#pragma unroll 1
            for (int e0 = lane; e0 < 128 * PIECES; e0 += 32 * AT_ONCE) {
              uint4 u[AT_ONCE];
#pragma unroll
              for (int i = 0; i < AT_ONCE; ++i) {
                const int e = e0 + i * 32, r = r0 + e / PIECES, c = e % PIECES, t = paged_token(p, r);
                u[i] = make_uint4(0, 0, 0, 0);
                if (r < it.rows && c * 8 < p.dim)
                  u[i] = __ldcg(reinterpret_cast<const uint4*>(static_cast<const T*>(p.q) + (int64_t)(it.q0 + t) * p.q_token +
                                                               (int64_t)(it.head * p.group + r - t * p.group) * p.q_head + c * 8));
              }
#pragma unroll
              for (int i = 0; i < AT_ONCE; ++i) {
                const int e = e0 + i * 32, r = e / PIECES, c = e % PIECES;
                *reinterpret_cast<uint4*>(smem + q * C::kQ + (c >> 3) * HALF + r * 128 + (((c & 7) ^ (r & 7)) << 4)) = u[i];
              }
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&q_ready[q]);
          }
        }
        int seen_lo, seen_hi;
        chunk_seen(p, it, seen_lo, seen_hi);
        for (int k = 0; k < 2 * cur.len; ++k) {  // K, V, K, V: every slot is let go by this warp too, so it never misses a phase
          const int j0 = (it.tile0 + cur.tile + (k >> 1)) * kChunkKeys;
          ok = __all_sync(0xffffffffu, ok && mbar_poll(&full[slot], phase, p.status));
          if ((k & 1) != 0 && (j0 + kChunkKeys > seen_hi || j0 < seen_lo)) {
            ++dirty;
            unsigned char* vs = ring + slot * C::kSlot;
            // whole boxes without a key are zeros already: clear what shares a box with one
            const int lo = min(kChunkKeys, max(0, it.first - j0)), lo0 = lo / args.box * args.box;
            const int hi = min(kChunkKeys, max(0, it.end - j0)), hi1 = min(kChunkKeys, (hi + args.box - 1) / args.box * args.box);
            if (ok) {
#pragma unroll 1
              for (int e = lane; e < (lo - lo0 + hi1 - hi) * (D / 8); e += 32) {
                const int i = e / (D / 8), c = e % (D / 8), j = i < lo - lo0 ? lo0 + i : hi + i - (lo - lo0);
                *reinterpret_cast<uint4*>(vs + (c >> 3) * HALF + j * 128 + (c & 7) * 16) = make_uint4(0, 0, 0, 0);
              }
              // keys that only some rows see: [lo, some) by the window, [rest, hi) by the causal mask
              const int some = max(lo, min(hi, seen_lo - j0)), rest = max(some, min(hi, seen_hi - j0));
              uint32_t taken = 0u;
              constexpr int PER = D / 8, STEP = 32 / PER, AT_ONCE = 8;  // 16-byte pieces a row, rows at once, and in flight
              const int c = lane % PER;
              unsigned char* col = vs + (c >> 3) * HALF + (c & 7) * 16;
#pragma unroll 1
              for (int part = 0; part < 2; ++part) {
                const int end = part == 0 ? some : hi;
#pragma unroll 1
                for (int j = (part == 0 ? lo : rest) + lane / PER; j < end; j += STEP * AT_ONCE) {
                  uint32_t seen = 0u;
#pragma unroll
                  for (int i = 0; i < AT_ONCE; ++i) {  // a row twice rather than one behind the end
                    const uint4 u = *reinterpret_cast<const uint4*>(col + min(j + i * STEP, end - 1) * 128);
                    seen = paged_taint<T>(u.w, paged_taint<T>(u.z, paged_taint<T>(u.y, paged_taint<T>(u.x, seen))));
                  }
                  if (seen == 0u) continue;
                  taken = 1u;
#pragma unroll 1
                  for (int i = j; i < min(end, j + STEP * AT_ONCE); i += STEP) {
                    uint4* at = reinterpret_cast<uint4*>(col + i * 128);
                    *at = make_uint4(paged_finite<T>(at->x), paged_finite<T>(at->y), paged_finite<T>(at->z), paged_finite<T>(at->w));
                  }
                }
              }
              if (taken != 0u) count_store(&s_taken, 1u);
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) count_store(&s_clean, dirty);
          }
          if (lane == 0) mbar_arrive(&empty[slot]);
          if (++slot == NS) {
            slot = 0;
            phase ^= 1;
          }
        }
        if (cur.advance()) next_item();
      }
      __syncwarp();
      if (s_skipped) paged_zero_uncomputed<T>(p, split.total > 0 ? INT_MAX : -1);
      else paged_zero_rest<T>(p);
    }
  } else {  // ---- softmax: warpgroup q, thread = row ----
    regs_up<216>();
    const int q = (warp >> 2) - 1, row = tid & 127;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_addr = tmem + lanes + S_COL + q * 128, o_addr = tmem + lanes + O_COL + q * D;
    const float sl = p.scale * 1.4426950408889634f;  // scores in powers of two
    uint32_t* tickets = static_cast<uint32_t*>(p.workspace);
    float* parts = reinterpret_cast<float*>(tickets + kPagedTickets);
    int n = 0;             // halves done
    bool lent = false;     // the other warpgroup still reads this one's O
    while (cur.take(it.n)) {
      const bool solo = chunk_solo(it);  // the warpgroups share its keys, half by half
      const int r_lo = it.rt * kChunkRows + (solo ? 0 : q * 128), r = r_lo + row;
      const int pq = it.kv - it.qn + paged_token(p, r);
      const int limit = r < it.rows ? pq + 1 : 0, floor_ = paged_first_key(p, pq);
      // key tiles that every row of this tile sees whole need no mask
      const int r_hi = min(it.rows, r_lo + 128) - 1;
      const int all_end = it.kv - it.qn + paged_token(p, r_lo) + 1,
                all_first = paged_first_key(p, it.kv - it.qn + paged_token(p, r_hi));
      const bool none = r - lane >= it.rows;  // no row in this warp: its lanes of P and O are never looked at
      float m = -INFINITY, l = 0.f;
      const int halves = solo ? cur.len : 2 * cur.len - chunk_odd(it, cur);
      for (int k = 0; k < halves; ++k, ++n) {
        const int b = n & 1;
        ok = ok && mbar_poll(&s_full[q][b], (n >> 1) & 1, p.status);
        __syncwarp();
        tc_fence_after();
        if (none) {
          if (lent) {
            named_barrier(5, 256);
            lent = false;
          }
          if (lane == 0) mbar_arrive(&p_ready[q][b]);
          continue;
        }
        uint32_t s[2][32];
        tmem_ld32_async(s_addr + b * 64, s[0]);
        tmem_ld32_async(s_addr + b * 64 + 32, s[1]);
        tmem_wait_ld();
        tie32(s[0]);
        tie32(s[1]);
        const int j0 = (it.tile0 + cur.tile) * kChunkKeys + (solo ? 2 * k + q : k) * kHalfKeys;
        if (j0 + kHalfKeys > all_end || j0 < all_first) {
          const int hi = limit - j0, lo = floor_ - j0;
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (c * 32 + i >= hi || c * 32 + i < lo) s[c][i] = 0xff800000u;  // -infinity
        }
        float top[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const uint32_t* x = &s[c >> 1][(c & 1) * 16];
          top[c] = __uint_as_float(x[0]);
#pragma unroll
          for (int i = 1; i < 15; i += 2) top[c] = max3(top[c], __uint_as_float(x[i]), __uint_as_float(x[i + 1]));
          top[c] = fmaxf(top[c], __uint_as_float(x[15]));
        }
        const float mx = fmaxf(max3(top[0], top[1], top[2]), top[3]) * sl;
        if (k == 0) {
          m = mx;
        } else {
          const bool raise = mx > m + kRaise;
          if (__any_sync(0xffffffffu, raise)) {
            // O holds the halves before this one once the last product is done
            ok = ok && mbar_poll(&pv_done[q][b ^ 1], ((n - 1) >> 1) & 1, p.status);
            __syncwarp();
            tc_fence_after();
            const float fix = raise ? exp2_fast(m - mx) : 1.f;
            if (raise) m = mx;
            l *= fix;
#pragma unroll 1
            for (int c = 0; c < D / 32; ++c) {
              uint32_t o[32];
              tmem_ld32_async(o_addr + c * 32, o);
              tmem_wait_ld();
              tie32(o);
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * fix);
              tmem_st32(o_addr + c * 32, o);
            }
          }
        }
        const float ref = (m == -INFINITY ? 0.f : m) - kUp;
        const uint64_t sl2 = pack2(sl, sl), ref2 = pack2(-ref, -ref);
        uint64_t sum[4] = {0, 0, 0, 0};
        uint32_t w[32], rest[32];  // P, two keys a column
#pragma unroll
        for (int i = 0; i < 64; i += 2) {
          const uint64_t x = fma2(pack2u(s[i >> 5][i & 31], s[i >> 5][(i & 31) + 1]), sl2, ref2);
          const float p0 = exp2_fast(lo_of(x)), p1 = exp2_fast(hi_of(x));
          const uint64_t pp = pack2(p0, p1);
          sum[(i >> 1) & 3] = add2(sum[(i >> 1) & 3], pp);
          // the upper bits as they are (in f16 rounded where they are subnormal), and what is left rounded
          const uint32_t u0 = __float_as_uint(p0) & kKeep, u1 = __float_as_uint(p1) & kKeep;
          if constexpr (Num<T>::is_bf16) w[i >> 1] = __byte_perm(u0, u1, 0x7632);
          else w[i >> 1] = pack_round2<T>(__uint_as_float(u0), __uint_as_float(u1));
          const uint64_t left = fma2(pack2u(u0, u1), pack2(-1.f, -1.f), pp);
          rest[i >> 1] = pack_round2<T>(lo_of(left), hi_of(left));
        }
        const uint64_t both = add2(add2(sum[0], sum[1]), add2(sum[2], sum[3]));
        l += lo_of(both) + hi_of(both);
        tmem_st32(s_addr + b * 64, w);
        tmem_st32(s_addr + b * 64 + 32, rest);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lent) {  // this half's product overwrites O
          named_barrier(5, 256);
          lent = false;
        }
        if (lane == 0) mbar_arrive(&p_ready[q][b]);
      }

      const ChunkItem done = it;
      const bool whole = cur.whole(it.n);
      const int item0 = cur.pos - cur.unit;
      const int tile0 = it.tile0 + cur.tile, tiles = cur.len;
      if (lane == 0) s_place[warp - 4] = {{done.req, done.head, done.kv, done.qn}, done.q0, r_lo, 1};
      if (cur.advance()) next_item();

      ok = ok && mbar_poll(&pv_done[q][(n - 1) & 1], ((n - 1) >> 1) & 1, p.status);
      __syncwarp();
      tc_fence_after();
      if (__any_sync(0xffffffffu, *const_cast<volatile uint32_t*>(&s_taken) != 0u)) {
        chunk_give_back<T, D>(p, o_addr, done.req, done.head, done.rt, done.qn, done.kv, r, tile0 * kChunkKeys,
                              (tile0 + tiles) * kChunkKeys, solo ? q : -1);
      }
      // An item that both warpgroups worked on: the first one reads the other's O too
      // (their threads of a row have the same TMEM lane).
      float own = 1.f, others = 0.f;  // what the two warpgroups' sums are multiplied by
      if (solo) {
        if (q == 1) {
          s_mate[row] = make_float2(m, l);
          tc_fence_before();
          named_arrive(4, 256);
          lent = true;
          continue;
        }
        named_barrier(4, 256);
        tc_fence_after();
        const float2 mate = s_mate[row];
        const float top = fmaxf(m, mate.x), base = top == -INFINITY ? 0.f : top;
        own = exp2_fast(m - base);
        others = exp2_fast(mate.x - base);
        l = l * own + mate.y * others;
        m = top;
      }
      const int t = paged_token(p, r);
      T* dst = static_cast<T*>(p.out) + (int64_t)(done.q0 + t) * p.out_token +
               (int64_t)(done.head * p.group + r - t * p.group) * p.out_head;
      auto store = [&](T* dst, int c, const float* v, float inv) {  // 16 columns: a thread a row, so whole sectors
        uint32_t u[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) u[i] = pack_round2<T>(v[2 * i] * inv, v[2 * i + 1] * inv);
        uint32_t odd = 0u;
#pragma unroll
        for (int i = 0; i < 8; ++i) odd = paged_taint<T>(u[i], odd);
        if (odd != 0u && inv == inv) atomicOr(&s_odd[warp - 4], 1u << lane);
        if (args.out32) {
          if (c < p.dim) store32(dst + c, u);
        } else {
          if (c < p.dim) *reinterpret_cast<uint4*>(dst + c) = make_uint4(u[0], u[1], u[2], u[3]);
          if (c + 8 < p.dim) *reinterpret_cast<uint4*>(dst + c + 8) = make_uint4(u[4], u[5], u[6], u[7]);
        }
      };
      // pieces: [column / 4][row] of four floats, then maxima, then sums
      auto piece = [&](int cta, int first_cta) {
        return parts + (((long long)cta * 2 + (cta == first_cta ? 1 : 0)) * 2 + q) * C::kPart;
      };
      const int c0 = whole ? 0 : split.first_cta(item0, done.n);
      float* part = piece(blockIdx.x, c0);
      const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
#pragma unroll 1
      for (int c = 0; c < (none ? 0 : D / 32); ++c) {
        uint32_t o[32];
        tmem_ld32_async(o_addr + c * 32, o);
        tmem_wait_ld();
        tie32(o);
        float v[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(o[i]);
        if (solo) {
          tmem_ld32_async(o_addr + D + c * 32, o);
          tmem_wait_ld();
          tie32(o);
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = fmaf(__uint_as_float(o[i]), others, v[i] * own);
        }
        if (whole) {
          if (r < done.rows) {
#pragma unroll
            for (int i = 0; i < 32; i += 16) store(dst, c * 32 + i, v + i, inv);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 32; i += 4)
            __stcg(reinterpret_cast<float4*>(part) + (c * 8 + i / 4) * 128 + row,
                   make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]));
        }
      }
      tc_fence_before();
      if (solo) named_arrive(5, 256);
      if (!whole) {
        __stcg(part + 128 * D + row, m);
        __stcg(part + 128 * (D + 1) + row, l);
        const int c1 = split.last_cta(item0, done.n);
        const PagedJoin run(c0, c1, blockIdx.x);
        auto last_of = [&](uint32_t* ticket, int n) {  // whether this warpgroup is the last of n to get here
          named_barrier(1 + q, 128);
          if (row == 0) {
            __threadfence();
            const bool last = atomicAdd(ticket, 1u) == (uint32_t)(n - 1);
            if (last) *ticket = 0u;
            __threadfence();
            s_last[q] = last;
          }
          named_barrier(1 + q, 128);
          const bool last = s_last[q];
          named_barrier(1 + q, 128);
          return last;
        };
        // Pieces x0, x0 + by, .. x1 of this tile of rows, to the output or as one piece to x0's
        // place; one, two or four threads a row, 32 columns of four pieces at once.
        auto join = [&](int x0, int x1, int by, bool final) {
          const int live = min(128, done.rows - r_lo), share = live <= 32 ? 4 : live <= 64 ? 2 : 1;
          const int jr = row & (128 / share - 1), c_from = row / (128 / share) * 32;
          float top = -INFINITY, total = 0.f;
          if (jr < live) {
#pragma unroll 4
            for (int x = x0; x <= x1; x += by) top = fmaxf(top, __ldcg(piece(x, c0) + 128 * D + jr));
            const float base = top == -INFINITY ? 0.f : top;
#pragma unroll 4
            for (int x = x0; x <= x1; x += by)
              total = fmaf(__ldcg(piece(x, c0) + 128 * (D + 1) + jr), exp2_fast(__ldcg(piece(x, c0) + 128 * D + jr) - base), total);
            const float inv_all = total > 0.f || total != total ? 1.f / total : 0.f;
            const int jt = paged_token(p, r_lo + jr);
            T* jdst = static_cast<T*>(p.out) + (int64_t)(done.q0 + jt) * p.out_token +
                      (int64_t)(done.head * p.group + r_lo + jr - jt * p.group) * p.out_head;
#pragma unroll 1
            for (int c = c_from; c < D; c += share * 32) {
              float v[32];
#pragma unroll
              for (int i = 0; i < 32; ++i) v[i] = 0.f;
#pragma unroll 1
              for (int x = x0; x <= x1; x += 4 * by) {
                float4 u[4][8];
                float w[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                  const int xk = x + k * by;
                  const float* src = piece(xk, c0);
                  w[k] = xk <= x1 ? exp2_fast(__ldcg(src + 128 * D + jr) - base) : 0.f;
#pragma unroll
                  for (int i = 0; i < 8; ++i)
                    u[k][i] = xk <= x1 ? __ldcg(reinterpret_cast<const float4*>(src) + (c / 4 + i) * 128 + jr)
                                       : make_float4(0.f, 0.f, 0.f, 0.f);
                }
#pragma unroll
                for (int k = 0; k < 4; ++k)
#pragma unroll
                  for (int i = 0; i < 8; ++i) {
                    v[4 * i] = fmaf(u[k][i].x, w[k], v[4 * i]);
                    v[4 * i + 1] = fmaf(u[k][i].y, w[k], v[4 * i + 1]);
                    v[4 * i + 2] = fmaf(u[k][i].z, w[k], v[4 * i + 2]);
                    v[4 * i + 3] = fmaf(u[k][i].w, w[k], v[4 * i + 3]);
                  }
              }
              if (final) {
                store(jdst, c, v, inv_all);
                store(jdst, c + 16, v + 16, inv_all);
              } else {
#pragma unroll
                for (int i = 0; i < 32; i += 4)
                  __stcg(reinterpret_cast<float4*>(piece(x0, c0)) + (c / 4 + i / 4) * 128 + jr,
                         make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]));
              }
            }
          }
          if (final && lane == 0) s_place[warp - 4].share = share;
          if (!final) {
            named_barrier(1 + q, 128);  // all threads of a row have read its statistics
            if (jr < live && c_from == 0) {
              __stcg(piece(x0, c0) + 128 * D + jr, top);
              __stcg(piece(x0, c0) + 128 * (D + 1) + jr, total);
            }
          }
        };
        uint32_t* ticket = tickets + c0 * 2 + q;
        uint32_t* run_ticket = tickets + gridDim.x * 2 + (run.x0 * 2 + (run.x0 == c0 ? 1 : 0)) * 2 + q;
        if (run.runs == 1) {
          if (last_of(ticket, c1 - c0 + 1)) join(c0, c1, 1, true);
        } else if (last_of(run_ticket, run.x1 - run.x0 + 1)) {
          join(run.x0, run.x1, 1, false);
          if (last_of(ticket, run.runs)) join(c0, c1, run.by, true);
        }
        __syncwarp();
      }
      __syncwarp();
      if (__builtin_expect(*const_cast<volatile uint32_t*>(&s_odd[warp - 4]) != 0u, 0))
        chunk_settle<T>(p, &s_place[warp - 4], &s_odd[warp - 4]);
    }
    if (lent) named_barrier(5, 256);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) tmem_free(tmem, 512);
}

namespace {

template <typename T, int D>
cudaError_t launch_chunk(const ChunkArgs& a, cudaStream_t st, bool pdl) {
  using C = ChunkCfg<D>;
  static_assert(C::kSmem <= 227 * 1024, "shared memory");
  auto kern = paged_attention_chunk_kernel<T, D>;
  static SmemLimit limit;
  if (const cudaError_t e = limit.raise(kern, C::kSmem); e != cudaSuccess) return e;
  const int ctas = device_sm_count();
  if (ctas * 6 > kPagedTickets || (size_t)ctas * 4 * C::kPart * 4 + kPagedTickets * 4 > kPagedWorkspaceBytes)
    return cudaErrorNotSupported;
  return launch_kernel(kern, dim3(ctas), dim3(kChunkThreads), C::kSmem, st, pdl, a);
}

}  // namespace

cudaError_t launch_paged_attention_chunk(const PagedAttnArgs& a, int dtype, cudaStream_t st, bool pdl) {
  if ((dtype != kBF16 && dtype != kF16) || a.dim > 128 || !(a.scale > 0.f))
    return cudaErrorNotSupported;  // a maximum of scores is one of scaled scores for a positive scale only
  // units of work (paged_sched.cuh) in 32 bits
  const long long items = (long long)a.tokens * a.group / kChunkRows + a.requests;
  if (items * a.kv_heads * ((long long)a.width * a.block_size / kChunkKeys + 2 + kChunkItem) >= INT_MAX)
    return cudaErrorNotSupported;
  ChunkArgs c{};
  c.a = a;
  c.box = paged_box(a.block_size, kChunkKeys);
  if (c.box < 8 || !paged_maps(a, dtype, c.box, &c.k_map, &c.v_map)) return cudaErrorNotSupported;
  c.q_tma = paged_q_map(a, dtype, 128, &c.q_map);
  c.out32 = reinterpret_cast<uintptr_t>(a.out) % 32 == 0 && a.out_token % 16 == 0 && a.out_head % 16 == 0 && a.dim % 16 == 0;
  if (dtype == kBF16)
    return a.dim <= 64 ? launch_chunk<__nv_bfloat16, 64>(c, st, pdl) : launch_chunk<__nv_bfloat16, 128>(c, st, pdl);
  return a.dim <= 64 ? launch_chunk<__half, 64>(c, st, pdl) : launch_chunk<__half, 128>(c, st, pdl);
}

}  // namespace mlora
