// Attention of chunks over a paged cache of e4m3 codes, on the fifth-generation tensor cores.
//
// Items, halves of tiles, TMEM and the running maximum are those of csrc/paged_attn_tc.cu. What differs is how K and V
// come to the tensor cores: TMA brings the codes' pages, and a warpgroup of its own writes them as 16-bit values into
// the swizzled tiles that the products read: K in the queries' type, V in f16, both exact. (It takes codes to registers
// before it waits for room to write, so its registers are a stage of the pipeline too.) Scales stay in fp32 outside
// the products:
//   S = Q C_K^T,  x = S f_K - m,  P = exp2(x) f_V u,  O += P C_V,   1 / u the unit of the row's sums
// with f constant over each eight keys, so a key's scale costs nothing beside the scale that a score has anyway (the
// maximum is taken of each eight scores first), and a value's one multiplication of two probabilities.
//
// P is f16 whatever the queries are: 11 bits of it, and nothing coarser than 2^-33 of the largest exp2(x) f_V that the
// row has met, which is 2^8 when u is chosen (paged_codes.cuh). For bf16 results, which keep 8 bits, that is one term and
// half as much work in the second product as the two that bf16 probabilities need; f16 results take two terms. (2^11 leaves
// less room above, and O is multiplied more often: drafts 124 us where 2^8 takes 119, prompts 103 and 98, 2048 tokens over
// 16384 keys 706 and 696.)
//
// Codes of keys that no row sees become zeros on the way, and NaN of those that only some rows see too, which is
// added to these rows' outputs at the end (codes have no infinities).
//
// A tile of 128 rows has two warpgroups, a thread half of a row's columns: with one, and twice the registers, drafts
// took 168 us where two took 134, prompts 105 and 100, and 2048 tokens over 16384 keys 673 and 690.
//
// What bounds it: for 256 rows the exponentials (2048 cycles a tile of 128 keys) and the tensor cores (2048, and for f16
// queries half as much again) beside all else that a softmax issues: a tile takes 5200 cycles, the tensor pipe is busy for two
// fifths of them and the schedulers for a half. For few rows it is the way of a half tile from its scores to its output and back,
// 4500 cycles for two of them, 2 TB/s. Beginnings and ends of short items cost 10 000 cycles each.
//
// Measured, heads of 128: 2048 tokens over 16384 keys, 32 heads over 8, 692 to 708 us in bf16 (0.58 TFLOP, counted without
// what is masked), 798 to 807 in f16; 8 prompts of 128 to 1024 tokens 95 to 98; 32 requests with 1 to 6 drafts to 8192
// keys, 64 heads over 8, f16 119 to 122, bf16 133.
#include <climits>

#include "device.h"
#include "kernels.h"
#include "paged_chunk.cuh"
#include "paged_codes.cuh"
#include "paged_tma.h"

namespace mlora {

constexpr int kCodeThreads = 768;  // Q, TMA and tensor cores; four warpgroups of softmax; one of codes

// Where a CTA begins.
struct CodeStart {
  ChunkSplit split;
  ChunkItem it;
  int pos, unit;  // of the cursor
  PagedRequest found;
  int req, before, in_req;
};
constexpr int kStartAt = 256;  // in shared memory, behind what paged_find_in has there

struct CodeChunkArgs {
  CUtensorMap k_map, v_map, q_map;
  PagedAttnArgs a;
  int box;    // rows of a TMA box of codes
  int q_tma;  // Q tiles are boxes of q_map (group divides 128)
  int out32;  // rows of the output allow 32-byte stores
};

// ROWS: of an item. Where no request has more than 128, the second tile of Q is room for two more tiles of codes on
// their way: they are what such a call, with little to compute a key, waits for. (64 requests of 2000 keys, 8 key heads: 48
// rows in f16 134 us with it and 151 without, 128 rows 149 and 160, 48 rows in bf16 151 and 156.)
template <int D, int ROWS>
struct CodeChunkCfg {
  static constexpr int kSlot = kChunkKeys * D * 2;  // K or V of a tile
  static constexpr int kQ = 128 * D * 2;            // one tile of Q
  static constexpr int kRaw = kChunkKeys * D;       // codes of K or V of a tile
  static constexpr int kTiles = ROWS / 128;         // of Q
  static constexpr int kRaws = (D == 128 ? 2 : 4) + (2 - kTiles) * kQ / kRaw;
  static constexpr int kSlots = D == 128 ? 4 : 8;
  static constexpr int kSmem = kTiles * kQ + kSlots * kSlot + kRaws * kRaw;
  static constexpr int kPart = 128 * (D + 2);  // floats of a tile's piece
  // tiles whose scales wait: K of a tile gets its slot when the scores of the second (D = 64: fourth) tile before it are
  // done, so all of the one before that is
  static constexpr int kScaleTiles = D == 128 ? 4 : 8;
};

__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]),
               "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
// 16 columns, waited for.
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}

// Whether any of the 64 threads at barrier `id` says so; all of them wait for one another.
__device__ __forceinline__ bool barrier_any(int id, bool mine) {
  uint32_t any;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 q, %1, 0;\n\t"
      "bar.red.or.pred p, %2, 64, q;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(any)
      : "r"((uint32_t)mine), "r"(id)
      : "memory");
  return any != 0u;
}

// NaN that was taken out of V, added in TMEM to the outputs of row r, if it sees it: the item's keys of [from, to) that
// not every row sees, those of every tile's half `half` if that is not negative. Seldom run.
template <int D, int ROWS>
__device__ __noinline__ void code_give_back(const PagedAttnArgs& p, uint32_t o_addr, int column, int req, int head, int rt, int qn,
                                            int kv, int r, int from, int to, int half) {
  ChunkItem it;
  it.qn = qn;
  it.kv = kv;
  it.rt = rt;
  it.rows = qn * p.group;
  int seen_lo, seen_hi;
  chunk_seen<ROWS>(p, it, seen_lo, seen_hi);
  const int pos = kv - qn + paged_token(p, r);
  if (r < it.rows) {
    from = max(from, paged_first_key(p, pos));
    to = min(to, pos + 1);
  } else {
    to = from;
  }
#pragma unroll 1
  for (int c = 0; c < D / 2; c += 16) {  // of the columns from `column` on
    uint32_t o[16];
    tmem_ld16(o_addr + c, o);
#pragma unroll 1
    for (int j = from; j < to; ++j) {
      if ((j >= seen_lo && j < seen_hi) || (half >= 0 && ((j / kHalfKeys) & 1) != half)) continue;
      const int block = __ldcg(p.tables + req * p.table_stride + j / p.block_size);
      if (block < 0 || block >= p.num_blocks) continue;
      const unsigned char* src = static_cast<const unsigned char*>(p.v) + block * p.v_block + (j % p.block_size) * p.v_slot +
                                 head * p.v_head + column + c;
#pragma unroll
      for (int i = 0; i < 2; ++i) {  // a dim is a multiple of 8
        if (column + c + 8 * i >= p.dim) continue;
        const uint2 u = __ldcg(reinterpret_cast<const uint2*>(src) + i);
        const uint32_t a = codes_nan(u.x), b = codes_nan(u.y);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (a >> (8 * e + 7) & 1u) o[8 * i + e] = 0x7fc00000u;
          if (b >> (8 * e + 7) & 1u) o[8 * i + 4 + e] = 0x7fc00000u;
        }
      }
    }
    __syncwarp();
    tmem_st16(o_addr + c, o);
  }
  tmem_wait_st();
}

// Sizes as whole numbers: 2^23 + 2^8 (code_log(f) + 127), and what 2^8 (x - m) and it may have as their sum: both
// logarithms, of f and of up, are too small by at most 0.09, so a w is below 2^(kCodeTop + 0.19).
constexpr float kCodeFine = 256.f;
__device__ __forceinline__ float code_size(float f) { return __uint_as_float((__float_as_uint(f) >> 15) + 0x4b000000u); }
__device__ __forceinline__ float code_size_limit(float up) {
  return __uint_as_float(0x4b000000u + (uint32_t)((kCodeTop + 254.f) * kCodeFine) - (__float_as_uint(up) >> 15));
}

// Four codes as values of T.
template <typename T>
__device__ __forceinline__ uint2 code_values(uint32_t x) {
  uint32_t a = codes_lo(x), b = codes_hi(x);
  if constexpr (Num<T>::is_bf16) {
    a = pack_round2<T>(Pack2<__half>::lo(a), Pack2<__half>::hi(a));
    b = pack_round2<T>(Pack2<__half>::lo(b), Pack2<__half>::hi(b));
  }
  return make_uint2(a, b);
}

// 16 codes as values of T: the chunk-th piece of a swizzled row of 128 bytes.
template <typename T>
__device__ __forceinline__ void code_put(unsigned char* row_at, int row, int chunk, const uint4& u) {
  const uint2 a = code_values<T>(u.x), b = code_values<T>(u.y), c = code_values<T>(u.z), d = code_values<T>(u.w);
  *reinterpret_cast<uint4*>(row_at + (((chunk * 2) ^ (row & 7)) << 4)) = make_uint4(a.x, a.y, b.x, b.y);
  *reinterpret_cast<uint4*>(row_at + (((chunk * 2 + 1) ^ (row & 7)) << 4)) = make_uint4(c.x, c.y, d.x, d.y);
}

template <typename T, int D, int ROWS>
__global__ void __launch_bounds__(kCodeThreads, 1)
paged_attention_code_chunk_kernel(const __grid_constant__ CodeChunkArgs args) {
  using C = CodeChunkCfg<D, ROWS>;
  constexpr int NS = C::kSlots, NR = C::kRaws, HALF = kChunkKeys * 128;
  constexpr bool TWO = !Num<T>::is_bf16;      // terms of P
  constexpr float kLeast = 0x1p-149f;         // positive
  constexpr uint32_t S_COL = 0, O_COL = 256;
  extern __shared__ __align__(1024) unsigned char s_raw[];
  __shared__ __align__(8) uint64_t full[NS], empty[NS], raw_full[NR], raw_empty[NR], q_ready[C::kTiles], q_free[C::kTiles], s_full[2][2], p_ready[2][2], pv_done[2][2];
  constexpr int kScaleTiles = C::kScaleTiles;
  __shared__ __align__(16) float s_scale[kScaleTiles][2][kChunkKeys / 8];  // of K and V, for each eight keys
  __shared__ __align__(16) float s_raw_scale[NR / 2][2][kChunkKeys / 8];  // of a tile whose codes have come, with K
  __shared__ uint32_t s_tmem;
  __shared__ bool s_last[2], s_skipped;
  // What the threads of a row tell one another: maximum, size or sum of each half of the columns; and, where both tiles'
  // warpgroups work on one, the second's maximum and sum, and its unit in the first's place.
  __shared__ float s_part[2][2][128];
  __shared__ uint32_t s_taken;      // a NaN was taken out of V
  const PagedAttnArgs& p = args.a;
  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = same_in_warp(tid >> 5);
  unsigned char* smem = s_raw;  // there is no room to align it in: it is, and if it were not nothing would be read or written
  if ((smem_addr(s_raw) & 1023u) != 0u) {
    if (tid == 0) flag_error(p.status, kErrTimeout);
    return;
  }
  unsigned char *ring = smem + C::kTiles * C::kQ, *raw = ring + NS * C::kSlot;

  if (tid == 0) {
    for (int s = 0; s < NS; ++s) {
      mbar_init(&full[s], 4);   // the warps that write codes
      mbar_init(&empty[s], 2);  // both warps of the tensor cores
    }
    for (int s = 0; s < NR; ++s) {
      mbar_init(&raw_full[s], 1);
      mbar_init(&raw_empty[s], 4);
    }
    for (int q = 0; q < 2; ++q) {
      if (q < C::kTiles) {
        mbar_init(&q_ready[q], 1);
        mbar_init(&q_free[q], 2);
      }
      for (int b = 0; b < 2; ++b) {
        mbar_init(&s_full[q][b], 1);
        mbar_init(&p_ready[q][b], 8);
        mbar_init(&pv_done[q][b], 1);
      }
    }
    fence_barrier_init();
    s_taken = 0u;
    tma_prefetch_map(&args.k_map);
    tma_prefetch_map(&args.v_map);
    if (args.q_tma) tma_prefetch_map(&args.q_map);
  }
  if (warp == 1) tmem_alloc(&s_tmem, 512);
  tc_fence_before();
  pdl_wait();
  pdl_trigger();

  // Where this CTA begins is found once, by warp 3 (with many requests by all), and read by the others: 24 warps that each
  // look for themselves take turns at every instruction, 6000 cycles. With two tiles of rows an item every warp still goes
  // from the request to the item by itself. (Drafts 119 us, 113 so; prompts 99 and 96; the item too would be another 1 us of
  // these, but costs the softmax registers: 2048 over 16384 707 us, 685 so, and 677 where every warp finds all.)
  constexpr bool ONCE = ROWS == 128;
  ChunkSplit split = {0, 0, 0, 0};
  ChunkItem it;
  int before, in_req;
  int req;
  PagedRequest found;
  bool skipped = false;  // a request that is not computed
  static_assert(kStartAt >= sizeof(PagedFindRoom<kCodeThreads>) && kStartAt + sizeof(CodeStart) <= sizeof(s_part), "shared memory");
  CodeStart& start = *reinterpret_cast<CodeStart*>(reinterpret_cast<unsigned char*>(s_part) + kStartAt);
  if (warp == 3 || p.requests > 32)
    paged_find_in<kCodeThreads, 32>(
        reinterpret_cast<PagedFindRoom<kCodeThreads>&>(s_part), p.requests,
        [&](int i, int part, int parts, PagedRequest& r) {
          r = paged_request(p, i, part == 0 && blockIdx.x == 0);
          skipped |= r.odd;
          ChunkItem x;
          chunk_request(p, x, i, r);
          int n = 0;
          for (x.rt = part; x.rt * ROWS < x.rows; x.rt += parts) {
            chunk_span<ROWS>(p, x);
            n += x.n + kChunkItem;
          }
          return n * p.kv_heads;
        },
        split, req, found, before, in_req);
  PagedCursor<ChunkSplit> cur(split);
  auto item_of_request = [&](int rel) {  // the item that holds unit `rel` of request it.req: a lane a tile of rows
    const int per_head = in_req / p.kv_heads;
    it.head = rel / per_head;
    rel -= it.head * per_head;
    it.rt = 0;
    for (int rt0 = 0; rt0 * ROWS < it.rows; rt0 += 32) {
      ChunkItem x = it;
      x.rt = rt0 + lane;
      int units = 0;
      if (x.rt * ROWS < x.rows) {
        chunk_span<ROWS>(p, x);
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
    chunk_span<ROWS>(p, it);
  };
  auto next_item = [&]() {
    if (++it.rt * ROWS >= it.rows) {
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
    chunk_span<ROWS>(p, it);
  };
  auto begin = [&]() {
    if (cur.pos < cur.end) {
      chunk_request(p, it, req, found);
      item_of_request(cur.pos - before);
      if (cur.begin(it.n)) next_item();
    }
  };
  if (warp == 3) {
    if (ONCE) begin();
    if (lane == 0) start = {split, it, cur.pos, cur.unit, found, req, before, in_req};
  }
  skipped = __syncthreads_or(skipped);  // and the barriers are initialised, and s_tmem and `start` are there
  if (tid == 0) s_skipped = skipped;    // for its own warp, at the end
  tc_fence_after();
  const uint32_t tmem = s_tmem;
  if constexpr (ONCE) {  // as values that the compiler knows to be uniform
    split = {same_in_warp(start.split.total), same_in_warp(start.split.base), same_in_warp(start.split.rem), same_in_warp(start.split.T)};
    it = {same_in_warp(start.it.req),   same_in_warp(start.it.head), same_in_warp(start.it.rt),    same_in_warp(start.it.q0),
          same_in_warp(start.it.qn),    same_in_warp(start.it.kv),   same_in_warp(start.it.rows),  same_in_warp(start.it.first),
          same_in_warp(start.it.end),   same_in_warp(start.it.tile0), same_in_warp(start.it.n)};
    cur.pos = same_in_warp(start.pos);
    cur.unit = same_in_warp(start.unit);
    cur.end = split.start(blockIdx.x + 1);
  } else {
    split = {same_in_warp(start.split.total), same_in_warp(start.split.base), same_in_warp(start.split.rem), same_in_warp(start.split.T)};
    found = {same_in_warp(start.found.q0), same_in_warp(start.found.qn), same_in_warp(start.found.kv), false};
    req = same_in_warp(start.req);
    before = same_in_warp(start.before);
    in_req = same_in_warp(start.in_req);
    cur.pos = split.start(blockIdx.x);
    cur.end = split.start(blockIdx.x + 1);
    begin();
  }
  __syncthreads();  // s_part is used again
  bool ok = true;

  // Registers: 768 threads are launched with 80 each (61440); the warps of Q, TMA and the tensor cores keep 72, those of
  // codes take 88, and the softmax warps stay: 128 * 72 + 128 * 88 + 512 * 80 = 61440.
  if (warp < 4) {
    regs_down<72>();
    if (warp == 1 || warp == 2) {  // ---- tensor cores, a warp a tile of rows: S of a half, then O of the half before ----
      const int q = warp - 1;
      constexpr uint32_t idesc_s = umma_idesc_f16(Num<T>::is_bf16, 128, kHalfKeys);
      constexpr uint32_t idesc_o = umma_idesc_f16(false, 128, D) | (1u << 16);  // B: columns contiguous
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
      auto values = [&]() {  // half n - 1 of this tile of rows is the newest, half `number` the held one
        const int number = n - 1, b = number & 1;
        wait(&p_ready[q][b], number >> 1);
        tc_fence_after();
        if (elect_one()) {
          const uint32_t a = s_col + b * 64;
#pragma unroll
          for (int i = 0; i < kHalfKeys / 16; ++i) umma_ts(o_col, a + i * 8, held_lo + i * 128, idesc_o, !held_first || i > 0);
          if (TWO) {
#pragma unroll
            for (int i = 0; i < kHalfKeys / 16; ++i) umma_ts(o_col, a + 32 + i * 8, held_lo + i * 128, idesc_o, true);
          }
          umma_commit(&pv_done[q][b]);
          if (held_last) umma_commit(&empty[held_slot]);
        }
        held = false;
      };
      while (cur.take(it.n)) {
        const bool solo = chunk_solo<ROWS>(it);  // this warp then has every other half of the one tile
        const int qs = solo ? 0 : q, h0 = solo ? q : 0;
        const bool odd = !solo && chunk_odd(it, cur);
        const uint32_t q_lo = smem_addr(smem + qs * C::kQ) >> 4;
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
            if (h == h0) wait(&full[vslot], v_phase);
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
    } else if (warp == 0) {  // ---- Q of each item, as soon as the scores of the item before are done ----
      int items[2] = {0, 0};
      while (cur.take(it.n)) {
#pragma unroll
        for (int q = 0; q < C::kTiles; ++q) {
          const int r0 = it.rt * ROWS + q * 128;
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
        if (cur.advance()) next_item();
      }
      __syncwarp();
      if (s_skipped) paged_zero_uncomputed<T>(p, split.total > 0 ? INT_MAX : -1);
      else paged_zero_rest<T>(p);
    } else {  // ---- codes of K and V of each tile, a box of a page a lane, and their scales ----
      const int boxes = kChunkKeys / args.box, eights = args.box / 8;
      int slot = 0, round = 0;
      while (cur.take(it.n)) {
        const int32_t* table = p.tables + it.req * p.table_stride;
        auto lookup = [&](int k, int& block, int& off) {
          const int j = (it.tile0 + cur.tile + k) * kChunkKeys + lane * args.box;
          block = (int)p.num_blocks;  // out of range: zeros
          off = 0;
          if (lane < boxes && j < it.end && j + args.box > it.first) {
            const int e = __ldcg(table + j / p.block_size);
            off = j % p.block_size;
            if (e >= 0 && e < p.num_blocks) block = e;
            else flag_error(p.status, kErrKvRange);
          }
        };
        auto scales_of = [&](int block, float& a, float& b) {
          a = b = 0.f;
          if (block < p.num_blocks) {
            a = __ldcg(p.k_scale + block * p.ks_block + it.head * p.ks_head);
            b = __ldcg(p.v_scale + block * p.vs_block + it.head * p.vs_head);
          }
        };
        // table entries are asked for two tiles ahead, the scales that hang on them one
        int next[2] = {(int)p.num_blocks, (int)p.num_blocks}, next_off[2] = {0, 0};
        float next_k, next_v;
        lookup(0, next[0], next_off[0]);
        if (cur.len > 1) lookup(1, next[1], next_off[1]);
        scales_of(next[0], next_k, next_v);
        for (int k = 0; k < cur.len; ++k) {
          const int block = next[0], off = next_off[0];
          const float fk = next_k, fv = next_v + 0.f;  // no minus zero: code_size reads its bits
          next[0] = next[1];
          next_off[0] = next_off[1];
          if (k + 1 < cur.len) scales_of(next[0], next_k, next_v);
          if (k + 2 < cur.len) lookup(k + 2, next[1], next_off[1]);
#pragma unroll
          for (int side = 0; side < 2; ++side) {
            if (round > 0) ok = __all_sync(0xffffffffu, ok && mbar_poll(&raw_empty[slot], (round - 1) & 1, p.status));
            if (ok) {
              if (side == 0 && lane < boxes)
                for (int i = 0; i < eights; ++i) {
                  s_raw_scale[slot / 2][0][lane * eights + i] = fk;
                  s_raw_scale[slot / 2][1][lane * eights + i] = fv;
                }
              __syncwarp();
              if (lane == 0) mbar_arrive_expect_tx(&raw_full[slot], C::kRaw);
              __syncwarp();
              if (lane < boxes)
                tma_load_4d(raw + slot * C::kRaw + lane * args.box * D, side == 0 ? &args.k_map : &args.v_map, 0, off, it.head,
                            block, &raw_full[slot]);
            }
            if (++slot == NR) {
              slot = 0;
              ++round;
            }
          }
        }
        if (cur.advance()) next_item();
      }
    }
  } else if (warp >= 20) {  // ---- codes to values, 32 keys of each tile a warp ----
    regs_up<88>();
    constexpr int PASSES = D / 16, KEYS = 32 / PASSES;  // pieces of 16 codes a thread, keys at once
    const int w = warp - 20;
    // Eight lanes side by side read and write all banks: the first four pieces of one key and the last four of
    // the next (D = 64: the four pieces of two keys).
    const int sub = lane >> 2 & 1, chunk = D == 128 ? (lane & 3) + 4 * sub : lane & 3;
    const int row0 = w * 32 + (D == 128 ? (lane >> 4) * 2 + (sub ^ (lane >> 3 & 1)) : lane >> 2);
    int slot = 0, round = 0, raw_slot = 0, raw_phase = 0;
    uint32_t tile_no = 0;
    float f = 0.f;  // scales of eight keys: K's in four lanes, V's in four
    uint4 u[PASSES];
    auto let_go = [&]() {  // of codes that have been read
      // These loads may still be under way when an arrival is not: without the fence the next codes came over them.
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&raw_empty[raw_slot]);
      if (++raw_slot == NR) {
        raw_slot = 0;
        raw_phase ^= 1;
      }
    };
    auto take = [&]() {  // the next codes
      ok = __all_sync(0xffffffffu, ok && mbar_poll(&raw_full[raw_slot], raw_phase, p.status));
#pragma unroll
      for (int i = 0; i < PASSES; ++i)
        u[i] = *reinterpret_cast<const uint4*>(raw + raw_slot * C::kRaw + code_at<D>(row0 + i * KEYS, chunk));
      if ((raw_slot & 1) == 0) f = s_raw_scale[raw_slot / 2][lane >> 2 & 1][w * 4 + (lane & 3)];
      if (C::kTiles == 2) let_go();
      if (round > 0) ok = __all_sync(0xffffffffu, ok && mbar_poll(&empty[slot], (round - 1) & 1, p.status));
      return ring + slot * C::kSlot + (chunk >> 2) * HALF;
    };
    auto filled = [&]() {
      if (C::kTiles == 2) {
        fence_proxy_async_smem();
        __syncwarp();
      } else {
        let_go();  // there are others to go on with, and one fence does
      }
      if (lane == 0) mbar_arrive(&full[slot]);
      if (++slot == NS) {
        slot = 0;
        ++round;
      }
    };
    while (cur.take(it.n)) {
      int seen_lo, seen_hi;
      chunk_seen<ROWS>(p, it, seen_lo, seen_hi);
      for (int k = 0; k < cur.len; ++k) {
        const int j0 = (it.tile0 + cur.tile + k) * kChunkKeys;
        unsigned char* to = take();
        if (lane < 8) s_scale[tile_no % kScaleTiles][lane >> 2][w * 4 + (lane & 3)] = f;
        ++tile_no;
#pragma unroll
        for (int i = 0; i < PASSES; ++i) code_put<T>(to + (row0 + i * KEYS) * 128, row0 + i * KEYS, chunk & 3, u[i]);
        filled();
        to = take();
        if (j0 + kChunkKeys > seen_hi || j0 < seen_lo) {  // keys that not every row sees
          bool taken = false;
#pragma unroll
          for (int i = 0; i < PASSES; ++i) {
            const int j = j0 + row0 + i * KEYS;
            if (j >= seen_lo && j < seen_hi) continue;
            const uint4 nan = make_uint4(codes_nan(u[i].x), codes_nan(u[i].y), codes_nan(u[i].z), codes_nan(u[i].w));
            const bool some = j >= it.first && j < it.end;
            taken |= some && (nan.x | nan.y | nan.z | nan.w) != 0u;
            u[i].x &= some ? ~((nan.x >> 7) * 0xffu) : 0u;
            u[i].y &= some ? ~((nan.y >> 7) * 0xffu) : 0u;
            u[i].z &= some ? ~((nan.z >> 7) * 0xffu) : 0u;
            u[i].w &= some ? ~((nan.w >> 7) * 0xffu) : 0u;
          }
          if (taken) count_store(&s_taken, 1u);
        }
#pragma unroll
        for (int i = 0; i < PASSES; ++i) code_put<__half>(to + (row0 + i * KEYS) * 128, row0 + i * KEYS, chunk & 3, u[i]);
        filled();
      }
      if (cur.advance()) next_item();
    }
  } else {  // ---- softmax: two warpgroups a tile of rows, a thread half of a row's columns ----
    const int group = (warp >> 2) - 1, q = group >> 1, side = group & 1, row = tid & 127;
    const int pair = 6 + q * 4 + (warp & 3);  // barrier of the two warps that share 32 rows
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_addr = tmem + lanes + S_COL + q * 128, o_addr = tmem + lanes + O_COL + q * D + side * (D / 2);
    const float sl = p.scale * 1.4426950408889634f;  // scores in powers of two
    uint32_t* tickets = static_cast<uint32_t*>(p.workspace);
    float* parts = reinterpret_cast<float*>(tickets + kPagedTickets);
    int n = 0;             // halves done
    uint32_t tile_no = 0;  // of the current item's first tile
    bool lent = false;     // the other tile's warpgroups still read this one's O and sums
    while (cur.take(it.n)) {
      if (lent) named_barrier(5, 512);
      lent = false;
      const bool solo = chunk_solo<ROWS>(it);  // the tiles' warpgroups share its keys, half by half
      const int r_lo = it.rt * ROWS + (solo ? 0 : q * 128), r = r_lo + row;
      const bool none = r - lane >= it.rows;  // no row in this warp: its lanes of P and O are never looked at
      float m = kCodeNone, l = 0.f;
      float up = kCodeMostUp;  // O is in units of 1 / up (paged_codes.cuh)
      {
        const int pq = it.kv - it.qn + paged_token(p, r);
        const int limit = r < it.rows ? pq + 1 : 0, floor_ = paged_first_key(p, pq);
        // key tiles that every row of this tile sees whole need no mask
        const int r_hi = min(it.rows, r_lo + 128) - 1;
        const int all_end = it.kv - it.qn + paged_token(p, r_lo) + 1,
                  all_first = paged_first_key(p, it.kv - it.qn + paged_token(p, r_hi));
        const int halves = solo ? cur.len : 2 * cur.len - chunk_odd(it, cur);
        const int key0 = (it.tile0 + cur.tile) * kChunkKeys;
#pragma unroll 1
        for (int k = 0; k < halves; ++k, ++n) {
          const int b = n & 1;
          ok = ok && mbar_poll(&s_full[q][b], (n >> 1) & 1, p.status);
          __syncwarp();
          tc_fence_after();
          if (none) {
            if (lane == 0) mbar_arrive(&p_ready[q][b]);
            continue;
          }
          uint32_t s[32];
          tmem_ld32_async(s_addr + b * 64 + side * 32, s);
          const int half = solo ? 2 * k + q : k;  // of the item
          const float* f = &s_scale[(tile_no + (half >> 1)) % kScaleTiles][0][(half & 1) * 8 + side * 4];
          const float4 f4 = *reinterpret_cast<const float4*>(f), g4 = *reinterpret_cast<const float4*>(f + kChunkKeys / 8);
          // not zero, so that minus infinity stays what it is
          float fk[4] = {fmaxf(f4.x * sl, kLeast), fmaxf(f4.y * sl, kLeast), fmaxf(f4.z * sl, kLeast), fmaxf(f4.w * sl, kLeast)};
          tmem_wait_ld();
          tie32(s);
          const int j0 = key0 + half * kHalfKeys + side * 32;
          if (j0 + 32 > all_end || j0 < all_first) {
            const int hi = limit - j0, lo = floor_ - j0;
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (i >= hi || i < lo) s[i] = 0xff800000u;  // -infinity
          }
          const float g[4] = {g4.x, g4.y, g4.z, g4.w};
          float top[4], over[4], size[4];  // of each eight scores: the largest; above m; and with the size of V's scale
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const uint32_t* x = &s[c * 8];
            top[c] = max3(__uint_as_float(x[0]), __uint_as_float(x[1]), __uint_as_float(x[2]));
            top[c] = max3(top[c], __uint_as_float(x[3]), __uint_as_float(x[4]));
            top[c] = fmaxf(max3(top[c], __uint_as_float(x[5]), __uint_as_float(x[6])), __uint_as_float(x[7]));
            over[c] = fmaf(top[c], fk[c], -m);
            size[c] = fmaf(over[c], kCodeFine, code_size(g[c]));
          }
          // Both warps of the rows go by the same maximum and unit. Seldom has one of them a row that needs others; and
          // neither writes P before the other one has its scores.
          const bool mine = fmaxf(max3(over[0], over[1], over[2]), over[3]) > kCodeRaise ||
                            fmaxf(max3(size[0], size[1], size[2]), size[3]) > code_size_limit(up);
          if (barrier_any(pair, mine)) {
            // What a row goes by must not hang on scores of others, which may be of keys that it does not see: its own
            // need is the lowest bit of what its threads tell one another.
            const float mx = fmaxf(max3(top[0] * fk[0], top[1] * fk[1], top[2] * fk[2]), top[3] * fk[3]);
            const uint32_t word = (__float_as_uint(mx) & ~1u) | (uint32_t)mine;
            s_part[q][side][row] = __uint_as_float(word);
            named_barrier(pair, 64);
            const uint32_t other = __float_as_uint(s_part[q][side ^ 1][row]);
            const bool again = ((word | other) & 1u) != 0u;
            const float most = fmaxf(__uint_as_float(word & ~1u), __uint_as_float(other & ~1u));
            const float raised = again && most > m ? most - m : 0.f, back = exp2_fast(-raised);
            if (again) m = fmaxf(m, most);
            float largest = 0.f;
#pragma unroll
            for (int c = 0; c < 4; ++c) largest = fmaxf(largest, g[c] * exp2_fast(fmaf(top[c], fk[c], -m)));
            s_part[q][side ^ 1][row] = largest;  // in the place that it has just read
            named_barrier(pair, 64);
            const float next = again ? code_new_up(0x1p8f, up, raised, fmaxf(largest, s_part[q][side][row])) : up;
            if (k > 0) {
              // O holds the halves before this one once the last product is done
              ok = ok && mbar_poll(&pv_done[q][b ^ 1], ((n - 1) >> 1) & 1, p.status);
              __syncwarp();
              tc_fence_after();
              const float fix = again ? code_rescale(back, up, next) : 1.f;
              l *= back;
#pragma unroll 1
              for (int c = 0; c < D / 2; c += 16) {
                uint32_t o[16];
                tmem_ld16(o_addr + c, o);
#pragma unroll
                for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * fix);
                tmem_st16(o_addr + c, o);
              }
            }
            up = next;
          }
          const uint64_t m2 = pack2(-m, -m);
          const float gk[4] = {code_weight(g[0], up), code_weight(g[1], up), code_weight(g[2], up), code_weight(g[3], up)};
          uint64_t sum[2] = {0, 0};
          constexpr int AT_ONCE = TWO ? 16 : 32;  // keys
#pragma unroll
          for (int c = 0; c < 32; c += AT_ONCE) {
            uint32_t w[AT_ONCE / 2], rest[AT_ONCE / 2];  // P, two keys a column
#pragma unroll
            for (int i = 0; i < AT_ONCE; i += 2) {
              const float f = fk[(c + i) / 8], w_f = gk[(c + i) / 8];
              const uint64_t x = fma2(pack2u(s[c + i], s[c + i + 1]), pack2(f, f), m2);
              const uint64_t pp = pack2(exp2_fast(lo_of(x)), exp2_fast(hi_of(x)));
              sum[(i >> 1) & 1] = add2(sum[(i >> 1) & 1], pp);
              const uint64_t pw = mul2(pp, pack2(w_f, w_f));
              w[i >> 1] = pack_round2<__half>(lo_of(pw), hi_of(pw));
              if constexpr (TWO)
                rest[i >> 1] = pack_round2<__half>(lo_of(pw) - Pack2<__half>::lo(w[i >> 1]), hi_of(pw) - Pack2<__half>::hi(w[i >> 1]));
            }
            const uint32_t to = s_addr + b * 64 + (side * 32 + c) / 2;
            if constexpr (TWO) {
              tmem_st8(to, w);
              tmem_st8(to + 32, rest);
            } else {
              tmem_st16(to, w);
            }
          }
          const uint64_t both = add2(sum[0], sum[1]);
          l += lo_of(both) + hi_of(both);
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&p_ready[q][b]);
        }
      }

      const ChunkItem done = it;
      const bool whole = cur.whole(it.n);
      const int item0 = cur.pos - cur.unit;
      const int tile0 = it.tile0 + cur.tile, tiles = cur.len;
      tile_no += cur.len;
      if (cur.advance()) next_item();

      if (!none) {  // the row's sum
        named_barrier(pair, 64);  // the other warp has read what it was told last
        s_part[q][side][row] = l;
        named_barrier(pair, 64);
        l += s_part[q][side ^ 1][row];
      }
      ok = ok && mbar_poll(&pv_done[q][(n - 1) & 1], ((n - 1) >> 1) & 1, p.status);
      __syncwarp();
      tc_fence_after();
      if (__any_sync(0xffffffffu, *const_cast<volatile uint32_t*>(&s_taken) != 0u))
        code_give_back<D, ROWS>(p, o_addr, side * (D / 2), done.req, done.head, done.rt, done.qn, done.kv, r, tile0 * kChunkKeys,
                          (tile0 + tiles) * kChunkKeys, solo ? q : -1);
      // An item that all four warpgroups worked on: the first two read the others' O too
      // (their threads of a row have the same TMEM lane).
      float own = code_inverse(up), others = 0.f;  // what the two tiles' sums are multiplied by
      if (solo) {
        if (q == 1) {
          if (!none) {
            named_barrier(pair, 64);  // both have the row's sum
            s_part[1][side][row] = side == 0 ? m : l;
          }
          named_barrier(14, 512);  // the first tile's warpgroups have their sums
          if (!none && side == 0) s_part[0][0][row] = up;
          tc_fence_before();
          named_arrive(4, 512);
          lent = true;
          continue;
        }
        named_arrive(14, 512);
        named_barrier(4, 512);
        tc_fence_after();
        const float mate = s_part[1][0][row];
        const float top = fmaxf(m, mate), a = exp2_fast(m - top), c = exp2_fast(mate - top);
        own *= a;
        others = c * code_inverse(s_part[0][0][row]);
        l = l * a + s_part[1][1][row] * c;
        m = top;
      }
      const int t = paged_token(p, r);
      T* dst = static_cast<T*>(p.out) + (int64_t)(done.q0 + t) * p.out_token +
               (int64_t)(done.head * p.group + r - t * p.group) * p.out_head;
      auto store = [&](T* dst, int c, const float* v, float inv) {  // 16 columns: a thread a row, so whole sectors
        uint32_t u[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) u[i] = pack_round2<T>(v[2 * i] * inv, v[2 * i + 1] * inv);
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
      for (int c = 0; c < (none ? 0 : D / 2); c += 16) {
        uint32_t o[16];
        tmem_ld16(o_addr + c, o);
        float v[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(o[i]) * own;
        if (solo) {
          tmem_ld16(o_addr + D + c, o);
#pragma unroll
          for (int i = 0; i < 16; ++i) v[i] = fmaf(__uint_as_float(o[i]), others, v[i]);
        }
        const int col = side * (D / 2) + c;
        if (whole) {
          if (r < done.rows) store(dst, col, v, inv);
        } else {
#pragma unroll
          for (int i = 0; i < 16; i += 4)
            __stcg(reinterpret_cast<float4*>(part) + ((col + i) / 4) * 128 + row, make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]));
        }
      }
      tc_fence_before();
      if (solo) named_arrive(5, 512);
      if (!whole) {
        if (side == 0) {
          __stcg(part + 128 * D + row, m);
          __stcg(part + 128 * (D + 1) + row, l);
        }
        const int c1 = split.last_cta(item0, done.n);
        const PagedJoin run(c0, c1, blockIdx.x);
        auto last_of = [&](uint32_t* ticket, int n) {  // whether this tile's warpgroups are the last of n to get here
          named_barrier(1 + q, 256);
          if (row == 0 && side == 0) {
            __threadfence();
            const bool last = atomicAdd(ticket, 1u) == (uint32_t)(n - 1);
            if (last) *ticket = 0u;
            __threadfence();
            s_last[q] = last;
          }
          named_barrier(1 + q, 256);
          const bool last = s_last[q];
          named_barrier(1 + q, 256);
          return last;
        };
        // Pieces x0, x0 + by, .. x1 of this tile of rows, to the output or as one piece to x0's
        // place; two, four or eight threads a row, 16 columns of two pieces at once.
        auto join = [&](int x0, int x1, int by, bool final) {
          const int live = min(128, done.rows - r_lo), share = live <= 32 ? 4 : live <= 64 ? 2 : 1;
          const int jr = row & (128 / share - 1), c_from = (side * share + row / (128 / share)) * 16;
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
              float v[16];
#pragma unroll
              for (int i = 0; i < 16; ++i) v[i] = 0.f;
#pragma unroll 1
              for (int x = x0; x <= x1; x += 2 * by) {
                float4 u[2][4];
                float w[2];
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                  const int xk = x + k * by;
                  const float* src = piece(xk, c0);
                  w[k] = xk <= x1 ? exp2_fast(__ldcg(src + 128 * D + jr) - base) : 0.f;
#pragma unroll
                  for (int i = 0; i < 4; ++i)
                    u[k][i] = xk <= x1 ? __ldcg(reinterpret_cast<const float4*>(src) + (c / 4 + i) * 128 + jr)
                                       : make_float4(0.f, 0.f, 0.f, 0.f);
                }
#pragma unroll
                for (int k = 0; k < 2; ++k)
#pragma unroll
                  for (int i = 0; i < 4; ++i) {
                    v[4 * i] = fmaf(u[k][i].x, w[k], v[4 * i]);
                    v[4 * i + 1] = fmaf(u[k][i].y, w[k], v[4 * i + 1]);
                    v[4 * i + 2] = fmaf(u[k][i].z, w[k], v[4 * i + 2]);
                    v[4 * i + 3] = fmaf(u[k][i].w, w[k], v[4 * i + 3]);
                  }
              }
              if (final) {
                store(jdst, c, v, inv_all);
              } else {
#pragma unroll
                for (int i = 0; i < 16; i += 4)
                  __stcg(reinterpret_cast<float4*>(piece(x0, c0)) + (c / 4 + i / 4) * 128 + jr,
                         make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]));
              }
            }
          }
          if (!final) {
            named_barrier(1 + q, 256);  // all threads of a row have read its statistics
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
    }
    if (lent) named_barrier(5, 512);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) tmem_free(tmem, 512);
}

namespace {

template <typename T, int D, int ROWS>
cudaError_t launch_code_chunk(const CodeChunkArgs& a, cudaStream_t st, bool pdl) {
  using C = CodeChunkCfg<D, ROWS>;
  static_assert(C::kSmem <= 227 * 1024, "shared memory");
  auto kern = paged_attention_code_chunk_kernel<T, D, ROWS>;
  static SmemLimit limit;
  if (const cudaError_t e = limit.raise(kern, C::kSmem); e != cudaSuccess) return e;
  const int ctas = device_sm_count();
  if (ctas * 6 > kPagedTickets || (size_t)ctas * 4 * C::kPart * 4 + kPagedTickets * 4 > kPagedWorkspaceBytes)
    return cudaErrorNotSupported;
  return launch_kernel(kern, dim3(ctas), dim3(kCodeThreads), C::kSmem, st, pdl, a);
}

template <typename T>
cudaError_t launch_code_chunk(const CodeChunkArgs& a, cudaStream_t st, bool pdl) {
  const bool one = (int64_t)a.a.max_q_len * a.a.group <= 128;  // tile of rows a request
  if (a.a.dim <= 64) return one ? launch_code_chunk<T, 64, 128>(a, st, pdl) : launch_code_chunk<T, 64, kChunkRows>(a, st, pdl);
  return one ? launch_code_chunk<T, 128, 128>(a, st, pdl) : launch_code_chunk<T, 128, kChunkRows>(a, st, pdl);
}

}  // namespace

cudaError_t launch_paged_attention_code_chunk(const PagedAttnArgs& a, int dtype, cudaStream_t st, bool pdl) {
  // a maximum of scores is one of scaled scores for a positive scale only
  if ((dtype != kBF16 && dtype != kF16) || a.dim > 128 || !(a.scale > 0.f)) return cudaErrorNotSupported;
  // units of work (paged_sched.cuh) in 32 bits
  const long long items = (long long)a.tokens * a.group / 128 + a.requests;
  if (items * a.kv_heads * ((long long)a.width * a.block_size / kChunkKeys + 2 + kChunkItem) >= INT_MAX)
    return cudaErrorNotSupported;
  CodeChunkArgs c{};
  c.a = a;
  c.box = paged_box(a.block_size, kChunkKeys);
  if (c.box < 8 || !paged_maps(a, kPagedCodes, a.dim <= 64 ? 64 : 128, c.box, &c.k_map, &c.v_map)) return cudaErrorNotSupported;
  c.q_tma = paged_q_map(a, dtype, 128, &c.q_map);
  c.out32 = reinterpret_cast<uintptr_t>(a.out) % 32 == 0 && a.out_token % 16 == 0 && a.out_head % 16 == 0 && a.dim % 16 == 0;
  return dtype == kBF16 ? launch_code_chunk<__nv_bfloat16>(c, st, pdl) : launch_code_chunk<__half>(c, st, pdl);
}

}  // namespace mlora
