// What the two kernels of chunks share (csrc/paged_attn_tc.cu and csrc/paged_attn_codes_tc.cu): items of 256 rows over
// tiles of 128 keys, and the tensor-core instructions with both halves of their descriptors in registers.
#pragma once

#include "float2.cuh"
#include "paged_sched.cuh"
#include "tc.cuh"

namespace mlora {

constexpr int kChunkKeys = 128;   // keys a tile
constexpr int kHalfKeys = 64;     // keys a step of the tensor cores and the softmax
constexpr int kChunkRows = 256;   // query rows an item: two tiles of 128
constexpr int kChunkJoin = 3;     // joining a piece costs about three key tiles
constexpr int kChunkItem = 2;     // an item costs about two besides its tiles (3 and 4: prompts 5 % slower)
using ChunkSplit = PagedSplit<kChunkJoin, kChunkItem>;

struct ChunkItem {
  int req, head, rt, q0, qn, kv, rows;  // rows: of the whole request
  int first, end;                       // keys that some row of the item sees
  int tile0, n;
};

// ROWS: of an item, kChunkRows or 128 (of which each is one tile).
template <int ROWS = kChunkRows>
__device__ __forceinline__ void chunk_span(const PagedAttnArgs& p, ChunkItem& it) {
  const int r0 = it.rt * ROWS, r1 = min(it.rows, r0 + ROWS);
  const int base = it.kv - it.qn;
  it.first = paged_first_key(p, base + paged_token(p, r0));
  it.end = max(0, base + paged_token(p, r1 - 1) + 1);
  it.tile0 = it.first / kChunkKeys;
  it.n = max(1, (it.end + kChunkKeys - 1) / kChunkKeys - it.tile0);
}

// Keys [lo, hi) that every row of the item sees (none when lo >= hi).
template <int ROWS = kChunkRows>
__device__ __forceinline__ void chunk_seen(const PagedAttnArgs& p, const ChunkItem& it, int& lo, int& hi) {
  const int r0 = it.rt * ROWS, r1 = min(it.rows, r0 + ROWS);
  const int base = it.kv - it.qn;
  lo = paged_first_key(p, base + paged_token(p, r1 - 1));
  hi = max(0, base + paged_token(p, r0) + 1);
}

// One tile of rows only: the warps of both tiles work on it, each on every other half of the keys.
template <int ROWS = kChunkRows>
__device__ __forceinline__ bool chunk_solo(const ChunkItem& it) {
  return ROWS == 128 || it.rows - it.rt * ROWS <= 128;
}

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

template <int N>
__device__ __forceinline__ void regs_down() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void regs_up() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}

}  // namespace mlora
