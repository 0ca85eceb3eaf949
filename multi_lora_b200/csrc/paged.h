// Launchers of the paged serving step: block tables and slots, cache write,
// attention over the paged cache, draft verification. The argument blocks
// mirror the C ABI (include/mlora_b200.h), validated by csrc/paged_capi.cu.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "rotary.cuh"

namespace mlora {

struct PlanArgs {
  const int32_t* ctx_lens;
  const int32_t* new_lens;
  const int32_t* held;        // may alias held_out
  const int32_t* free_blocks;
  const int32_t* free_head;   // may alias free_head_out
  int32_t* tables;            // [requests, width], rows table_stride apart
  int64_t table_stride;
  int32_t* q_indptr;
  int32_t* kv_lens;
  int32_t* held_out;
  int32_t* free_head_out;
  int32_t* positions;
  int32_t* slot_map;
  int requests, width, block, num_free, max_tokens;
  uint32_t* ticket;           // one word, zero between calls
  uint32_t* status;
};
constexpr int kPlanMaxRequests = 8192;
cudaError_t launch_paged_plan(const PlanArgs& a, cudaStream_t st, bool pdl);

// One side (K or V) of the cache and of the new rows; strides in elements.
struct PagedSide {
  const void* src;
  int64_t src_token, src_head;
  void* dst;
  int64_t block, slot, head;
};
struct PagedWriteArgs {
  PagedSide side[2];
  const int32_t* slot_map;
  int tokens, heads, dim, block_size;
  int64_t num_blocks;
  uint32_t* status;
};
// es: bytes per element; piece: bytes at once that rows and strides allow (32, 16, or es).
cudaError_t launch_paged_write(const PagedWriteArgs& a, int es, int piece, cudaStream_t st, bool pdl);

// Rows of q rotated into `out`, new keys rotated into the cache and values beside them (csrc/paged_append.cu).
struct PagedAppendArgs {
  RotaryAngles angles;
  const void* q;
  int64_t q_token, q_head;
  void* out;
  int64_t out_token, out_head;
  PagedSide side[2];          // K and V; their heads are kv_heads (0: there is no cache, and no slot_map)
  const int32_t* slot_map;
  int tokens, q_heads, kv_heads, dim, block_size;
  int wide;                   // rows and strides are whole pieces of 32 bytes
  int64_t num_blocks;
  // a cache of e4m3 codes: a scale for each block and head
  float* scale[2];
  int64_t scale_block[2], scale_head[2];
  uint32_t* status;
};
constexpr int kAppendMaxBlock = 2048;  // slots of a block of codes, at most
// vec: elements at once that rows, strides and pairs allow: 16 bytes, 8 or one element.
cudaError_t launch_paged_append(const PagedAppendArgs& a, int dtype, int vec, cudaStream_t st, bool pdl);
cudaError_t launch_paged_append_codes(const PagedAppendArgs& a, int dtype, int vec, cudaStream_t st, bool pdl);

struct PagedAttnArgs {
  const void* q;
  int64_t q_token, q_head;
  const void* k;
  const void* v;
  int64_t k_block, k_slot, k_head, v_block, v_slot, v_head;
  const int32_t* tables;
  int64_t table_stride;
  const int32_t* kv_lens;
  const int32_t* q_indptr;
  void* out;
  int64_t out_token, out_head;
  int tokens, requests, q_heads, kv_heads, dim, block_size, width, max_q_len;
  int group;                  // q_heads / kv_heads
  uint32_t group_magic;       // ceil(2^32 / group), 0 for 1: row / group by a multiplication
  int64_t num_blocks;
  int window;                 // keys a query sees at most, its own among them; 0: no limit
  float scale;
  void* workspace;
  uint32_t* status;
  // K and V are e4m3 codes where these are not null: a scale for each block and head
  const float* k_scale;
  const float* v_scale;
  int64_t ks_block, ks_head, vs_block, vs_head;
};
// Any dtype, head_dim <= 256, block size and stride.
cudaError_t launch_paged_attention_general(const PagedAttnArgs& a, int dtype, bool vec, cudaStream_t st, bool pdl);

// 16-bit caches with head_dim up to 128, block size a multiple of 8, 16-byte pieces
// everywhere. Decode: up to kDecodeMaxRows rows (max_q_len * q_heads / kv_heads);
// chunk: any number. cudaErrorNotSupported: the shape is not one of these.
cudaError_t launch_paged_attention_decode(const PagedAttnArgs& a, int dtype, cudaStream_t st, bool pdl);
constexpr int kDecodeMaxRows = 16;

cudaError_t launch_paged_attention_chunk(const PagedAttnArgs& a, int dtype, cudaStream_t st, bool pdl);
// the same over a cache of codes
cudaError_t launch_paged_attention_code_chunk(const PagedAttnArgs& a, int dtype, cudaStream_t st, bool pdl);

struct VerifyArgs {
  const void* target;         // [rows, vocab]
  int64_t target_row;
  const void* draft;          // [requests, max_drafts, vocab] or null
  int64_t draft_req, draft_pos;
  const int64_t* draft_tokens;  // [requests, max_drafts]
  const int32_t* row_indptr;
  const float* accept_u;      // [requests, max_drafts]
  const float* sample_u;      // [requests]
  int64_t* tokens;            // [requests, max_drafts + 1]
  int32_t* num_emitted;
  int rows, requests, max_drafts, vocab;
  uint32_t* status;
};
cudaError_t launch_verify_draft(const VerifyArgs& a, int dtype, bool vec, cudaStream_t st, bool pdl);

// Bits of the status word beside those of common.cuh (MLORA_STATUS_* of the C ABI).
enum PagedStatusBits : uint32_t {
  kErrLength = 1u << 5,
  kErrExhausted = 1u << 6,
  kErrKvRange = 1u << 7,
  kErrDraftRange = 1u << 8,
};

}  // namespace mlora
