// C-ABI entry points of the paged serving step (include/mlora_b200.h): argument
// validation and launch.
#include <climits>
#include <cstdarg>
#include <cstdio>

#include "../../include/mlora_b200.h"
#include "common.cuh"
#include "kernels.h"
#include "paged.h"

namespace {

using mlora::report_error;

int refuse(int code, const char* fmt, ...) {
  char msg[256];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(msg, sizeof(msg), fmt, ap);
  va_end(ap);
  return report_error(code, msg);
}

int launched(cudaError_t e, const char* what) {
  if (e == cudaSuccess) return MLORA_OK;
  return refuse(MLORA_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
}

int bytes_of(int32_t dtype) { return dtype == MLORA_BF16 || dtype == MLORA_F16 ? 2 : dtype == MLORA_F32 ? 4 : 0; }

// Pieces of `bytes`: base aligned, strides whole pieces.
bool pieces(const void* p, int es, int64_t a, int64_t b, int64_t c = 0, int bytes = 16) {
  const int v = bytes / es;
  return reinterpret_cast<uintptr_t>(p) % bytes == 0 && a % v == 0 && b % v == 0 && c % v == 0;
}

int check_cache(const mlora_paged_cache_t* c) {
  if (c == nullptr) return refuse(MLORA_ERR_INVALID_ARGUMENT, "cache is NULL");
  if (bytes_of(c->dtype) == 0) return refuse(MLORA_ERR_UNSUPPORTED_DTYPE, "unsupported dtype code %d", c->dtype);
  if (c->block_size < 1 || c->kv_heads < 1 || c->head_dim < 1 || c->num_blocks < 0)
    return refuse(MLORA_ERR_INVALID_ARGUMENT, "cache of %lld blocks of %d slots, %d heads of %d",
                  (long long)c->num_blocks, c->block_size, c->kv_heads, c->head_dim);
  if (c->num_blocks > INT32_MAX / c->block_size)
    return refuse(MLORA_ERR_INVALID_ARGUMENT, "%lld blocks of %d: slots pass 32 bits", (long long)c->num_blocks,
                  c->block_size);
  if (c->num_blocks > 0 && (c->k == nullptr || c->v == nullptr))
    return refuse(MLORA_ERR_INVALID_ARGUMENT, "k / v of the cache are NULL");
  if (c->k_block_stride < 0 || c->k_slot_stride < 0 || c->k_head_stride < 0 || c->v_block_stride < 0 ||
      c->v_slot_stride < 0 || c->v_head_stride < 0)
    return refuse(MLORA_ERR_INVALID_ARGUMENT, "negative cache stride");
  return MLORA_OK;
}

}  // namespace

extern "C" {

int mlora_plan_paged_step(const int32_t* ctx_lens, const int32_t* new_lens, const int32_t* held_blocks,
                          int64_t requests, const int32_t* free_blocks, int64_t num_free, const int32_t* free_head,
                          int32_t* block_tables, int64_t table_row_stride, int64_t max_blocks, int32_t block_size,
                          int32_t* q_indptr, int32_t* kv_lens, int32_t* held_out, int32_t* free_head_out,
                          int32_t* positions, int32_t* slot_map, int64_t max_tokens, uint32_t* ticket,
                          uint32_t* status, void* stream) {
  report_error(0, "");
  if (requests < 0 || requests > mlora::kPlanMaxRequests)
    return refuse(MLORA_ERR_INVALID_ARGUMENT, "%lld requests: 0 to %d are planned at once", (long long)requests,
                  mlora::kPlanMaxRequests);
  if (block_size < 1) return refuse(MLORA_ERR_INVALID_ARGUMENT, "block_size %d < 1", block_size);
  if (max_blocks < 0 || max_blocks * (requests > 0 ? requests : 1) > INT32_MAX || table_row_stride < max_blocks)
    return refuse(MLORA_ERR_INVALID_ARGUMENT, "block tables of %lld x %lld, rows %lld apart", (long long)requests,
                  (long long)max_blocks, (long long)table_row_stride);
  if (num_free < 0 || num_free > INT32_MAX || max_tokens < 0 || max_tokens >= INT32_MAX)
    return refuse(MLORA_ERR_INVALID_ARGUMENT, "%lld free blocks, %lld tokens", (long long)num_free,
                  (long long)max_tokens);
  if ((max_tokens + 1) * (requests > 0 ? requests : 1) > (int64_t)UINT32_MAX)  // sums of clamped lengths in 32 bits
    return refuse(MLORA_ERR_INVALID_ARGUMENT, "%lld requests of %lld tokens: the product passes 32 bits",
                  (long long)requests, (long long)max_tokens);
  if (q_indptr == nullptr || free_head == nullptr || free_head_out == nullptr || ticket == nullptr)
    return refuse(MLORA_ERR_INVALID_ARGUMENT, "q_indptr / free_head / free_head_out / ticket is NULL");
  if (requests > 0 && (ctx_lens == nullptr || new_lens == nullptr || held_blocks == nullptr || kv_lens == nullptr ||
                       held_out == nullptr || (max_blocks > 0 && block_tables == nullptr)))
    return refuse(MLORA_ERR_INVALID_ARGUMENT, "a per-request array is NULL");
  if ((num_free > 0 && free_blocks == nullptr) || (max_tokens > 0 && (positions == nullptr || slot_map == nullptr)))
    return refuse(MLORA_ERR_INVALID_ARGUMENT, "free_blocks / positions / slot_map is NULL");
  mlora::PlanArgs a{};
  a.ctx_lens = ctx_lens;
  a.new_lens = new_lens;
  a.held = held_blocks;
  a.free_blocks = free_blocks;
  a.free_head = free_head;
  a.tables = block_tables;
  a.table_stride = table_row_stride;
  a.q_indptr = q_indptr;
  a.kv_lens = kv_lens;
  a.held_out = held_out;
  a.free_head_out = free_head_out;
  a.positions = positions;
  a.slot_map = slot_map;
  a.requests = (int)requests;
  a.width = (int)max_blocks;
  a.block = block_size;
  a.num_free = (int)num_free;
  a.max_tokens = (int)max_tokens;
  a.ticket = ticket;
  a.status = status;
  return launched(mlora::launch_paged_plan(a, (cudaStream_t)stream, mlora_get_pdl() != 0), "plan launch");
}

int mlora_write_paged_kv(const void* k, int64_t k_token_stride, int64_t k_head_stride, const void* v,
                         int64_t v_token_stride, int64_t v_head_stride, int64_t tokens,
                         const mlora_paged_cache_t* cache, const int32_t* slot_map, uint32_t* status, void* stream) {
  report_error(0, "");
  if (int rc = check_cache(cache)) return rc;
  if (tokens < 0 || tokens > INT32_MAX) return refuse(MLORA_ERR_INVALID_ARGUMENT, "%lld tokens", (long long)tokens);
  if (k_token_stride < 0 || k_head_stride < 0 || v_token_stride < 0 || v_head_stride < 0)
    return refuse(MLORA_ERR_INVALID_ARGUMENT, "negative k / v stride");
  if (tokens == 0) return MLORA_OK;
  if (k == nullptr || v == nullptr || slot_map == nullptr)
    return refuse(MLORA_ERR_INVALID_ARGUMENT, "k / v / slot_map is NULL");
  const mlora_paged_cache_t& c = *cache;
  mlora::PagedWriteArgs a{};
  a.side[0] = {k, k_token_stride, k_head_stride, c.k, c.k_block_stride, c.k_slot_stride, c.k_head_stride};
  a.side[1] = {v, v_token_stride, v_head_stride, c.v, c.v_block_stride, c.v_slot_stride, c.v_head_stride};
  a.slot_map = slot_map;
  a.tokens = (int)tokens;
  a.heads = c.kv_heads;
  a.dim = c.head_dim;
  a.block_size = c.block_size;
  a.num_blocks = c.num_blocks;
  a.status = status;
  const int es = bytes_of(c.dtype);
  int piece = 32;
  for (; piece > es; piece = piece == 32 ? 16 : es)
    if (c.head_dim % (piece / es) == 0 && pieces(k, es, k_token_stride, k_head_stride, 0, piece) &&
        pieces(v, es, v_token_stride, v_head_stride, 0, piece) &&
        pieces(c.k, es, c.k_block_stride, c.k_slot_stride, c.k_head_stride, piece) &&
        pieces(c.v, es, c.v_block_stride, c.v_slot_stride, c.v_head_stride, piece))
      break;
  if (tokens * c.kv_heads * (int64_t)(c.head_dim * es / piece) > INT32_MAX)
    return refuse(MLORA_ERR_INVALID_ARGUMENT, "%lld tokens of %d x %d: too many for one call", (long long)tokens,
                  c.kv_heads, c.head_dim);
  return launched(mlora::launch_paged_write(a, es, piece, (cudaStream_t)stream, mlora_get_pdl() != 0),
                  "cache write launch");
}

size_t mlora_paged_attention_workspace_bytes(void) { return (size_t)64 << 20; }

int mlora_paged_attention(const void* q, int64_t q_token_stride, int64_t q_head_stride, int64_t tokens,
                          int32_t q_heads, const mlora_paged_cache_t* cache, const int32_t* block_tables,
                          int64_t table_row_stride, int64_t max_blocks, const int32_t* kv_lens,
                          const int32_t* q_indptr, int64_t requests, int64_t max_q_len, float scale, int32_t window,
                          void* out, int64_t out_token_stride, int64_t out_head_stride, void* workspace,
                          size_t workspace_bytes, uint32_t* status, void* stream) {
  report_error(0, "");
  if (int rc = check_cache(cache)) return rc;
  const mlora_paged_cache_t& c = *cache;
  if (c.head_dim > 256 || c.head_dim % 8 != 0)
    return refuse(MLORA_ERR_INVALID_ARGUMENT, "head_dim %d: a multiple of 8, at most 256, is wanted", c.head_dim);
  if (q_heads < 1 || q_heads % c.kv_heads != 0)
    return refuse(MLORA_ERR_INVALID_ARGUMENT, "%d query heads over %d key heads", q_heads, c.kv_heads);
  if (tokens < 0 || tokens * q_heads > INT32_MAX || requests < 0 || requests > INT32_MAX || max_q_len < 0)
    return refuse(MLORA_ERR_INVALID_ARGUMENT, "%lld tokens of %lld requests, %lld at most each", (long long)tokens,
                  (long long)requests, (long long)max_q_len);
  if (max_blocks < 0 || max_blocks > (INT32_MAX - 256) / c.block_size || table_row_stride < max_blocks)
    return refuse(MLORA_ERR_INVALID_ARGUMENT, "block tables %lld wide, rows %lld apart", (long long)max_blocks,
                  (long long)table_row_stride);
  if (window < 0) return refuse(MLORA_ERR_INVALID_ARGUMENT, "window %d < 0", window);
  if (q_token_stride < 0 || q_head_stride < 0 || out_token_stride < 0 || out_head_stride < c.head_dim)
    return refuse(MLORA_ERR_INVALID_ARGUMENT, "q / out stride");
  if (tokens > 1 && out_token_stride < c.head_dim)
    return refuse(MLORA_ERR_INVALID_ARGUMENT, "rows of out %lld apart overlap", (long long)out_token_stride);
  if (workspace == nullptr || workspace_bytes < mlora_paged_attention_workspace_bytes() ||
      reinterpret_cast<uintptr_t>(workspace) % 256 != 0)
    return refuse(MLORA_ERR_INVALID_ARGUMENT, "workspace of %zu bytes: %zu, 256-byte aligned, are wanted",
                  workspace_bytes, mlora_paged_attention_workspace_bytes());
  if (tokens == 0) return MLORA_OK;
  if (q == nullptr || out == nullptr) return refuse(MLORA_ERR_INVALID_ARGUMENT, "q / out is NULL");
  if (requests > 0 && (kv_lens == nullptr || q_indptr == nullptr || (max_blocks > 0 && block_tables == nullptr)))
    return refuse(MLORA_ERR_INVALID_ARGUMENT, "block_tables / kv_lens / q_indptr is NULL");
  mlora::PagedAttnArgs a{};
  a.q = q;
  a.q_token = q_token_stride;
  a.q_head = q_head_stride;
  a.k = c.k;
  a.v = c.v;
  a.k_block = c.k_block_stride;
  a.k_slot = c.k_slot_stride;
  a.k_head = c.k_head_stride;
  a.v_block = c.v_block_stride;
  a.v_slot = c.v_slot_stride;
  a.v_head = c.v_head_stride;
  a.tables = block_tables;
  a.table_stride = table_row_stride;
  a.kv_lens = kv_lens;
  a.q_indptr = q_indptr;
  a.out = out;
  a.out_token = out_token_stride;
  a.out_head = out_head_stride;
  a.tokens = (int)tokens;
  a.requests = (int)requests;
  a.q_heads = q_heads;
  a.kv_heads = c.kv_heads;
  a.group = q_heads / c.kv_heads;
  a.group_magic = a.group > 1 ? (uint32_t)((0x100000000ull + a.group - 1) / a.group) : 0u;
  a.dim = c.head_dim;
  a.block_size = c.block_size;
  a.width = (int)max_blocks;
  a.max_q_len = (int)(max_q_len < tokens ? max_q_len : tokens);
  a.num_blocks = c.num_blocks;
  a.window = window;
  a.scale = scale;
  a.workspace = workspace;
  a.status = status;
  const int es = bytes_of(c.dtype);
  const bool vec = pieces(q, es, q_token_stride, q_head_stride) && pieces(out, es, out_token_stride, out_head_stride) &&
                   pieces(c.k, es, c.k_block_stride, c.k_slot_stride, c.k_head_stride) &&
                   pieces(c.v, es, c.v_block_stride, c.v_slot_stride, c.v_head_stride);
  const bool pdl = mlora_get_pdl() != 0;
  const cudaStream_t st = (cudaStream_t)stream;
  // rows (tokens x group) times group below 2^32: where division by multiplication is exact
  const bool rows_ok = (int64_t)a.tokens * a.group * a.group < (1ll << 32);
  if (vec && es == 2 && rows_ok) {
    const bool few = (int64_t)a.max_q_len * (q_heads / c.kv_heads) <= mlora::kDecodeMaxRows;
    const cudaError_t e = few ? mlora::launch_paged_attention_decode(a, c.dtype, st, pdl)
                              : mlora::launch_paged_attention_chunk(a, c.dtype, st, pdl);
    if (e != cudaErrorNotSupported) return launched(e, "paged attention launch");
  }
  return launched(mlora::launch_paged_attention_general(a, c.dtype, vec, st, pdl), "paged attention launch");
}

int mlora_verify_draft(const void* target, int64_t rows, int64_t vocab, int64_t target_row_stride, const void* draft,
                       int64_t draft_request_stride, int64_t draft_row_stride, const int64_t* draft_tokens,
                       const int32_t* row_indptr, int64_t requests, int32_t max_drafts, const float* accept_u,
                       const float* sample_u, int64_t* tokens, int32_t* num_emitted, int32_t dtype, uint32_t* status,
                       void* stream) {
  report_error(0, "");
  const int es = bytes_of(dtype);
  if (es == 0) return refuse(MLORA_ERR_UNSUPPORTED_DTYPE, "unsupported dtype code %d", dtype);
  if (vocab < 1 || vocab > (1 << 22))
    return refuse(MLORA_ERR_INVALID_ARGUMENT, "vocabulary of %lld: 1 to 4194304 are verified", (long long)vocab);
  if (rows < 0 || rows > INT32_MAX || requests < 0 || requests > 65535 || max_drafts < 0 || max_drafts > 65535)
    return refuse(MLORA_ERR_INVALID_ARGUMENT, "%lld rows of %lld requests, %d drafts at most each", (long long)rows,
                  (long long)requests, max_drafts);
  if (target_row_stride < vocab || (draft != nullptr && (draft_row_stride < vocab || draft_request_stride < 0)))
    return refuse(MLORA_ERR_INVALID_ARGUMENT, "rows of probabilities closer than the vocabulary is long");
  if (requests == 0) return MLORA_OK;
  if ((rows > 0 && target == nullptr) || row_indptr == nullptr || sample_u == nullptr || tokens == nullptr ||
      num_emitted == nullptr || (max_drafts > 0 && (draft_tokens == nullptr || accept_u == nullptr)))
    return refuse(MLORA_ERR_INVALID_ARGUMENT, "an array is NULL");
  mlora::VerifyArgs a{};
  a.target = target;
  a.target_row = target_row_stride;
  a.draft = draft;
  a.draft_req = draft_request_stride;
  a.draft_pos = draft_row_stride;
  a.draft_tokens = draft_tokens;
  a.row_indptr = row_indptr;
  a.accept_u = accept_u;
  a.sample_u = sample_u;
  a.tokens = tokens;
  a.num_emitted = num_emitted;
  a.rows = (int)rows;
  a.requests = (int)requests;
  a.max_drafts = max_drafts;
  a.vocab = (int)vocab;
  a.status = status;
  const bool vec = pieces(target, es, target_row_stride, 0) &&
                   (draft == nullptr || pieces(draft, es, draft_request_stride, draft_row_stride));
  return launched(mlora::launch_verify_draft(a, dtype, vec, (cudaStream_t)stream, mlora_get_pdl() != 0),
                  "verify launch");
}

}  // extern "C"
