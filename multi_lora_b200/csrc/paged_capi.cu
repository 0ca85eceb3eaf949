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

int check_cache(const mlora_paged_cache_t* c, bool codes = false) {
  if (c == nullptr) return refuse(MLORA_ERR_INVALID_ARGUMENT, "cache is NULL");
  if (codes ? c->dtype != MLORA_E4M3 : bytes_of(c->dtype) == 0) return refuse(MLORA_ERR_UNSUPPORTED_DTYPE, "unsupported dtype code %d", c->dtype);
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

int check_scales(const mlora_paged_scales_t* s) {
  if (s->k == nullptr || s->v == nullptr) return refuse(MLORA_ERR_INVALID_ARGUMENT, "k / v of the scales are NULL");
  if (s->k_block_stride < 0 || s->k_head_stride < 0 || s->v_block_stride < 0 || s->v_head_stride < 0)
    return refuse(MLORA_ERR_INVALID_ARGUMENT, "negative stride of the scales");
  return MLORA_OK;
}

// Two dimensions of pieces of `size` elements, none on another: the pieces side by side along the one with the smaller stride, and
// runs of them along the other.
bool apart(int64_t n0, int64_t stride0, int64_t n1, int64_t stride1, int64_t size) {
  if (n0 <= 1) return n1 <= 1 || stride1 >= size;
  if (n1 <= 1) return stride0 >= size;
  const int64_t near = stride0 < stride1 ? stride0 : stride1, far = stride0 < stride1 ? stride1 : stride0,
                n = stride0 < stride1 ? n0 : n1;
  return near >= size && (far - size) / near >= n - 1;
}

// Scales that are written: each block and head has one of its own.
int check_scales_apart(const mlora_paged_scales_t* s, const mlora_paged_cache_t& c) {
  if (!apart(c.num_blocks, s->k_block_stride, c.kv_heads, s->k_head_stride, 1) ||
      !apart(c.num_blocks, s->v_block_stride, c.kv_heads, s->v_head_stride, 1))
    return refuse(MLORA_ERR_INVALID_ARGUMENT, "scales that blocks or heads share cannot be appended to");
  return MLORA_OK;
}

int check_rotary(const mlora_rotary_t* r, const int32_t* positions, int32_t head_dim) {
  if (r->pairs < 1 || r->pairs > head_dim / 2)
    return refuse(MLORA_ERR_INVALID_ARGUMENT, "%d pairs of a head_dim of %d", r->pairs, head_dim);
  if (r->turns == nullptr || positions == nullptr) return refuse(MLORA_ERR_INVALID_ARGUMENT, "turns / positions is NULL");
  return MLORA_OK;
}

constexpr int32_t kAppendMaxDim = 512;

// Rows that are written: they must not overlap one another.
bool rows_apart(int64_t tokens, int64_t token_stride, int64_t heads, int64_t head_stride, int64_t dim) {
  return token_stride >= 0 && head_stride >= 0 && apart(tokens, token_stride, heads, head_stride, dim);
}

// What is checked and set alike for a rotation and an append.
int append_common(mlora::PagedAppendArgs& a, const mlora_rotary_t* rotary, const int32_t* positions, int32_t head_dim) {
  if (head_dim < 1 || head_dim > kAppendMaxDim)
    return refuse(MLORA_ERR_INVALID_ARGUMENT, "head_dim %d: 1 to %d are rotated", head_dim, kAppendMaxDim);
  a.dim = head_dim;
  if (rotary == nullptr) return MLORA_OK;
  if (int rc = check_rotary(rotary, positions, head_dim)) return rc;
  a.angles = {rotary->turns, positions, rotary->pairs, rotary->interleaved != 0, rotary->factor};
  return MLORA_OK;
}

// Elements at once that the rows of q, out, k and v allow: 16 bytes, 8 or one element; `wide`: 32 bytes where a
// unit's two vectors lie side by side.
int append_vec(mlora::PagedAppendArgs& a, int es, bool codes) {
  for (int bytes = 32; bytes >= 8; bytes /= 2) {
    const int v = (bytes < 16 ? bytes : 16) / es;
    if (v < 2 || a.dim % v != 0 || a.angles.pairs % v != 0) continue;
    if (a.q_heads > 0 && !(pieces(a.q, es, a.q_token, a.q_head, 0, bytes) && pieces(a.out, es, a.out_token, a.out_head, 0, bytes)))
      continue;
    bool ok = true;
    for (const mlora::PagedSide& s : a.side)
      if (a.kv_heads > 0)
        ok = ok && pieces(s.src, es, s.src_token, s.src_head, 0, bytes) &&
             pieces(s.dst, codes ? 1 : es, s.block, s.slot, s.head, codes ? v : bytes);
    a.wide = ok && bytes == 32;
    if (ok) return v;
  }
  return 1;
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

int mlora_rotate(const void* x, int64_t x_token_stride, int64_t x_head_stride, int64_t tokens, int32_t heads,
                 int32_t head_dim, const int32_t* positions, const mlora_rotary_t* rotary, void* out,
                 int64_t out_token_stride, int64_t out_head_stride, int32_t dtype, void* stream) {
  report_error(0, "");
  const int es = bytes_of(dtype);
  if (es == 0) return refuse(MLORA_ERR_UNSUPPORTED_DTYPE, "unsupported dtype code %d", dtype);
  if (tokens < 0 || heads < 0 || tokens * (heads > 0 ? heads : 1) > INT32_MAX)
    return refuse(MLORA_ERR_INVALID_ARGUMENT, "%lld tokens of %d heads", (long long)tokens, heads);
  if (rotary == nullptr) return refuse(MLORA_ERR_INVALID_ARGUMENT, "rotary is NULL");
  if (head_dim < 1 || head_dim > kAppendMaxDim || rotary->pairs < 1 || rotary->pairs > head_dim / 2)
    return refuse(MLORA_ERR_INVALID_ARGUMENT, "%d pairs of a head_dim of %d: head_dim 2 to %d", rotary->pairs, head_dim,
                  kAppendMaxDim);
  if (x_token_stride < 0 || x_head_stride < 0 || !rows_apart(tokens, out_token_stride, heads, out_head_stride, head_dim))
    return refuse(MLORA_ERR_INVALID_ARGUMENT, "x / out stride");
  if (tokens == 0 || heads == 0) return MLORA_OK;
  if (x == nullptr || out == nullptr) return refuse(MLORA_ERR_INVALID_ARGUMENT, "x / out is NULL");
  mlora::PagedAppendArgs a{};
  if (int rc = append_common(a, rotary, positions, head_dim)) return rc;
  a.q = x;
  a.q_token = x_token_stride;
  a.q_head = x_head_stride;
  a.out = out;
  a.out_token = out_token_stride;
  a.out_head = out_head_stride;
  a.tokens = (int)tokens;
  a.q_heads = heads;
  a.block_size = 1;
  return launched(mlora::launch_paged_append(a, dtype, append_vec(a, es, false), (cudaStream_t)stream, mlora_get_pdl() != 0),
                  "rotation launch");
}

int mlora_append_paged_kv(const void* q, int64_t q_token_stride, int64_t q_head_stride, int32_t q_heads, void* q_out,
                          int64_t q_out_token_stride, int64_t q_out_head_stride, const void* k, int64_t k_token_stride,
                          int64_t k_head_stride, const void* v, int64_t v_token_stride, int64_t v_head_stride,
                          int64_t tokens, int32_t dtype, const mlora_paged_cache_t* cache,
                          const mlora_paged_scales_t* scales, const mlora_rotary_t* rotary, const int32_t* positions,
                          const int32_t* slot_map, uint32_t* status, void* stream) {
  report_error(0, "");
  const int es = bytes_of(dtype);
  if (es == 0) return refuse(MLORA_ERR_UNSUPPORTED_DTYPE, "unsupported dtype code %d", dtype);
  const bool codes = scales != nullptr;
  if (int rc = check_cache(cache, codes)) return rc;
  const mlora_paged_cache_t& c = *cache;
  if (codes) {
    if (c.num_blocks > 0) {
      if (int rc = check_scales(scales)) return rc;
      if (int rc = check_scales_apart(scales, c)) return rc;
    }
    if (c.block_size > mlora::kAppendMaxBlock)
      return refuse(MLORA_ERR_INVALID_ARGUMENT, "blocks of %d codes: at most %d are appended to", c.block_size, mlora::kAppendMaxBlock);
  } else if (c.dtype != dtype) {
    return refuse(MLORA_ERR_INVALID_ARGUMENT, "rows of dtype %d for a cache of %d", dtype, c.dtype);
  }
  if (tokens < 0 || q_heads < 0 || q_heads > INT32_MAX / 4 || c.kv_heads > INT32_MAX / 4 ||
      tokens * ((int64_t)q_heads + 2 * c.kv_heads) > INT32_MAX)
    return refuse(MLORA_ERR_INVALID_ARGUMENT, "%lld tokens of %d and %d heads", (long long)tokens, q_heads, c.kv_heads);
  if (q_heads > 0 && rotary == nullptr) return refuse(MLORA_ERR_INVALID_ARGUMENT, "queries without rotary");
  if (k_token_stride < 0 || k_head_stride < 0 || v_token_stride < 0 || v_head_stride < 0)
    return refuse(MLORA_ERR_INVALID_ARGUMENT, "negative k / v stride");
  if (q_heads > 0 && (q_token_stride < 0 || q_head_stride < 0 ||
                      !rows_apart(tokens, q_out_token_stride, q_heads, q_out_head_stride, c.head_dim)))
    return refuse(MLORA_ERR_INVALID_ARGUMENT, "q / q_out stride");
  if (c.head_dim > kAppendMaxDim || (rotary != nullptr && (rotary->pairs < 1 || rotary->pairs > c.head_dim / 2)))
    return refuse(MLORA_ERR_INVALID_ARGUMENT, "%d pairs of a head_dim of %d: at most %d", rotary != nullptr ? rotary->pairs : 0,
                  c.head_dim, kAppendMaxDim);
  if (tokens == 0) return MLORA_OK;
  if (k == nullptr || v == nullptr || slot_map == nullptr || (q_heads > 0 && (q == nullptr || q_out == nullptr)))
    return refuse(MLORA_ERR_INVALID_ARGUMENT, "q / q_out / k / v / slot_map is NULL");
  mlora::PagedAppendArgs a{};
  if (int rc = append_common(a, rotary, positions, c.head_dim)) return rc;
  a.q = q;
  a.q_token = q_token_stride;
  a.q_head = q_head_stride;
  a.out = q_out;
  a.out_token = q_out_token_stride;
  a.out_head = q_out_head_stride;
  a.side[0] = {k, k_token_stride, k_head_stride, c.k, c.k_block_stride, c.k_slot_stride, c.k_head_stride};
  a.side[1] = {v, v_token_stride, v_head_stride, c.v, c.v_block_stride, c.v_slot_stride, c.v_head_stride};
  a.slot_map = slot_map;
  a.tokens = (int)tokens;
  a.q_heads = q_heads;
  a.kv_heads = c.kv_heads;
  a.block_size = c.block_size;
  a.num_blocks = c.num_blocks;
  a.status = status;
  const int vec = append_vec(a, es, codes);
  const cudaStream_t st = (cudaStream_t)stream;
  const bool pdl = mlora_get_pdl() != 0;
  if (!codes) return launched(mlora::launch_paged_append(a, dtype, vec, st, pdl), "append launch");
  a.scale[0] = scales->k;
  a.scale[1] = scales->v;
  a.scale_block[0] = scales->k_block_stride;
  a.scale_block[1] = scales->v_block_stride;
  a.scale_head[0] = scales->k_head_stride;
  a.scale_head[1] = scales->v_head_stride;
  return launched(mlora::launch_paged_append_codes(a, dtype, vec, st, pdl), "append launch");
}

size_t mlora_paged_attention_workspace_bytes(void) { return (size_t)64 << 20; }

}  // extern "C"

namespace {

int attention(const void* q, int64_t q_token_stride, int64_t q_head_stride, int64_t tokens, int32_t q_heads, int32_t dtype,
              const mlora_paged_cache_t* cache, const mlora_paged_scales_t* scales, const int32_t* block_tables,
              int64_t table_row_stride, int64_t max_blocks, const int32_t* kv_lens, const int32_t* q_indptr,
              int64_t requests, int64_t max_q_len, float scale, int32_t window, void* out, int64_t out_token_stride,
              int64_t out_head_stride, void* workspace, size_t workspace_bytes, uint32_t* status, void* stream) {
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
  const int es = bytes_of(dtype), ces = scales != nullptr ? 1 : es;
  if (scales != nullptr) {
    a.k_scale = scales->k;
    a.v_scale = scales->v;
    a.ks_block = scales->k_block_stride;
    a.ks_head = scales->k_head_stride;
    a.vs_block = scales->v_block_stride;
    a.vs_head = scales->v_head_stride;
  }
  const bool vec = pieces(q, es, q_token_stride, q_head_stride) && pieces(out, es, out_token_stride, out_head_stride) &&
                   pieces(c.k, ces, c.k_block_stride, c.k_slot_stride, c.k_head_stride) &&
                   pieces(c.v, ces, c.v_block_stride, c.v_slot_stride, c.v_head_stride);
  const bool pdl = mlora_get_pdl() != 0;
  const cudaStream_t st = (cudaStream_t)stream;
  // rows (tokens x group) times group below 2^32: where division by multiplication is exact
  const bool rows_ok = (int64_t)a.tokens * a.group * a.group < (1ll << 32);
  if (vec && es == 2 && rows_ok) {
    const bool few = (int64_t)a.max_q_len * (q_heads / c.kv_heads) <= mlora::kDecodeMaxRows;
    const cudaError_t e = few                 ? mlora::launch_paged_attention_decode(a, dtype, st, pdl)
                          : scales == nullptr ? mlora::launch_paged_attention_chunk(a, dtype, st, pdl)
                                              : mlora::launch_paged_attention_code_chunk(a, dtype, st, pdl);
    if (e != cudaErrorNotSupported) return launched(e, "paged attention launch");
  }
  return launched(mlora::launch_paged_attention_general(a, dtype, vec, st, pdl), "paged attention launch");
}

}  // namespace

extern "C" {

int mlora_paged_attention(const void* q, int64_t q_token_stride, int64_t q_head_stride, int64_t tokens,
                          int32_t q_heads, const mlora_paged_cache_t* cache, const int32_t* block_tables,
                          int64_t table_row_stride, int64_t max_blocks, const int32_t* kv_lens,
                          const int32_t* q_indptr, int64_t requests, int64_t max_q_len, float scale, int32_t window,
                          void* out, int64_t out_token_stride, int64_t out_head_stride, void* workspace,
                          size_t workspace_bytes, uint32_t* status, void* stream) {
  report_error(0, "");
  if (int rc = check_cache(cache)) return rc;
  return attention(q, q_token_stride, q_head_stride, tokens, q_heads, cache->dtype, cache, nullptr, block_tables,
                   table_row_stride, max_blocks, kv_lens, q_indptr, requests, max_q_len, scale, window, out,
                   out_token_stride, out_head_stride, workspace, workspace_bytes, status, stream);
}

int mlora_paged_attention_8bit(const void* q, int64_t q_token_stride, int64_t q_head_stride, int64_t tokens,
                               int32_t q_heads, int32_t dtype, const mlora_paged_cache_t* cache,
                               const mlora_paged_scales_t* scales, const int32_t* block_tables,
                               int64_t table_row_stride, int64_t max_blocks, const int32_t* kv_lens,
                               const int32_t* q_indptr, int64_t requests, int64_t max_q_len, float scale,
                               int32_t window, void* out, int64_t out_token_stride, int64_t out_head_stride,
                               void* workspace, size_t workspace_bytes, uint32_t* status, void* stream) {
  report_error(0, "");
  if (bytes_of(dtype) == 0) return refuse(MLORA_ERR_UNSUPPORTED_DTYPE, "unsupported dtype code %d", dtype);
  if (int rc = check_cache(cache, true)) return rc;
  if (scales == nullptr) return refuse(MLORA_ERR_INVALID_ARGUMENT, "scales is NULL");
  if (cache->num_blocks > 0)
    if (int rc = check_scales(scales)) return rc;
  return attention(q, q_token_stride, q_head_stride, tokens, q_heads, dtype, cache, scales, block_tables,
                   table_row_stride, max_blocks, kv_lens, q_indptr, requests, max_q_len, scale, window, out,
                   out_token_stride, out_head_stride, workspace, workspace_bytes, status, stream);
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
