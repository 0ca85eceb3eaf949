// Tensor maps over a paged cache (see paged_tma.h).
#include "paged_tma.h"

#include "common.cuh"

namespace mlora {
namespace {

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                 const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiled encode_tiled() {
  static const EncodeTiled fn = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess) {
      (void)cudaGetLastError();
      f = nullptr;
    }
    return reinterpret_cast<EncodeTiled>(f);
  }();
  return fn;
}

bool one_map(CUtensorMap* map, const void* base, int dtype, const PagedAttnArgs& a, int64_t slot, int64_t head,
             int64_t block, int columns, int box) {
  const int es = dtype == kPagedCodes ? 1 : 2;
  const EncodeTiled enc = encode_tiled();
  if (enc == nullptr || a.num_blocks < 1) return false;
  const cuuint64_t dims[4] = {(cuuint64_t)a.dim, (cuuint64_t)a.block_size, (cuuint64_t)a.kv_heads,
                              (cuuint64_t)a.num_blocks};
  // the stride of a dimension of one is never used, but has to be a valid one
  const auto bytes = [&](int64_t s, cuuint64_t n) { return n > 1 ? (cuuint64_t)s * es : ((cuuint64_t)a.dim * es + 15) / 16 * 16; };
  const cuuint64_t strides[3] = {bytes(slot, dims[1]), bytes(head, dims[2]), bytes(block, dims[3])};
  for (const cuuint64_t s : strides)
    if (s == 0 || s % 16 != 0 || s >= (1ull << 40)) return false;
  // What L2 fetches at once is no more than a head's rows have side by side: behind them lies another head's, which is read
  // by another CTA at another time. Caches stored token by token, 96 requests to 4095 keys of 32 heads and 4 to 131071 of 8,
  // codes: heads of 128 bytes, 128 at once 312 and 126 us, 256 at once 376 and 159; of 64 bytes, 64 at once 291 and 80 us, 128 at
  // once 301 and 107, 256 at once 324 and 114.
  const int64_t row = (int64_t)a.dim * es;
  const CUtensorMapL2promotion promotion = slot == a.dim || row >= 256 ? CU_TENSOR_MAP_L2_PROMOTION_L2_256B
                                           : row >= 128                ? CU_TENSOR_MAP_L2_PROMOTION_L2_128B
                                                                       : CU_TENSOR_MAP_L2_PROMOTION_L2_64B;
  const cuuint32_t boxes[4] = {(cuuint32_t)columns, (cuuint32_t)box, 1, 1}, ones[4] = {1, 1, 1, 1};
  return enc(map, dtype == kPagedCodes ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                  : dtype == kBF16     ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                       : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
             4, const_cast<void*>(base), dims, strides, boxes, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
             columns * es == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, promotion,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace

bool paged_maps(const PagedAttnArgs& a, int dtype, int columns, int box, CUtensorMap* k, CUtensorMap* v) {
  return one_map(k, a.k, dtype, a, a.k_slot, a.k_head, a.k_block, columns, box) &&
         one_map(v, a.v, dtype, a, a.v_slot, a.v_head, a.v_block, columns, box);
}

bool paged_q_map(const PagedAttnArgs& a, int dtype, int rows, CUtensorMap* q) {
  const EncodeTiled enc = encode_tiled();
  if (enc == nullptr || rows % a.group != 0 || a.tokens < 1) return false;
  const cuuint64_t dims[3] = {(cuuint64_t)a.dim, (cuuint64_t)a.q_heads, (cuuint64_t)a.tokens};
  const cuuint64_t strides[2] = {a.q_heads > 1 ? (cuuint64_t)a.q_head * 2 : (cuuint64_t)a.dim * 2,
                                 a.tokens > 1 ? (cuuint64_t)a.q_token * 2 : (cuuint64_t)a.dim * 2};
  for (const cuuint64_t s : strides)
    if (s == 0 || s % 16 != 0 || s >= (1ull << 40)) return false;
  const cuuint32_t box[3] = {64, (cuuint32_t)a.group, (cuuint32_t)(rows / a.group)}, ones[3] = {1, 1, 1};
  return enc(q, dtype == kBF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
             const_cast<void*>(a.q), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace mlora
