// New keys and values into their slots of the paged cache:
//   cache[slot / B, slot % B, h, :] = new[t, h, :]  for slot = slot_map[t] >= 0
// Rows of `dim` elements are copied as bytes, so every dtype goes the same way.
// A copy of 2 * tokens * heads rows, bound by memory: each thread moves one
// 16-byte piece (one element where alignment or `dim` do not allow that).
// A slot of -1 (padding, or a token without a block) is skipped; a slot past
// the cache is skipped and reported.
#include "common.cuh"
#include "kernels.h"
#include "paged.h"

namespace mlora {

constexpr int kWriteNT = 256;

template <typename P>  // a piece: uint4, or one element's bytes
__global__ void __launch_bounds__(kWriteNT) paged_write_kernel(const PagedWriteArgs p, int per_row, int per_elem) {
  pdl_wait();
  pdl_trigger();
  const int64_t pieces = (int64_t)p.tokens * p.heads * per_row;
  const int64_t at = (int64_t)blockIdx.x * kWriteNT + threadIdx.x;
  if (at >= pieces) return;
  const int c = (int)(at % per_row);
  const int64_t row = at / per_row;
  const int h = (int)(row % p.heads);
  const int64_t t = row / p.heads;
  const int slot = __ldcg(p.slot_map + t);
  if (slot < 0) return;
  const int block = slot / p.block_size, off = slot - block * p.block_size;
  if (block >= p.num_blocks) {
    if (c == 0 && h == 0) flag_error(p.status, kErrKvRange);
    return;
  }
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    const PagedSide& d = p.side[s];
    const P* src = static_cast<const P*>(d.src) + (t * d.src_token + h * d.src_head) / per_elem + c;
    P* dst = static_cast<P*>(d.dst) + (block * d.block + off * d.slot + h * d.head) / per_elem + c;
    *dst = __ldcg(src);
  }
}

cudaError_t launch_paged_write(const PagedWriteArgs& a, int es, bool vec, cudaStream_t st, bool pdl) {
  const int per_elem = vec ? 16 / es : 1;  // elements in a piece
  const int per_row = a.dim / per_elem;
  const int64_t pieces = (int64_t)a.tokens * a.heads * per_row;
  const int64_t grid = (pieces + kWriteNT - 1) / kWriteNT;
  if (grid > INT32_MAX) return cudaErrorInvalidValue;
  const dim3 g((unsigned)grid), b(kWriteNT);
  if (vec) return launch_kernel(paged_write_kernel<uint4>, g, b, 0, st, pdl, a, per_row, per_elem);
  if (es == 2) return launch_kernel(paged_write_kernel<unsigned short>, g, b, 0, st, pdl, a, per_row, per_elem);
  return launch_kernel(paged_write_kernel<unsigned int>, g, b, 0, st, pdl, a, per_row, per_elem);
}

}  // namespace mlora
