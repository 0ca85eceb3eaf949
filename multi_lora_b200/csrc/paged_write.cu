// New keys and values into their slots of the paged cache:
//   cache[slot / B, slot % B, h, :] = new[t, h, :]  for slot = slot_map[t] >= 0
// Rows of `dim` elements are copied as bytes, so every dtype goes the same way.
// A copy of 2 * tokens * heads rows, bound by memory: each thread moves one piece of K
// and the same of V, 32 bytes each (16, or one element, where alignment or
// `dim` do not allow that). Measured, bf16 heads of 128: 4340 tokens of 8 heads
// (36 MB read and written) 8.3 us over sets of inputs larger than L2, 4.3 TB/s (4.9 us from and to L2);
// 64 tokens of 32 heads 2.7 us (2.1), which is a launch and its dependent loads.
// A slot of -1 (padding, or a token without a block) is skipped; a slot past
// the cache is skipped and reported.
#include <climits>

#include "common.cuh"
#include "kernels.h"
#include "paged.h"

namespace mlora {

constexpr int kWriteNT = 256;

struct alignas(32) Piece32 {
  uint32_t w[8];
};
template <typename P>
__device__ __forceinline__ P load_piece(const P* p) {
  if constexpr (sizeof(P) == 32) {
    P v;
    asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(v.w[0]), "=r"(v.w[1]), "=r"(v.w[2]), "=r"(v.w[3]), "=r"(v.w[4]), "=r"(v.w[5]), "=r"(v.w[6]),
                   "=r"(v.w[7])
                 : "l"(p)
                 : "memory");
    return v;
  } else {
    return __ldcg(p);
  }
}
template <typename P>
__device__ __forceinline__ void store_piece(P* p, const P& v) {
  if constexpr (sizeof(P) == 32) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(v.w[0]), "r"(v.w[1]),
                 "r"(v.w[2]), "r"(v.w[3]), "r"(v.w[4]), "r"(v.w[5]), "r"(v.w[6]), "r"(v.w[7])
                 : "memory");
  } else {
    *p = v;
  }
}

template <typename P>  // a piece
__global__ void __launch_bounds__(kWriteNT) paged_write_kernel(const PagedWriteArgs p, uint32_t per_row, int per_elem) {
  pdl_wait();
  pdl_trigger();
  const uint32_t pieces = (uint32_t)p.tokens * (uint32_t)p.heads * per_row;  // below 2^31: checked on the host
  const uint32_t at = blockIdx.x * kWriteNT + threadIdx.x;
  if (at >= pieces) return;
  const uint32_t row = at / per_row, c = at - row * per_row;
  const uint32_t t = row / (uint32_t)p.heads, h = row - t * (uint32_t)p.heads;
  P v[2];
#pragma unroll
  for (int s = 0; s < 2; ++s)
    v[s] = load_piece(static_cast<const P*>(p.side[s].src) + (t * p.side[s].src_token + h * p.side[s].src_head) / per_elem + c);
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
    store_piece(static_cast<P*>(d.dst) + (block * d.block + off * d.slot + h * d.head) / per_elem + c, v[s]);
  }
}

cudaError_t launch_paged_write(const PagedWriteArgs& a, int es, int piece, cudaStream_t st, bool pdl) {
  const int per_elem = piece > es ? piece / es : 1;  // elements in a piece
  const int64_t per_row = a.dim / per_elem, pieces = (int64_t)a.tokens * a.heads * per_row;
  if (pieces > INT_MAX) return cudaErrorInvalidValue;
  const dim3 g((unsigned)((pieces + kWriteNT - 1) / kWriteNT)), b(kWriteNT);
  const uint32_t n = (uint32_t)per_row;
  if (piece == 32) return launch_kernel(paged_write_kernel<Piece32>, g, b, 0, st, pdl, a, n, per_elem);
  if (piece == 16) return launch_kernel(paged_write_kernel<uint4>, g, b, 0, st, pdl, a, n, per_elem);
  if (es == 2) return launch_kernel(paged_write_kernel<unsigned short>, g, b, 0, st, pdl, a, n, 1);
  return launch_kernel(paged_write_kernel<unsigned int>, g, b, 0, st, pdl, a, n, 1);
}

}  // namespace mlora
