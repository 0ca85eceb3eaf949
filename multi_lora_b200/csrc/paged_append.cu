// Rotary positions, alone and on the way into the paged cache (16 or 32 bits): one launch rotates the
// step's queries into `out`, its keys into their slots, and copies its values beside them.
//
//   (a, b) -> factor * (a cos - b sin, b cos + a sin),  angle = position * f_pair  (rotary.cuh)
//
// in fp32, rounded once. Every element is read and written once, three operations each, so memory bounds it.
// A CTA takes a few tokens with all their heads: the {cos, sin} of a token are made once, in shared memory, for
// every head, while the CTA's first rows are on their way. A thread has both halves of a pair, so `out` may be the
// input itself. One unit (two vectors) a thread at a time and four CTAs an SM: what hides the loads' latency is the other
// CTAs. (Four units in flight a thread and two CTAs: 30 and 46 us where this takes 15.3 and 22.4.)
//
// Measured over sets of inputs larger than L2, bf16 heads of 128: 64 tokens of 32 heads rotated 2.1 us, 4340 tokens
// 15.3 us (4.6 TB/s; torch's copy of as many bytes takes 25 us); with 8 heads of K and V beside them into the cache 2.9
// and 22.4 us (5.1 TB/s). fp32, over four sets: 25.6 us (5.6 TB/s) and 39.5 (5.8).
#include "kernels.h"
#include "paged_append.cuh"

namespace mlora {

template <typename T, int V>
__global__ void __launch_bounds__(kRotNT, 4) paged_append_kernel(const PagedAppendArgs p, int per_cta, int units) {
  extern __shared__ __align__(16) float2 s_turn[];  // [per_cta][pairs]
  pdl_wait();
  pdl_trigger();
  append_rows<T, V>(p, p.kv_heads, blockIdx.x, per_cta, units, s_turn);
}

namespace {

template <typename T, int V>
cudaError_t append_v(const PagedAppendArgs& a, cudaStream_t st, bool pdl) {
  const int units = (a.dim + 2 * V - 1) / (2 * V);
  const int per_cta = tokens_per_cta(a, units);
  const size_t smem = a.angles.turns != nullptr ? (size_t)per_cta * a.angles.pairs * sizeof(float2) : 0;
  if (smem > 48 * 1024) return cudaErrorInvalidValue;
  return launch_kernel(paged_append_kernel<T, V>, dim3((unsigned)((a.tokens + per_cta - 1) / per_cta)), dim3(kRotNT), smem, st,
                       pdl, a, (int)per_cta, units);
}

template <typename T>
cudaError_t append_t(const PagedAppendArgs& a, int vec, cudaStream_t st, bool pdl) {
  if (vec * sizeof(T) == 16) return append_v<T, 16 / (int)sizeof(T)>(a, st, pdl);
  if (vec * sizeof(T) == 8) return append_v<T, 8 / (int)sizeof(T)>(a, st, pdl);
  return append_v<T, 1>(a, st, pdl);
}

}  // namespace

cudaError_t launch_paged_append(const PagedAppendArgs& a, int dtype, int vec, cudaStream_t st, bool pdl) {
  switch (dtype) {
    case kBF16: return append_t<__nv_bfloat16>(a, vec, st, pdl);
    case kF16: return append_t<__half>(a, vec, st, pdl);
    case kF32: return append_t<float>(a, vec, st, pdl);
  }
  return cudaErrorInvalidValue;
}

}  // namespace mlora
