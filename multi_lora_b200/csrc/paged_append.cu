// Rotary positions, alone and on the way into the paged cache (16 or 32 bits): one launch rotates the
// step's queries into `out`, its keys into their slots, and copies its values beside them.
//
//   (a, b) -> factor * (a cos - b sin, b cos + a sin),  angle = position * f_pair  (rotary.cuh)
//
// in fp32, rounded once. Every element is read and written once, three operations each, so memory bounds it.
// A CTA takes a few tokens with all their heads: the {cos, sin} of a token are made once, in shared memory, for
// every head, while the CTA's first rows (four units a thread, 8 x 16 bytes) are on
// their way. A thread has both halves of a pair, so `out` may be the input itself.
#include "kernels.h"
#include "paged_append.cuh"

namespace mlora {

template <typename T, int V>
__global__ void __launch_bounds__(kRotNT) paged_append_kernel(const PagedAppendArgs p, int per_cta, int units) {
  extern __shared__ float2 s_turn[];  // [per_cta][pairs]
  pdl_wait();
  pdl_trigger();
  append_rows<T, V>(p, p.kv_heads, blockIdx.x, per_cta, units, s_turn);
}

namespace {

template <typename T, int V>
cudaError_t append_v(const PagedAppendArgs& a, cudaStream_t st, bool pdl) {
  const int units = (a.dim + 2 * V - 1) / (2 * V), heads = a.q_heads + 2 * a.kv_heads;
  const int per_cta = tokens_per_cta(a, heads, units);
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
