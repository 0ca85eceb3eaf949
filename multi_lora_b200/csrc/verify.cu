// Verification of drafted tokens against the target's probabilities, from given
// uniform numbers.
//
// Request i has rows row_indptr[i] .. of target probabilities p_0 .. p_n and n
// drafts x_0 .. x_{n-1} with the drafter's probabilities q_0 .. q_{n-1} (without
// them every draft counts as certain: q(x) = 1). Draft j is kept while
// u_j * q_j(x_j) < p_j(x_j); at the first refusal a one token comes from the
// positive part of p_a - q_a, after n kept ones from p_n:
//   w_v = floor(2^40 * min(1, max(0, p_v - q_v))),  S = sum_v w_v
//   token = the first v with w_0 + .. + w_v > floor(S * U / 2^24),  U = floor(u * 2^24)
// The weights are whole numbers in 64 bits, so their sums do not depend on the
// order of summation and a draw is the same whatever the split of the
// vocabulary. A row of p - q without any positive part (equal rows) draws from
// p; a row without any probability gives -1.
//
// One CTA per request reads its row twice: once for S, once for the place.
#include "common.cuh"
#include "kernels.h"
#include "paged.h"

namespace mlora {

constexpr int kVerifyNT = 512;

// A probability in 40-bit fixed point; NaN and everything not positive give 0.
__device__ __forceinline__ long long verify_fixed(float x) {
  return x > 0.f ? (long long)(fminf(x, 1.f) * 1099511627776.f) : 0;
}

// floor(total * U / 2^24) without a 128-bit product: both parts are exact.
__device__ __forceinline__ long long verify_place(long long total, long long U) {
  return (total >> 32) * U * 256 + (((total & 0xffffffffll) * U) >> 24);
}

template <typename T>
__global__ void __launch_bounds__(kVerifyNT) verify_draft_kernel(const VerifyArgs p) {
  __shared__ long long s_warp[kVerifyNT / 32];
  __shared__ int s_kept, s_token;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int i = blockIdx.x;
  pdl_wait();
  pdl_trigger();
  int64_t* out = p.tokens + (int64_t)i * (p.max_drafts + 1);
  int r0 = __ldcg(p.row_indptr + i), n = __ldcg(p.row_indptr + i + 1) - r0 - 1;
  if (r0 < 0 || n < 0 || (int64_t)r0 + n >= p.rows || n > p.max_drafts) {
    // no row for this request (fine), or rows that are not there
    if (tid == 0 && !(n == -1 && r0 >= 0)) flag_error(p.status, kErrIndptr);
    for (int j = tid; j <= p.max_drafts; j += kVerifyNT) out[j] = -1;
    if (tid == 0) p.num_emitted[i] = 0;
    return;
  }
  const T* target = static_cast<const T*>(p.target) + (int64_t)r0 * p.target_row;
  const T* draft = static_cast<const T*>(p.draft) + (int64_t)i * p.draft_req;
  if (tid == 0) {
    int kept = 0;
    for (; kept < n; ++kept) {
      const int64_t x = __ldcg(p.draft_tokens + (int64_t)i * p.max_drafts + kept);
      if (x < 0 || x >= p.vocab) {  // refused
        flag_error(p.status, kErrDraftRange);
        break;
      }
      const float pt = ldcg_f(target + kept * p.target_row + x);
      const float qt = p.draft != nullptr ? ldcg_f(draft + kept * p.draft_pos + x) : 1.f;
      if (!(__fmul_rn(__ldcg(p.accept_u + (int64_t)i * p.max_drafts + kept), qt) < pt)) break;
    }
    s_kept = kept;
    s_token = -1;
  }
  __syncthreads();
  const int kept = s_kept;
  const bool refused = kept < n;
  const T* pr = target + kept * p.target_row;
  const T* qr = draft + kept * p.draft_pos;
  const bool less = refused && p.draft != nullptr;
  const int64_t drop = refused && p.draft == nullptr ? __ldcg(p.draft_tokens + (int64_t)i * p.max_drafts + kept) : -1;
  const float u = __ldcg(p.sample_u + i);
  const long long U = u > 0.f ? (long long)(fminf(u * 16777216.f, 16777215.f)) : 0;

  for (int pass = 0; pass < 2; ++pass) {  // pass 1: p itself, where p - q has no positive part
    auto weight = [&](int v) {
      const float x = ldcg_f(pr + v);
      if (pass == 1) return verify_fixed(x);
      if (v == drop) return 0ll;
      return verify_fixed(less ? x - ldcg_f(qr + v) : x);
    };
    auto block_sum = [&](long long v, long long& before) {  // total; `before`: sum of the warps before this one
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
      __syncthreads();
      if (lane == 0) s_warp[warp] = v;
      __syncthreads();
      long long all = 0;
      before = 0;
      for (int w = 0; w < kVerifyNT / 32; ++w) {
        before += w < warp ? s_warp[w] : 0;
        all += s_warp[w];
      }
      return all;
    };
    long long sum = 0, before;
    for (int v = tid; v < p.vocab; v += kVerifyNT) sum += weight(v);
    const long long total = block_sum(sum, before);
    if (total == 0) continue;
    const long long place = verify_place(total, U);
    long long base = 0;
    for (int v0 = 0; v0 < p.vocab; v0 += kVerifyNT) {
      const int v = v0 + tid;
      const long long w = v < p.vocab ? weight(v) : 0;
      long long incl = w;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long up = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += up;
      }
      const long long all = block_sum(w, before);
      const long long at = base + before + incl;
      if (w > 0 && at > place && at - w <= place) s_token = v;
      base += all;
      if (base > place) break;
    }
    break;
  }
  __syncthreads();
  for (int j = tid; j <= p.max_drafts; j += kVerifyNT)
    out[j] = j < kept ? __ldcg(p.draft_tokens + (int64_t)i * p.max_drafts + j) : j == kept ? (int64_t)s_token : -1;
  if (tid == 0) p.num_emitted[i] = kept + 1;
}

cudaError_t launch_verify_draft(const VerifyArgs& a, int dtype, bool vec, cudaStream_t st, bool pdl) {
  (void)vec;
  const dim3 grid((unsigned)a.requests), block(kVerifyNT);
  switch (dtype) {
    case kBF16: return launch_kernel(verify_draft_kernel<__nv_bfloat16>, grid, block, 0, st, pdl, a);
    case kF16: return launch_kernel(verify_draft_kernel<__half>, grid, block, 0, st, pdl, a);
    case kF32: return launch_kernel(verify_draft_kernel<float>, grid, block, 0, st, pdl, a);
  }
  return cudaErrorInvalidValue;
}

}  // namespace mlora
