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
// What bounds it is reading one or two rows of the vocabulary a request, behind
// three dependent loads (offsets, drafts, their probabilities). A cluster of up to 8
// CTAs takes one request: its warps, with a contiguous stretch of the vocabulary
// each, sum their weights in one pass, the CTAs tell one another their sums over
// distributed shared memory, and the CTA that has the place reads the one warp's
// stretch again (from L2), 16 bytes a thread, to find the token. The weights are
// exact, so no order of these sums has to be kept. Measured: 256 requests of 0 to 4
// drafts over 128256 words in fp32 47.5 us, 4.1 TB/s (63 % of the measured copy): the loads pause while
// drafts are accepted and sums exchanged; one request of 32000 words 5.2 us.
#include <type_traits>

#include "common.cuh"
#include "kernels.h"
#include "paged.h"
#include "tma.cuh"

namespace mlora {

constexpr int kVerifyNT = 256;
constexpr int kVerifyMaxCtas = 8;  // of a cluster

// floor(2^40 x) as 2^23 hi + lo, x clamped to [0, 1] (NaN gives 0), by exact steps in
// fp32: x 2^17 + 2^23 rounded down ends in the bits of floor(x 2^17), and the
// rest times 2^23 likewise. A conversion to 64 bits costs several times as much.
// hi and lo come with the bits of 2^23 on top (kVerifyBias each).
constexpr uint32_t kVerifyBias = 0x4B000000u;
__device__ __forceinline__ void verify_fixed(float x, uint32_t& hi, uint32_t& lo) {
  x = fminf(fmaxf(x, 0.f), 1.f);
  const float t = __fmaf_rd(x, 131072.f, 8388608.f);
  const float rest = __fmaf_rn(x, 131072.f, -__fadd_rn(t, -8388608.f));
  hi = __float_as_uint(t);
  lo = __float_as_uint(__fmaf_rd(rest, 8388608.f, 8388608.f));
}

// floor(total * U / 2^24) without a 128-bit product: both parts are exact.
__device__ __forceinline__ long long verify_place(long long total, long long U) {
  return (total >> 32) * U * 256 + (((total & 0xffffffffll) * U) >> 24);
}

__device__ __forceinline__ void verify_tell(long long* p, uint32_t rank, long long v) {  // into a peer's shared memory
  asm volatile("st.shared::cluster.s64 [%0], %1;" ::"r"(cluster_map(smem_addr(p), rank)), "l"(v) : "memory");
}

// CTAs an SM: eight where the registers allow it (256 x 128256 in fp32, before the search below took 16 bytes a thread: 51 us; 54 with six, or with four of 512 threads)
template <typename T, int V>  // V elements a load: 16 bytes, or one
__global__ void __launch_bounds__(kVerifyNT, sizeof(T) == 4 ? 8 : 6) verify_draft_kernel(const VerifyArgs p, int segment) {
  constexpr int kWarps = kVerifyNT / 32;
  __shared__ long long s_warp[kWarps], s_find[kWarps], s_cta[2][kVerifyMaxCtas];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int ctas = gridDim.x, rank = blockIdx.x, i = blockIdx.y;
  if (ctas > 1) cluster_arrive_release();  // waited for before the first store to a peer
  pdl_wait();
  pdl_trigger();
  int64_t* out = p.tokens + (int64_t)i * (p.max_drafts + 1);
  const int64_t* drafts = p.draft_tokens + (int64_t)i * p.max_drafts;
  // loads that depend on nothing, all at once
  const int r0 = __ldcg(p.row_indptr + i), n = __ldcg(p.row_indptr + i + 1) - r0 - 1;
  int64_t x = lane < p.max_drafts ? __ldcg(drafts + lane) : -1;
  float au = lane < p.max_drafts ? __ldcg(p.accept_u + (int64_t)i * p.max_drafts + lane) : 0.f;
  const float u = __ldcg(p.sample_u + i);
  const bool rows_ok = r0 >= 0 && n >= 0 && (int64_t)r0 + n < p.rows && n <= p.max_drafts;
  if (!rows_ok) {  // no row for this request (fine), or rows that are not there; the same in the whole cluster
    if (rank == 0) {
      if (tid == 0 && !(n == -1 && r0 >= 0)) flag_error(p.status, kErrIndptr);
      for (int j = tid; j <= p.max_drafts; j += kVerifyNT) out[j] = -1;
      if (tid == 0) p.num_emitted[i] = 0;
    }
    if (ctas > 1) cluster_wait_acquire();
    return;
  }
  const T* target = static_cast<const T*>(p.target) + (int64_t)r0 * p.target_row;
  const T* draft = static_cast<const T*>(p.draft) + (int64_t)i * p.draft_req;
  // every warp for itself: a draft a lane, and the first one that does not pass
  int kept = n;
  int64_t wrong = -1;  // the refused draft
  for (int j0 = 0; j0 < n; j0 += 32) {
    const int j = j0 + lane;
    if (j0 > 0) {
      x = j < n ? __ldcg(drafts + j) : -1;
      au = j < n ? __ldcg(p.accept_u + (int64_t)i * p.max_drafts + j) : 0.f;
    }
    bool pass = j >= n;
    if (!pass && x >= 0 && x < p.vocab) {
      const float pt = ldcg_f(target + j * p.target_row + x);
      const float qt = p.draft != nullptr ? ldcg_f(draft + j * p.draft_pos + x) : 1.f;
      pass = __fmul_rn(au, qt) < pt;
    }
    const unsigned refused = __ballot_sync(0xffffffffu, !pass);
    if (refused != 0u) {
      kept = j0 + __ffs(refused) - 1;
      wrong = __shfl_sync(0xffffffffu, x, kept - j0);
      break;
    }
  }
  const T* pr = target + kept * p.target_row;
  const T* qr = kept < n && p.draft != nullptr ? draft + kept * p.draft_pos : nullptr;
  int64_t drop = -1;  // the refused draft of a drafter without probabilities
  if (kept < n) {
    if (wrong < 0 || wrong >= p.vocab) {
      if (rank == 0 && tid == 0) flag_error(p.status, kErrDraftRange);
    } else if (p.draft == nullptr) {
      drop = wrong;
    }
  }

  auto weight_of = [](uint32_t hi, uint32_t lo) { return ((long long)(hi - kVerifyBias) << 23) + (lo - kVerifyBias); };
  // hi and lo of elements v .. v + W - 1 below `end`
  auto weights = [&](auto width, int v, int end, uint32_t* hi, uint32_t* lo) {
    constexpr int W = decltype(width)::value;
    float f[W], g[W];
    if (W > 1 && v + W <= end) {
      Chunk<T, W> a, b;
      a.ldcg(pr + v);
      if (qr != nullptr) b.ldcg(qr + v);
      a.to_f(f);
      if (qr != nullptr) b.to_f(g);
    } else {
#pragma unroll
      for (int e = 0; e < W; ++e) {
        f[e] = v + e < end ? ldcg_f(pr + v + e) : 0.f;
        g[e] = qr != nullptr && v + e < end ? ldcg_f(qr + v + e) : 0.f;
      }
    }
    if (drop >= v && drop < v + W) {
#pragma unroll
      for (int e = 0; e < W; ++e) f[e] = v + e == drop ? 0.f : f[e];
    }
#pragma unroll
    for (int e = 0; e < W; ++e) verify_fixed(qr != nullptr ? f[e] - g[e] : f[e], hi[e], lo[e]);
  };

  const int64_t first = (int64_t)rank * kWarps * segment;  // of this CTA's stretches
  const int v0 = (int)min((int64_t)p.vocab, first + (int64_t)warp * segment), v1 = min((int64_t)p.vocab, (int64_t)v0 + segment);
  for (int pass = 0; pass < 2; ++pass) {  // pass 1: p itself, where p - q has no positive part
    if (pass == 1) {
      qr = nullptr;
      drop = -1;
    }
    long long sum = 0;
#pragma unroll 4
    for (int v = v0 + lane * V; v < v1; v += 32 * V) {
      uint32_t hi[V], lo[V], hs = 0u - V * kVerifyBias, ls = 0u - V * kVerifyBias;
      weights(std::integral_constant<int, V>(), v, v1, hi, lo);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        hs += hi[e];
        ls += lo[e];
      }
      sum += ((long long)hs << 23) + ls;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) s_warp[warp] = sum;
    __syncthreads();
    long long own = 0;
    for (int w = 0; w < kWarps; ++w) own += s_warp[w];
    long long total = own, before = 0;  // of the row; of the CTAs before this one
    if (ctas > 1) {
      if (pass == 0) cluster_wait_acquire();  // every CTA of the cluster has begun
      if (tid < ctas) verify_tell(&s_cta[pass][rank], tid, own);
      cluster_arrive_release();
      cluster_wait_acquire();
      total = 0;
      for (int c = 0; c < ctas; ++c) {
        before += c < rank ? s_cta[pass][c] : 0;
        total += s_cta[pass][c];
      }
    }
    if (total > 0) {
      const long long U = u > 0.f ? (long long)(fminf(u * 16777216.f, 16777215.f)) : 0;
      long long place = verify_place(total, U) - before;  // within this CTA's stretches
      if (place >= 0 && place < own) {
        int w = 0;
        while (place >= s_warp[w]) place -= s_warp[w++];
        // the stretch that holds it, by the whole CTA: PER elements side by side a thread (one element each: 256 x 128256 51 us, 47.5 so)
        constexpr int PIECES = V == 1 ? 4 : 1, PER = PIECES * V;
        const int b0 = (int)(first + (int64_t)w * segment), b1 = min(p.vocab, b0 + segment);
        long long at = 0;
        for (int b = b0; b < b1 && at <= place; b += kVerifyNT * PER) {
          const int v = b + tid * PER;
          uint32_t hi[PIECES][V], lo[PIECES][V];
          long long mine = 0;
#pragma unroll
          for (int k = 0; k < PIECES; ++k) {
            weights(std::integral_constant<int, V>(), v + k * V, b1, hi[k], lo[k]);
#pragma unroll
            for (int e = 0; e < V; ++e) mine += weight_of(hi[k][e], lo[k][e]);
          }
          long long incl = mine;
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const long long up = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += up;
          }
          if (lane == 31) s_find[warp] = incl;
          __syncthreads();
          long long all = 0;
          incl += at;
          for (int k = 0; k < kWarps; ++k) {
            incl += k < warp ? s_find[k] : 0;
            all += s_find[k];
          }
          if (place < incl && place >= incl - mine) {
            long long left = place - (incl - mine);
            int found = -1;
#pragma unroll
            for (int k = 0; k < PIECES; ++k)
#pragma unroll
              for (int e = 0; e < V; ++e) {
                left -= weight_of(hi[k][e], lo[k][e]);
                if (left < 0 && found < 0) found = v + k * V + e;
              }
            out[kept] = found;
          }
          at += all;
          __syncthreads();
        }
      }
      break;
    }
    if (pass == 1 && rank == 0 && tid == 0) out[kept] = -1;
    __syncthreads();  // s_warp is written again
  }
  if (rank == 0) {
    for (int j = tid; j <= p.max_drafts; j += kVerifyNT)
      if (j != kept) out[j] = j < kept ? __ldcg(drafts + j) : -1;
    if (tid == 0) p.num_emitted[i] = kept + 1;
  }
}

namespace {

template <typename T>
cudaError_t launch_verify_t(const VerifyArgs& a, bool vec, cudaStream_t st, bool pdl) {
  constexpr int V = 16 / (int)sizeof(T);
  // more than 2048 elements a CTA: below that the CTAs of a cluster only wait for one another
  int ctas = 1;
  while (ctas < kVerifyMaxCtas && a.vocab > 4096 * ctas) ctas *= 2;
  const int unit = 32 * V, warps = ctas * (kVerifyNT / 32);
  const int segment = ((a.vocab + warps - 1) / warps + unit - 1) / unit * unit;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)ctas, (unsigned)a.requests);
  cfg.blockDim = dim3(kVerifyNT);
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)ctas;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = pdl ? 1 : 0;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  if (vec) return cudaLaunchKernelEx(&cfg, verify_draft_kernel<T, V>, a, segment);
  return cudaLaunchKernelEx(&cfg, verify_draft_kernel<T, 1>, a, segment);
}

}  // namespace

cudaError_t launch_verify_draft(const VerifyArgs& a, int dtype, bool vec, cudaStream_t st, bool pdl) {
  switch (dtype) {
    case kBF16: return launch_verify_t<__nv_bfloat16>(a, vec, st, pdl);
    case kF16: return launch_verify_t<__half>(a, vec, st, pdl);
    case kF32: return launch_verify_t<float>(a, vec, st, pdl);
  }
  return cudaErrorInvalidValue;
}

}  // namespace mlora
