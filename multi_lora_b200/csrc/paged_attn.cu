// Attention of new tokens over the paged cache, for every shape: any of the
// three dtypes, head_dim up to 256, any block size and stride.
//
// Query t of request i (q_len_i new tokens, kv_len_i in the cache, its own
// among them) sits at position pos = kv_len_i - q_len_i + t and sees keys
// max(0, pos - window + 1) .. pos:
//   o = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),  s_j = scale * q . k_j, m = max_j s_j
// in one pass, with the running maximum and sum rescaled when a larger score
// comes (all in fp32). A query that sees no key gives zeros.
//
// One warp per (token, query head), 32 keys at a time: each lane takes one
// key's whole dot product (q in shared memory, K row by row), the warp agrees
// on maximum and sum by shuffles, and then every lane sums its columns of V
// with the 32 probabilities broadcast. Nothing is shared between the query heads
// of a group; csrc/paged_attn_decode.cu and csrc/paged_attn_tc.cu are for that.
#include "common.cuh"
#include "kernels.h"
#include "paged.h"

namespace mlora {

constexpr int kAttnWarps = 4;
constexpr int kAttnMaxDim = 256;

template <typename T, int V>
__global__ void __launch_bounds__(kAttnWarps * 32) paged_attention_general_kernel(const PagedAttnArgs p) {
  __shared__ float s_q[kAttnWarps][kAttnMaxDim];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_wait();
  pdl_trigger();
  const int64_t item = (int64_t)blockIdx.x * kAttnWarps + warp;
  if (item >= (int64_t)p.tokens * p.q_heads) return;
  const int t = (int)(item / p.q_heads), h = (int)(item % p.q_heads);
  T* o = static_cast<T*>(p.out) + t * p.out_token + h * p.out_head;

  // the request of this token: the last one that starts at or before it
  int lo = 0, hi = p.requests - 1;
  while (lo < hi) {
    const int m = (lo + hi + 1) >> 1;
    if (__ldcg(p.q_indptr + m) <= t) lo = m;
    else hi = m - 1;
  }
  int q0 = 0, q1 = 0;
  if (p.requests > 0) {
    q0 = __ldcg(p.q_indptr + lo);
    q1 = __ldcg(p.q_indptr + lo + 1);
  }
  const int64_t cap = (int64_t)p.width * p.block_size;
  int kv = 0;
  if (t >= q0 && t < q1 && q0 >= 0 && q1 <= p.tokens) {
    kv = __ldcg(p.kv_lens + lo);
    if (kv < 0 || kv > cap) {
      if (lane == 0) flag_error(p.status, kErrLength);
      kv = kv < 0 ? 0 : (int)cap;
    }
  } else {
    if (lane == 0 && t < q1) flag_error(p.status, kErrIndptr);
    q1 = q0 = t;
  }
  const int pos = kv - (q1 - q0) + (t - q0);
  const int end = q1 > q0 ? pos + 1 : 0;  // keys [begin, end)
  const int begin = p.window > 0 ? max(0, end - p.window) : 0;

  for (int c = lane; c < p.dim; c += 32)
    s_q[warp][c] = ldcg_f(static_cast<const T*>(p.q) + t * p.q_token + h * p.q_head + c) * p.scale;
  __syncwarp();
  const int g = h / (p.q_heads / p.kv_heads);
  const int32_t* table = p.tables + lo * p.table_stride;
  constexpr int kCols = kAttnMaxDim / 32;
  float acc[kCols];
#pragma unroll
  for (int c = 0; c < kCols; ++c) acc[c] = 0.f;
  float m = -INFINITY, l = 0.f;
  for (int j0 = begin; j0 < end; j0 += 32) {
    const int j = j0 + lane;
    float s = -INFINITY;
    int block = -1;
    if (j < end) {
      block = __ldcg(table + j / p.block_size);
      if (block < 0 || block >= p.num_blocks) {  // such keys and values count as zeros
        flag_error(p.status, kErrKvRange);
        block = -1;
        s = 0.f;
      } else {
        const T* k = static_cast<const T*>(p.k) + block * p.k_block + (j % p.block_size) * p.k_slot + g * p.k_head;
        s = 0.f;
        for (int c = 0; c < p.dim; c += V) {
          Chunk<T, V> ch;
          ch.ldcg(k + c);
          float f[V];
          ch.to_f(f);
#pragma unroll
          for (int e = 0; e < V; ++e) s = fmaf(s_q[warp][c + e], f[e], s);
        }
      }
    }
    float top = s;
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
    const float m_new = fmaxf(m, top);
    const float fix = m_new == -INFINITY ? 1.f : __expf(m - m_new);
    const float w = s == -INFINITY ? 0.f : expf(s - m_new);
    l = l * fix + warp_sum(w);
    m = m_new;
#pragma unroll
    for (int c = 0; c < kCols; ++c) acc[c] *= fix;
    const int n = min(32, end - j0);
    for (int i = 0; i < n; ++i) {
      const float wi = __shfl_sync(0xffffffffu, w, i);
      const int b = __shfl_sync(0xffffffffu, block, i);
      if (b < 0) continue;
      const T* v = static_cast<const T*>(p.v) + b * p.v_block + ((j0 + i) % p.block_size) * p.v_slot + g * p.v_head;
#pragma unroll
      for (int c = 0; c < kCols; ++c)
        if (c * 32 + lane < p.dim) acc[c] = fmaf(wi, ldcg_f(v + c * 32 + lane), acc[c]);
    }
  }
  const float inv = l > 0.f ? 1.f / l : 0.f;
#pragma unroll
  for (int c = 0; c < kCols; ++c)
    if (c * 32 + lane < p.dim) o[c * 32 + lane] = Num<T>::from_f(acc[c] * inv);
}

namespace {
template <typename T>
cudaError_t general_t(const PagedAttnArgs& a, bool vec, cudaStream_t st, bool pdl) {
  const int64_t items = (int64_t)a.tokens * a.q_heads;
  const dim3 grid((unsigned)((items + kAttnWarps - 1) / kAttnWarps)), block(kAttnWarps * 32);
  if (vec) return launch_kernel(paged_attention_general_kernel<T, 16 / (int)sizeof(T)>, grid, block, 0, st, pdl, a);
  return launch_kernel(paged_attention_general_kernel<T, 1>, grid, block, 0, st, pdl, a);
}
}  // namespace

cudaError_t launch_paged_attention_general(const PagedAttnArgs& a, int dtype, bool vec, cudaStream_t st, bool pdl) {
  if (a.dim > kAttnMaxDim || (int64_t)a.tokens * a.q_heads > (int64_t)INT32_MAX) return cudaErrorInvalidValue;
  switch (dtype) {
    case kBF16: return general_t<__nv_bfloat16>(a, vec, st, pdl);
    case kF16: return general_t<__half>(a, vec, st, pdl);
    case kF32: return general_t<float>(a, vec, st, pdl);
  }
  return cudaErrorInvalidValue;
}

}  // namespace mlora
