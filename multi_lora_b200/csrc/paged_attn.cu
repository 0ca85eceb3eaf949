// Attention of new tokens over the paged cache, for every shape: any of the
// three dtypes, head_dim up to 256, any block size and stride; the cache of the queries'
// dtype or of e4m3 codes with a scale for each block and head (a key's scale multiplies
// its score, a value's the probability that goes to the product).
//
// Query t of request i (q_len_i new tokens, kv_len_i in the cache, its own
// among them) sits at position pos = kv_len_i - q_len_i + t and sees keys
// max(0, pos - window + 1) .. pos:
//   o = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),  s_j = scale * q . k_j, m = max_j s_j
// in one pass, with the running maximum and sum rescaled when a larger score
// comes (all in fp32). A query that sees no key gives zeros.
//
// A CTA takes one token and up to four query heads of one key head, its eight
// warps 32 keys each in turn, with sums of their own that are joined at the end. For the
// scores eight lanes share a key (whole sectors of its row; three shuffles join
// their parts), for the output every lane has four columns of all 32 keys. Sums,
// statistics and probabilities are fp32. A cluster of eight CTAs shares
// the keys where a GPU would otherwise have few CTAs, and joins over distributed
// shared memory. What bounds it: the shared keys are fetched again for every
// token and every four heads, mostly from L2; csrc/paged_attn_decode.cu and
// csrc/paged_attn_tc.cu fetch them once. Measured in fp32 (8 key heads of 128, 32 query
// heads): 64 requests of 2000 keys 298 us, 3.5 TB/s of keys and values; one of 60000
// keys 475 us; 512 new tokens 256 us. A warp a (token, query head) and a lane a key
// took 2596, 72700 and 948 us.
// Over codes (64 requests of 2000 keys) fp32 queries take 282 us, and 16 bits with blocks of 12 slots as many: it is
// the work a key and query head, not the bytes.
#include <cuda_fp8.h>

#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "device.h"
#include "kernels.h"
#include "paged.h"
#include "tma.cuh"

namespace mlora {

constexpr int kAttnWarps = 8;
constexpr int kAttnMaxDim = 256;
constexpr int kAttnCtas = 8;  // of a cluster

// V e4m3 codes as they lie in memory.
template <int V>
struct CodeChunk {
  typename RawBytes<V>::type u;
  __device__ __forceinline__ void zero() { u = {}; }
  __device__ __forceinline__ void ldcg(const unsigned char* p) { u = __ldcg(reinterpret_cast<const typename RawBytes<V>::type*>(p)); }
  __device__ __forceinline__ void to_f(float* f) const {
    unsigned char c[V];
    memcpy(c, &u, V);
#pragma unroll
    for (int i = 0; i < V; i += 2) {
      const float2 x = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((unsigned short)(c[i] | c[i + 1] << 8), __NV_E4M3)));
      f[i] = x.x;
      f[i + 1] = x.y;
    }
  }
};
template <>
struct CodeChunk<1> {
  unsigned char u;
  __device__ __forceinline__ void zero() { u = 0; }
  __device__ __forceinline__ void ldcg(const unsigned char* p) { u = __ldcg(p); }
  __device__ __forceinline__ void to_f(float* f) const { f[0] = __half2float(__half(__nv_cvt_fp8_to_halfraw(u, __NV_E4M3))); }
};

// V elements a load of K and Q: 16 bytes of T, or one; H query heads; CODES: K and V are codes with scales
template <typename T, int V, int H, bool CODES>
__global__ void __launch_bounds__(kAttnWarps * 32) paged_attention_general_kernel(const PagedAttnArgs p, int ctas) {
  __shared__ __align__(16) float s_q[H][kAttnMaxDim];
  __shared__ __align__(16) float s_acc[kAttnWarps][H][kAttnMaxDim];
  __shared__ __align__(16) float2 s_stat[kAttnWarps][H];  // maximum and sum
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  pdl_wait();
  pdl_trigger();
  const int parts = (p.group + H - 1) / H;
  const int rank = blockIdx.x % ctas;
  const int item = blockIdx.x / ctas;
  const int t = item / (p.kv_heads * parts), g = item / parts % p.kv_heads, part = item % parts;
  const int h0 = g * p.group + part * H, heads = min(H, p.group - part * H);
  T* out = static_cast<T*>(p.out) + t * p.out_token + h0 * p.out_head;

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
      if (tid == 0) flag_error(p.status, kErrLength);
      kv = kv < 0 ? 0 : (int)cap;
    }
  } else {
    if (tid == 0 && (t < q1 || q1 < q0)) flag_error(p.status, kErrIndptr);
    q1 = q0 = t;
  }
  const int pos = kv - (q1 - q0) + (t - q0);
  const int end = q1 > q0 ? pos + 1 : 0;  // keys [begin, end)
  const int begin = p.window > 0 ? max(0, end - p.window) : 0;

  for (int e = tid; e < H * p.dim; e += kAttnWarps * 32) {
    const int h = e / p.dim, c = e - h * p.dim;
    s_q[h][c] = h < heads ? ldcg_f(static_cast<const T*>(p.q) + t * p.q_token + (h0 + h) * p.q_head + c) * p.scale : 0.f;
  }
  __syncthreads();
  const int32_t* table = p.tables + lo * p.table_stride;
  using E = typename std::conditional<CODES, unsigned char, T>::type;  // an element of the cache
  using Piece = typename std::conditional<CODES, CodeChunk<V>, Chunk<T, V>>::type;
  const E* kbase = static_cast<const E*>(p.k) + g * p.k_head;
  const E* vbase = static_cast<const E*>(p.v) + g * p.v_head;
  constexpr int kCols = kAttnMaxDim / 128;  // runs of 128 columns, four of each a lane
  float acc[H][kCols][4], m[H], l[H];
#pragma unroll
  for (int h = 0; h < H; ++h) {
    m[h] = -INFINITY;
    l[h] = 0.f;
#pragma unroll
    for (int c = 0; c < kCols; ++c) acc[h][c][0] = acc[h][c][1] = acc[h][c][2] = acc[h][c][3] = 0.f;
  }
  // key i of 32 belongs to lane (i % 4) * 8 + i / 4: the eight lanes that share a key have
  // one of their own among them
  const int mine = (lane & 7) * 4 + (lane >> 3);
  for (int64_t j0 = begin + (int64_t)(rank * kAttnWarps + warp) * 32; j0 < end; j0 += (int64_t)ctas * kAttnWarps * 32) {
    const int j = (int)j0 + mine;
    int block = -1, off = 0;
    const bool real = j0 + mine < end;
    if (real) {
      block = __ldcg(table + j / p.block_size);
      off = j % p.block_size;
      if (block < 0 || block >= p.num_blocks) {  // such keys and values count as zeros
        flag_error(p.status, kErrKvRange);
        block = -1;
      }
    }
    float k_scale = 0.f, v_scale = 0.f;
    if (CODES && block >= 0) {
      k_scale = __ldcg(p.k_scale + block * p.ks_block + g * p.ks_head);
      v_scale = __ldcg(p.v_scale + block * p.vs_block + g * p.vs_head);
    }
    float s[H];
#pragma unroll
    for (int h = 0; h < H; ++h) s[h] = 0.f;
    constexpr int AT_ONCE = 4;
#pragma unroll
    for (int i0 = 0; i0 < 8; i0 += AT_ONCE) {  // four keys in each of these steps
      const E* row[AT_ONCE];
      float d[AT_ONCE][H];
#pragma unroll
      for (int i = 0; i < AT_ONCE; ++i) {
        const int from = (lane & 24) | (i0 + i), b = __shfl_sync(0xffffffffu, block, from),
                  o = __shfl_sync(0xffffffffu, off, from);
        row[i] = b < 0 ? nullptr : kbase + b * p.k_block + o * p.k_slot;
#pragma unroll
        for (int h = 0; h < H; ++h) d[i][h] = 0.f;
      }
      for (int c = (lane & 7) * V; c < p.dim; c += 8 * V) {
        Piece ch[AT_ONCE];
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) {
          ch[i].zero();
          if (row[i] != nullptr) ch[i].ldcg(row[i] + c);
        }
        float f[AT_ONCE][V];
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) ch[i].to_f(f[i]);
#pragma unroll
        for (int h = 0; h < H; ++h)
#pragma unroll
          for (int e = 0; e < V; ++e) {
            const float q = s_q[h][c + e];
#pragma unroll
            for (int i = 0; i < AT_ONCE; ++i) d[i][h] = fmaf(q, f[i][e], d[i][h]);
          }
      }
#pragma unroll
      for (int i = 0; i < AT_ONCE; ++i)
#pragma unroll
        for (int h = 0; h < H; ++h) {
          float x = d[i][h];
          x += __shfl_xor_sync(0xffffffffu, x, 1);
          x += __shfl_xor_sync(0xffffffffu, x, 2);
          x += __shfl_xor_sync(0xffffffffu, x, 4);
          if ((lane & 7) == i0 + i) s[h] = x;
        }
    }
    float w[H];
#pragma unroll
    for (int h = 0; h < H; ++h) {
      if (CODES) s[h] *= k_scale;
      if (!real) s[h] = -INFINITY;
      float top = s[h];
#pragma unroll
      for (int x = 16; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
      const float m_new = fmaxf(m[h], top);
      const float fix = m_new == -INFINITY ? 1.f : expf(m[h] - m_new);
      w[h] = s[h] == -INFINITY ? 0.f : expf(s[h] - m_new);
      l[h] = fmaf(l[h], fix, w[h]);
      if (CODES) w[h] *= v_scale;  // of the value that it is multiplied by
      m[h] = m_new;
      if (fix != 1.f) {
#pragma unroll
        for (int c = 0; c < kCols; ++c)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[h][c][e] *= fix;
      }
    }
    const int n = (int)min((int64_t)32, end - j0);
    for (int i0 = 0; i0 < n; i0 += AT_ONCE) {
      float v[AT_ONCE][kCols][4];
#pragma unroll
      for (int i = 0; i < AT_ONCE; ++i) {
        const int from = i * 8 + (i0 >> 2), b = __shfl_sync(0xffffffffu, block, from), o = __shfl_sync(0xffffffffu, off, from);
        const E* src = vbase + b * p.v_block + o * p.v_slot + lane * 4;
#pragma unroll
        for (int c = 0; c < kCols; ++c) {
          v[i][c][0] = v[i][c][1] = v[i][c][2] = v[i][c][3] = 0.f;
          if (b >= 0 && c * 128 + lane * 4 < p.dim) {
            if constexpr (CODES && V > 1) {
              CodeChunk<4> u;
              u.ldcg(src + c * 128);
              u.to_f(v[i][c]);
            } else if constexpr (CODES) {
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                CodeChunk<1> u;
                u.ldcg(src + c * 128 + e);
                u.to_f(&v[i][c][e]);
              }
            } else if constexpr (V > 1 && sizeof(T) == 4) {
              const float4 u = __ldcg(reinterpret_cast<const float4*>(src + c * 128));
              v[i][c][0] = u.x;
              v[i][c][1] = u.y;
              v[i][c][2] = u.z;
              v[i][c][3] = u.w;
            } else if constexpr (V > 1) {
              const uint2 u = __ldcg(reinterpret_cast<const uint2*>(src + c * 128));
              v[i][c][0] = Pack2<T>::lo(u.x);
              v[i][c][1] = Pack2<T>::hi(u.x);
              v[i][c][2] = Pack2<T>::lo(u.y);
              v[i][c][3] = Pack2<T>::hi(u.y);
            } else {
#pragma unroll
              for (int e = 0; e < 4; ++e) v[i][c][e] = ldcg_f(static_cast<const T*>(src) + c * 128 + e);
            }
          }
        }
      }
#pragma unroll
      for (int i = 0; i < AT_ONCE; ++i)
#pragma unroll
        for (int h = 0; h < H; ++h) {
          const float wi = __shfl_sync(0xffffffffu, w[h], i * 8 + (i0 >> 2));
#pragma unroll
          for (int c = 0; c < kCols; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[h][c][e] = fmaf(wi, v[i][c][e], acc[h][c][e]);
        }
    }
  }

  // ---- join: the warps, then the CTAs ----
#pragma unroll
  for (int h = 0; h < H; ++h) {
    l[h] = warp_sum(l[h]);
    if (lane == 0) s_stat[warp][h] = make_float2(m[h], l[h]);
#pragma unroll
    for (int c = 0; c < kCols; ++c)
      *reinterpret_cast<float4*>(&s_acc[warp][h][c * 128 + lane * 4]) = make_float4(acc[h][c][0], acc[h][c][1], acc[h][c][2], acc[h][c][3]);
  }
  __syncthreads();
  auto weight = [](float x, float top) { return top == -INFINITY ? 0.f : expf(x - top); };
  for (int e = tid; e < heads * (p.dim / 4); e += kAttnWarps * 32) {
    const int h = e / (p.dim / 4), c = (e - h * (p.dim / 4)) * 4;
    float top = -INFINITY, sum = 0.f;
#pragma unroll
    for (int x = 0; x < kAttnWarps; ++x) top = fmaxf(top, s_stat[x][h].x);
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int x = 0; x < kAttnWarps; ++x) {
      const float f = weight(s_stat[x][h].x, top);
      const float4 u = *reinterpret_cast<const float4*>(&s_acc[x][h][c]);
      sum = fmaf(s_stat[x][h].y, f, sum);
      v.x = fmaf(u.x, f, v.x);
      v.y = fmaf(u.y, f, v.y);
      v.z = fmaf(u.z, f, v.z);
      v.w = fmaf(u.w, f, v.w);
    }
    if (ctas == 1) {
      const float inv = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
      T* o = out + h * p.out_head + c;
      o[0] = Num<T>::from_f(v.x * inv);
      o[1] = Num<T>::from_f(v.y * inv);
      o[2] = Num<T>::from_f(v.z * inv);
      o[3] = Num<T>::from_f(v.w * inv);
    } else {  // over Q, which nobody reads any more
      *reinterpret_cast<float4*>(&s_q[h][c]) = v;
    }
  }
  if (ctas == 1) return;
  __syncthreads();
  if (tid < heads) {  // the CTA's own, in the first warp's place
    float top = -INFINITY, sum = 0.f;
    for (int x = 0; x < kAttnWarps; ++x) top = fmaxf(top, s_stat[x][tid].x);
    for (int x = 0; x < kAttnWarps; ++x) sum = fmaf(s_stat[x][tid].y, weight(s_stat[x][tid].x, top), sum);
    s_stat[0][tid] = make_float2(top, sum);
  }
  cluster_arrive_release();
  cluster_wait_acquire();
  for (int e = tid * kAttnCtas + rank; e < heads * (p.dim / 4); e += kAttnWarps * 32 * kAttnCtas) {
    const int h = e / (p.dim / 4), c = (e - h * (p.dim / 4)) * 4;
    float2 stat[kAttnCtas];
    float4 u[kAttnCtas];
#pragma unroll
    for (int x = 0; x < kAttnCtas; ++x) {
      stat[x] = ld_dsmem_v2(cluster_map(smem_addr(&s_stat[0][h]), x));
      u[x] = ld_dsmem_v4(cluster_map(smem_addr(&s_q[h][c]), x));
    }
    float top = -INFINITY, sum = 0.f;
#pragma unroll
    for (int x = 0; x < kAttnCtas; ++x) top = fmaxf(top, stat[x].x);
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int x = 0; x < kAttnCtas; ++x) {
      const float f = weight(stat[x].x, top);
      sum = fmaf(stat[x].y, f, sum);
      v.x = fmaf(u[x].x, f, v.x);
      v.y = fmaf(u[x].y, f, v.y);
      v.z = fmaf(u[x].z, f, v.z);
      v.w = fmaf(u[x].w, f, v.w);
    }
    const float inv = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
    T* o = out + h * p.out_head + c;
    o[0] = Num<T>::from_f(v.x * inv);
    o[1] = Num<T>::from_f(v.y * inv);
    o[2] = Num<T>::from_f(v.z * inv);
    o[3] = Num<T>::from_f(v.w * inv);
  }
  cluster_arrive_release();  // no CTA leaves while another reads its sums
  cluster_wait_acquire();
}

namespace {
template <typename T, int V, int H, bool CODES>
cudaError_t general_h(const PagedAttnArgs& a, cudaStream_t st, bool pdl) {
  const int64_t items = (int64_t)a.tokens * a.kv_heads * ((a.group + H - 1) / H);
  // A cluster an item where there are fewer items than SMs, if the tables have room for enough keys; the
  // start of more clusters costs as much as more keys do. fp32, 32 query heads over 8 of 128, us with and without: 1
  // request (8 items) of 777 keys 15 and 35, 200 keys 12 and 10; 16 requests (128 items) of 2000 keys 101 and 135, 800
  // keys 95 and 68; 64 requests of 2000 keys 395 and 298.
  const bool few = items <= device_sm_count() && (int64_t)a.width * a.block_size > std::max<int64_t>(256, 8 * items);
  const int ctas = few ? kAttnCtas : 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(items * ctas));
  cfg.blockDim = dim3(kAttnWarps * 32);
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = pdl ? 1 : 0;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = ctas;
  at[1].val.clusterDim.y = 1;
  at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, paged_attention_general_kernel<T, V, H, CODES>, a, ctas);
}
template <typename T, bool CODES>
cudaError_t general_c(const PagedAttnArgs& a, bool vec, cudaStream_t st, bool pdl) {
  constexpr int V = 16 / (int)sizeof(T);
  if (a.group == 1) return vec ? general_h<T, V, 1, CODES>(a, st, pdl) : general_h<T, 1, 1, CODES>(a, st, pdl);
  return vec ? general_h<T, V, 4, CODES>(a, st, pdl) : general_h<T, 1, 4, CODES>(a, st, pdl);
}
template <typename T>
cudaError_t general_t(const PagedAttnArgs& a, bool vec, cudaStream_t st, bool pdl) {
  return a.k_scale != nullptr ? general_c<T, true>(a, vec, st, pdl) : general_c<T, false>(a, vec, st, pdl);
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
