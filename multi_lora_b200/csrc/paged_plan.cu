// Block tables, slots and positions of one step, from the requests' lengths.
//
// Request i has ctx_i tokens in the cache, gets new_i more and holds held_i
// blocks of B slots. With W the width of a table row:
//   want_i  = min(ceil((ctx_i + new_i) / B), W)
//   grant_i = max(want_i - held_i, 0), cut off in request order where the free
//             list ends
//   table[i, held_i + j] = free[head + sum_{k<i} grant_k + j],  j < grant_i
//   token t of request i: position p = ctx_i + t, slot = table[i, p / B] * B + p % B
//
// The work is a few thousand integers, so latency is all there is: one launch,
// and no grid-wide barrier. Every CTA scans all requests for itself (the
// lengths come from L2; both prefix sums ride in one 64-bit scan), keeps the
// prefixes in shared memory, and then takes its share of the tokens and of the
// granted blocks, each found by binary search. A token's block comes from the
// old part of its table row or straight from the free list, never from an
// entry that this launch writes. held_out and free_head_out may be the inputs'
// own memory: the CTA that counts itself last (every other one has read its
// inputs by then) writes them.
//
// Measured: 64 requests of one token 3.5 us, 256 requests with 131000 tokens 5.2 us
// (1.0 MB written), of which an empty launch is about 2.5.
//
// The kernel never triggers dependent launches: kernels that follow may read
// q_indptr as segment routing before their own wait.
#include <climits>

#include "common.cuh"
#include "device.h"
#include "kernels.h"
#include "paged.h"

namespace mlora {

constexpr int kPlanNT = 512;

struct PlanRow {
  int ctx, held, tok, first;  // tokens and granted blocks before this request
};

// Inclusive scan of one 64-bit value a thread over the block; `total` is the sum.
__device__ __forceinline__ unsigned long long plan_scan(unsigned long long v, unsigned long long* s_warp,
                                                        unsigned long long& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned long long u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  if (lane == 31) s_warp[warp] = v;
  __syncthreads();
  unsigned long long before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kPlanNT / 32; ++w) {
    const unsigned long long u = s_warp[w];
    before += w < warp ? u : 0;
    all += u;
  }
  total = all;
  __syncthreads();
  return v + before;
}

// Last row whose prefix (`tok` or `first`) is <= x; rows that add nothing are stepped over.
template <bool TOKENS>
__device__ __forceinline__ int plan_find(const PlanRow* rows, int n, int x) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int m = (lo + hi + 1) >> 1;
    if ((TOKENS ? rows[m].tok : rows[m].first) <= x) lo = m;
    else hi = m - 1;
  }
  return lo;
}

__global__ void __launch_bounds__(kPlanNT) paged_plan_kernel(const PlanArgs p) {
  extern __shared__ __align__(16) unsigned char s_dyn[];
  PlanRow* rows = reinterpret_cast<PlanRow*>(s_dyn);
  __shared__ unsigned long long s_warp[kPlanNT / 32];
  __shared__ bool s_last;
  const int tid = threadIdx.x;
  const bool reporter = blockIdx.x == 0;
  pdl_wait();

  int head = __ldcg(p.free_head);
  uint32_t err = 0;
  if (head < 0 || head > p.num_free) {
    err |= kErrLength;
    head = head < 0 ? 0 : p.num_free;
  }
  const long long avail = p.num_free - head;
  unsigned long long base = 0;  // tokens << 32 | wanted blocks before this pass (their sums fit 32 bits each)
  for (int r0 = 0; r0 < p.requests; r0 += kPlanNT) {
    const int i = r0 + tid;
    int ctx = 0, fresh = 0, held = 0, want = 0;
    if (i < p.requests) {
      ctx = __ldcg(p.ctx_lens + i);
      fresh = __ldcg(p.new_lens + i);
      held = __ldcg(p.held + i);
      if (ctx < 0 || fresh < 0 || held < 0 || held > p.width) {
        err |= kErrLength;
        ctx = max(ctx, 0);
        fresh = max(fresh, 0);
        held = min(max(held, 0), p.width);
      }
      const long long end = (long long)ctx + fresh;
      const long long blocks = (end + p.block - 1) / p.block;
      if (blocks > p.width || end > INT_MAX) err |= kErrLength;
      want = max((int)min(blocks, (long long)p.width) - held, 0);
    }
    unsigned long long all;
    const uint32_t counted = (uint32_t)min((long long)fresh, p.max_tokens + 1ll);
    const unsigned long long mine = ((unsigned long long)counted << 32) | (uint32_t)want;
    const unsigned long long before = base + plan_scan(mine, s_warp, all) - mine;
    base += all;
    if (i < p.requests) {
      PlanRow r;
      r.ctx = ctx;
      r.held = held;
      r.tok = (int)min((unsigned long long)p.max_tokens, before >> 32);
      r.first = (int)min((long long)(before & 0xffffffffu), avail);
      rows[i] = r;
      if ((long long)(before & 0xffffffffu) + want > avail) err |= kErrExhausted;
      if (reporter) {
        p.kv_lens[i] = (int)min((long long)ctx + fresh, (long long)INT_MAX);
        p.q_indptr[i] = r.tok;
      }
    }
  }
  const int tokens = (int)min((unsigned long long)p.max_tokens, base >> 32);
  const int granted = (int)min((long long)(base & 0xffffffffu), avail);
  if (base >> 32 > (unsigned long long)p.max_tokens) err |= kErrLength;
  if (reporter) {
    if (tid == 0) p.q_indptr[p.requests] = tokens;
    if (err != 0) flag_error(p.status, err);
  }
  if (tid == 0) {
    PlanRow end;
    end.ctx = end.held = 0;
    end.tok = tokens;
    end.first = granted;
    rows[p.requests] = end;
  }
  __syncthreads();  // every read of held and free_head by this CTA is done
  if (tid == 0) {
    s_last = true;
    if (gridDim.x > 1) {
      __threadfence();
      s_last = atomicAdd(p.ticket, 1u) == gridDim.x - 1;
      if (s_last) *p.ticket = 0u;
    }
  }

  const int step = gridDim.x * kPlanNT, at = blockIdx.x * kPlanNT + tid;
  for (int t = at; t < p.max_tokens; t += step) {
    uint32_t pos = 0;  // below 2^32: a context length plus a token index
    int slot = -1;
    if (t < tokens) {
      const int i = plan_find<true>(rows, p.requests, t);
      const PlanRow r = rows[i];
      const uint32_t holds = r.held + rows[i + 1].first - r.first;
      pos = (uint32_t)r.ctx + (uint32_t)(t - r.tok);
      const uint32_t page = pos / (uint32_t)p.block;
      if (page < holds) {
        const int b = page < (uint32_t)r.held ? __ldcg(p.tables + i * p.table_stride + page)
                                              : __ldg(p.free_blocks + head + r.first + (page - r.held));
        const long long s = (long long)b * p.block + (pos - page * p.block);
        slot = b >= 0 && s <= INT_MAX ? (int)s : -1;
      }
    }
    p.positions[t] = (int)min(pos, (uint32_t)INT_MAX);
    p.slot_map[t] = slot;
  }
  for (int g = at; g < granted; g += step) {
    const int i = plan_find<false>(rows, p.requests, g);
    p.tables[i * p.table_stride + rows[i].held + (g - rows[i].first)] = __ldg(p.free_blocks + head + g);
  }
  __syncthreads();
  if (s_last) {
    for (int i = tid; i < p.requests; i += kPlanNT) p.held_out[i] = rows[i].held + rows[i + 1].first - rows[i].first;
    if (tid == 0) *p.free_head_out = head + granted;
  }
}

cudaError_t launch_paged_plan(const PlanArgs& a, cudaStream_t st, bool pdl) {
  const int smem = (a.requests + 1) * (int)sizeof(PlanRow);
  static SmemLimit limit;
  const cudaError_t e = limit.raise(paged_plan_kernel, (kPlanMaxRequests + 1) * (int)sizeof(PlanRow));
  if (e != cudaSuccess) return e;
  // one CTA where the tokens fit it (no count of CTAs needed), at most one an SM else
  const long long work = a.max_tokens > a.requests ? a.max_tokens : a.requests;
  long long grid = (work + 2 * kPlanNT - 1) / (2 * kPlanNT);
  grid = grid < 1 ? 1 : grid > 148 ? 148 : grid;
  return launch_kernel(paged_plan_kernel, dim3((unsigned)grid), dim3(kPlanNT), (size_t)smem, st, pdl, a);
}

}  // namespace mlora
