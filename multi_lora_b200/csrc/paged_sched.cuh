// What the paged attention kernels share: a request's lengths with their
// checks, the split of all key tiles over the CTAs, and the tensor maps' limits.
//
// The work of a launch is a sequence of items (request, key head, and for long
// chunks a tile of query rows), each a run of key tiles. CTA c of G takes the
// c-th G-th of all tiles, wherever item boundaries fall: every CTA reads the
// same number of keys whatever the lengths are, and a single long request spreads over the
// whole GPU. An item inside one CTA is finished there; of an item that
// several CTAs share each writes its unnormalised sums, maximum and total to
// the workspace, and the CTA that counts itself last (of a run of CTAs, then of the
// runs, where they are many) joins them in CTA order, the same every time, so the bits are too. A CTA has at most two such
// pieces: the rest of an item that an earlier CTA began (slot 0), and the
// beginning of one that a later CTA ends (slot 1).
#pragma once

#include <climits>
#include <type_traits>

#include "common.cuh"
#include "paged.h"
#include "tma.cuh"

namespace mlora {

// A value that every lane has, as one that the compiler knows to be uniform.
template <typename V>
__device__ __forceinline__ V same_in_warp(V v) {
  return __shfl_sync(0xffffffffu, v, 0);
}

struct PagedRequest {
  int q0, qn, kv;  // first row, rows, keys
  bool odd;        // offsets that make no sense (no rows then)
};

__device__ __forceinline__ PagedRequest paged_request(const PagedAttnArgs& p, int i, bool report) {
  PagedRequest r;
  r.q0 = __ldcg(p.q_indptr + i);
  const int q1 = __ldcg(p.q_indptr + i + 1);
  r.kv = __ldcg(p.kv_lens + i);
  r.qn = q1 - r.q0;
  r.odd = r.q0 < 0 || q1 < r.q0 || q1 > p.tokens;
  if (r.odd) {
    if (report) flag_error(p.status, kErrIndptr);
    r.q0 = r.qn = 0;
  }
  const long long cap = (long long)p.width * p.block_size;
  if (r.kv < 0 || r.kv > cap) {
    if (report) flag_error(p.status, kErrLength);
    r.kv = r.kv < 0 ? 0 : (int)cap;
  }
  return r;
}

// Token of a row (row / group).
__device__ __forceinline__ int paged_token(const PagedAttnArgs& p, int row) {
  return p.group_magic != 0 ? (int)__umulhi((uint32_t)row, p.group_magic) : row;
}

// First key that query row `pos` of a request sees.
__device__ __forceinline__ int paged_first_key(const PagedAttnArgs& p, int pos) {
  return p.window > 0 ? max(0, pos - p.window + 1) : 0;
}

// The even split over the CTAs, in units of a key tile's time (the caller sees to
// it that their sum stays below 2^31). An item of n tiles
// counts n + C units: C for what it costs besides its tiles (its Q, its join or
// its output), so that many short items weigh what they take. Boundaries that fall
// within T units of an item's edge move to that edge: joining a piece costs about as much as T
// tiles, so no piece is shorter than that, and short items stay whole.
template <int T_MOST, int C>
struct PagedSplit {
  static constexpr int kItem = C;
  int total, base, rem;        // CTA c has base units, the first `rem` CTAs one more
  int T;                       // T_MOST, or less where the CTAs have less to do than that
  __device__ void set(int units, int ctas) {
    if (units == INT_MAX) units = 0;  // see paged_sum
    total = units;
    base = units / ctas;
    rem = units - base * ctas;
    T = min(T_MOST, base);
  }
  __device__ int start(int c) const { return c * base + min(c, rem); }
  __device__ int owner(int unit) const {
    const int wide = rem * (base + 1);
    return unit < wide ? unit / (base + 1) : rem + (unit - wide) / base;
  }
  // Boundaries up to here into an item of n tiles go to its beginning (all those
  // within the C units among them: no piece is without tiles), others to its end or stay.
  __device__ int low(int n) const { return max(C, min(T + C, (n + C) / 2)); }
  __device__ int snap(int x, int n) const { return x >= n + C ? n + C : x <= low(n) ? 0 : n + C - x <= T ? n + C : x; }
  // The CTAs that share an item of n tiles beginning at unit `item`; more than one of them.
  __device__ int first_cta(int item, int n) const { return owner(item + low(n)); }
  __device__ int last_cta(int item, int n) const { return owner(item + n + C - T - 1); }
};

// A CTA's way through its units: the current item begins at `pos - unit`, and the
// CTA's part of it is the tiles [tile, tile + len).
template <typename S>
struct PagedCursor {
  const S& split;
  int pos, end;
  int unit, tile, len, step;
  __device__ explicit PagedCursor(const S& s)
      : split(s), pos(s.start(blockIdx.x)), end(s.start(blockIdx.x + 1)), unit(0), tile(0), len(0), step(0) {}
  // The CTA's part of an item of n tiles; false: nothing is left for it.
  __device__ __forceinline__ bool take(int n) {
    if (pos >= end) return false;
    const int stop = split.snap(end - (pos - unit), n);
    step = stop - unit;
    tile = unit == 0 ? 0 : unit - S::kItem;
    len = stop - S::kItem - tile;
    return step > 0;
  }
  __device__ __forceinline__ bool whole(int n) const { return unit == 0 && step == n + S::kItem; }
  // Past that part; true when the next item has to be looked up.
  __device__ __forceinline__ bool advance() {
    pos += step;
    unit = 0;
    return pos < end;
  }
  // The first boundary, `unit` units into an item of n tiles; true as for advance.
  __device__ __forceinline__ bool begin(int n) {
    const int at = split.snap(unit, n);
    pos += at - unit;
    unit = at;
    if (at < n + S::kItem) return false;
    unit = 0;
    return pos < split.total;
  }
};

// Sums of units stop at INT_MAX. The caller keeps the sum over requests that share no rows below it; offsets that go back
// and forth may give the same rows to many requests, and their work may pass it: then nothing is computed.
__device__ __forceinline__ int paged_sum(int a, int b) { return (int)min((unsigned)a + (unsigned)b, (unsigned)INT_MAX); }

// Whole block of NT threads: the split over the grid, the request that this CTA's first
// unit lies in with its lengths, the units before that request and in it.
// `units(i, part, parts, r)`: the units of request i (its lengths go to r), or one of
// `parts` parts of them (a request's items dealt out; up to MAX_PARTS threads
// count for one request when there are few).
template <int MAX_PARTS, typename F, typename S>
__device__ __forceinline__ void paged_find_warp(int requests, F units, S& split, int& req, PagedRequest& found,
                                                int& before, int& in_req) {
  const int lane = threadIdx.x & 31;
  int parts = 1;
  while (parts < MAX_PARTS && 2 * parts * requests <= 32) parts *= 2;
  const int i = lane / parts, part = lane & (parts - 1);
  PagedRequest last = {0, 0, 0, false};
  const int mine = i < requests ? units(i, part, parts, last) : 0;
  int incl = mine, all_parts = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl = paged_sum(incl, u);
    const int w = __shfl_xor_sync(0xffffffffu, all_parts, o);
    if (o < parts) all_parts = paged_sum(all_parts, w);
  }
  split.set(__shfl_sync(0xffffffffu, incl, 31), gridDim.x);
  const int a = split.start(blockIdx.x), upto = incl - mine;
  const unsigned hit = __ballot_sync(0xffffffffu, part == 0 && a >= upto && a < upto + all_parts);
  const int src = hit != 0u ? __ffs(hit) - 1 : 0;
  req = __shfl_sync(0xffffffffu, i, src);
  before = __shfl_sync(0xffffffffu, upto, src);
  in_req = __shfl_sync(0xffffffffu, all_parts, src);
  found.q0 = __shfl_sync(0xffffffffu, last.q0, src);
  found.qn = __shfl_sync(0xffffffffu, last.qn, src);
  found.kv = __shfl_sync(0xffffffffu, last.kv, src);
}

// What its threads tell one another, in shared memory.
template <int NT>
struct PagedFindRoom {
  int warp[NT / 32];
  int before, sum, req;
  PagedRequest found;
};

template <int NT, int MAX_PARTS, typename F, typename S>
__device__ __forceinline__ void paged_find_in(PagedFindRoom<NT>& room, int requests, F units, S& split, int& req,
                                              PagedRequest& found, int& before, int& in_req) {
  if (requests <= 32) {  // every warp for itself, without a barrier
    paged_find_warp<MAX_PARTS>(requests, units, split, req, found, before, in_req);
    return;
  }
  PagedRequest last = {0, 0, 0, false};
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int parts = 1;
  while (parts < MAX_PARTS && 2 * parts * requests <= NT) parts *= 2;
  const int per = (requests * parts + NT - 1) / NT;  // 1 when parts > 1
  const int r0 = min(requests, parts > 1 ? tid / parts : tid * per), r1 = min(requests, r0 + per);
  const int part = tid & (parts - 1);
  int mine = 0;
  for (int i = r0; i < r1; ++i) mine = paged_sum(mine, units(i, part, parts, last));
  int incl = mine, all_parts = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl = paged_sum(incl, u);
    const int w = __shfl_xor_sync(0xffffffffu, all_parts, o);
    if (o < parts) all_parts = paged_sum(all_parts, w);
  }
  if (lane == 31) room.warp[warp] = incl;
  if (tid == 0) room.req = requests;
  __syncthreads();
  int total = 0, upto = incl - mine;
#pragma unroll
  for (int w = 0; w < NT / 32; ++w) {
    const int u = room.warp[w];
    upto += w < warp ? u : 0;
    total = paged_sum(total, u);
  }
  split.set(same_in_warp(total), gridDim.x);
  const int a = split.start(blockIdx.x);
  if (part == 0 && a >= upto && a < upto + all_parts) {
    int i = r0;
    if (per > 1) {
      for (all_parts = units(i, 0, 1, last); a >= upto + all_parts && i + 1 < r1; all_parts = units(++i, 0, 1, last))
        upto += all_parts;
    }
    room.req = i;
    room.before = upto;
    room.sum = all_parts;
    room.found = last;
  }
  __syncthreads();
  req = same_in_warp(room.req);
  before = same_in_warp(room.before);
  in_req = same_in_warp(room.sum);
  found.q0 = same_in_warp(room.found.q0);
  found.qn = same_in_warp(room.found.qn);
  found.kv = same_in_warp(room.found.kv);
}

template <int NT, int MAX_PARTS, typename F, typename S>
__device__ __forceinline__ void paged_find(int requests, F units, S& split, int& req, PagedRequest& found,
                                           int& before, int& in_req) {
  __shared__ PagedFindRoom<NT> room;
  paged_find_in<NT, MAX_PARTS>(room, requests, units, split, req, found, before, in_req);
}

// The first request from i on with rows, at most `most` of them (tokens x group), in the rare case that there
// is none among the 32 before: 128 at once, which are one round trip to L2.
__device__ __forceinline__ int paged_skip_idle(const PagedAttnArgs& p, int i, int most) {
  constexpr int AT_ONCE = 4;
  const int lane = threadIdx.x & 31;
#pragma unroll 1
  for (int i0 = i; i0 < p.requests; i0 += 32 * AT_ONCE) {
    int q0[AT_ONCE], q1[AT_ONCE];
#pragma unroll
    for (int k = 0; k < AT_ONCE; ++k) {
      const int at = min(i0 + k * 32 + lane, p.requests - 1);  // the last one again, rather than one behind it
      q0[k] = __ldcg(p.q_indptr + at);
      q1[k] = __ldcg(p.q_indptr + at + 1);
    }
#pragma unroll
    for (int k = 0; k < AT_ONCE; ++k) {
      const bool has = q0[k] >= 0 && q1[k] > q0[k] && q1[k] <= p.tokens && (q1[k] - q0[k]) * p.group <= most;
      const unsigned hit = __ballot_sync(0xffffffffu, has);
      if (hit != 0u) return min(i0 + k * 32 + __ffs(hit) - 1, p.requests - 1);
    }
  }
  return p.requests;
}
// The next request after i with rows (as above) and its lengths, p.requests if there is none: the whole warp. Idle
// requests may be many: a cache plans all that it has room for at every step.
__device__ __forceinline__ int paged_next(const PagedAttnArgs& p, int i, int most, PagedRequest& r) {
  const int at = i + 1 + (threadIdx.x & 31);
  r = {0, 0, 0, false};
  if (at < p.requests) r = paged_request(p, at, false);
  const unsigned hit = __ballot_sync(0xffffffffu, r.qn > 0 && r.qn * p.group <= most);
  if (__builtin_expect(hit == 0u, 0)) {
    i = paged_skip_idle(p, i + 33, most);
    if (i < p.requests) r = paged_request(p, i, false);
    return i;
  }
  const int src = __ffs(hit) - 1;
  r.q0 = __shfl_sync(0xffffffffu, r.q0, src);
  r.qn = __shfl_sync(0xffffffffu, r.qn, src);
  r.kv = __shfl_sync(0xffffffffu, r.kv, src);
  return i + 1 + src;
}

// Rows behind the last request's give zeros; one warp of every CTA takes a share.
template <typename T>
__device__ __forceinline__ void paged_zero_rest(const PagedAttnArgs& p) {
  const int last = p.requests > 0 ? __ldcg(p.q_indptr + p.requests) : 0;
  if (last < 0 || last >= p.tokens) return;
  const int64_t pieces = p.dim / 8, n = (int64_t)(p.tokens - last) * p.q_heads * pieces;
  for (int64_t e = (int64_t)blockIdx.x * 32 + (threadIdx.x & 31); e < n; e += (int64_t)gridDim.x * 32) {
    const int64_t row = e / pieces;
    T* o = static_cast<T*>(p.out) + (last + row / p.q_heads) * p.out_token + (row % p.q_heads) * p.out_head +
           (e % pieces) * 8;
    *reinterpret_cast<uint4*>(o) = make_uint4(0, 0, 0, 0);
  }
}

// Zeros in every row that no request has, where some requests are not computed: their offsets make no sense, or they have
// more rows (tokens x group) than `most`. One warp of every CTA takes a share. Only for calls that
// report an error, so simple: each row asks all requests.
template <typename T>
__device__ __noinline__ void paged_zero_uncomputed(const PagedAttnArgs& p, int most) {
  const int lane = threadIdx.x & 31, pieces = p.q_heads * (p.dim / 8);
  for (int t = blockIdx.x; t < p.tokens; t += gridDim.x) {
    bool computed = false;
    for (int i0 = 0; i0 < p.requests && !computed; i0 += 32) {
      PagedRequest r = {0, 0, 0, true};
      if (i0 + lane < p.requests) r = paged_request(p, i0 + lane, false);
      computed = __any_sync(0xffffffffu, t >= r.q0 && t < r.q0 + r.qn && r.qn * p.group <= most);
    }
    if (computed) continue;
    T* row = static_cast<T*>(p.out) + t * p.out_token;
    for (int e = lane; e < pieces; e += 32)
      *reinterpret_cast<uint4*>(row + e / (p.dim / 8) * p.out_head + e % (p.dim / 8) * 8) = make_uint4(0, 0, 0, 0);
  }
}

// Infinities and NaN in pairs of 16-bit values: fma(w, 0, seen) stays zero while everything is finite.
template <typename T>
__device__ __forceinline__ uint32_t paged_taint(uint32_t w, uint32_t seen) {
  if constexpr (Num<T>::is_bf16) asm("fma.rn.bf16x2 %0, %1, %2, %0;" : "+r"(seen) : "r"(w), "r"(0u));
  else asm("fma.rn.f16x2 %0, %1, %2, %0;" : "+r"(seen) : "r"(w), "r"(0u));
  return seen;
}
// The pair with zeros in their place.
template <typename T>
__device__ __forceinline__ uint32_t paged_finite(uint32_t w) {
  constexpr uint32_t kExp = Num<T>::is_bf16 ? 0x7f807f80u : 0x7c007c00u, kOne = Num<T>::is_bf16 ? 0x00800080u : 0x04000400u;
  return w & ~(((((w & kExp) + kOne) & 0x80008000u) >> 15) * 0xffffu);  // a carry where all exponent bits are set
}

// Outputs that are NaN although the sum of their P is a number: V is not finite at a key that they see. P is
// positive, so what is right there is the sum of V's infinities and NaN in that column; but a P that is zero in the type
// of its product, or whose second term is zero or negative, makes a NaN of an infinity. Whole warp: the
// 2 W columns from c of a lane's row lie at dst, and `mine` says that they may
// be such outputs. The lanes look at 128 keys at once and tell one another what is not finite. Seldom run: the
// keys are read again, about 1.5 us for 128 of them and 2 W columns.
// The request and key head wait in shared memory, not in registers that the tiles need.
struct PagedPlace {
  int req, head, kv, qn;
};
template <typename T, int W>
__device__ __noinline__ void paged_settle(const PagedAttnArgs& p, const PagedPlace* at, int row, int c, T* dst, bool mine) {
  const int req = at->req, head = at->head;
  const int pos = at->kv - at->qn + paged_token(p, row), first = paged_first_key(p, pos), limit = pos + 1;
  using Words = typename std::conditional<W == 4, uint4, uint2>::type;
  constexpr int AT_ONCE = 4;
  union Pieces {
    Words all;
    uint32_t w[W];
  };
  const int lane = threadIdx.x & 31;
  Pieces o;
  uint32_t nans = 0u;  // a bit a column
#pragma unroll
  for (int i = 0; i < W; ++i) o.w[i] = 0u;
  if (mine) {
    o.all = *reinterpret_cast<const Words*>(dst);
#pragma unroll
    for (int i = 0; i < W; ++i) {
      if (isnan(Pack2<T>::lo(o.w[i]))) nans |= 1u << (2 * i);
      if (isnan(Pack2<T>::hi(o.w[i]))) nans |= 2u << (2 * i);
    }
  }
  unsigned todo = __ballot_sync(0xffffffffu, nans != 0u);
  while (todo != 0u) {
    const int col = __shfl_sync(0xffffffffu, c, __ffs(todo) - 1);
    const bool with = nans != 0u && c == col;
    const int from = __reduce_min_sync(0xffffffffu, with ? first : INT_MAX);
    const int to = __reduce_max_sync(0xffffffffu, with ? limit : 0);
    const T* base = static_cast<const T*>(p.v) + head * p.v_head + col;
    const int32_t* table = p.tables + req * p.table_stride;
    float sum[2 * W];
#pragma unroll
    for (int i = 0; i < 2 * W; ++i) sum[i] = 0.f;
    bool open = true;  // some column may still change: a NaN stays one
#pragma unroll 1
    for (int j0 = from; open && j0 < to; j0 += 32 * AT_ONCE) {
      Pieces v[AT_ONCE];
      uint32_t odd[AT_ONCE];
#pragma unroll
      for (int k = 0; k < AT_ONCE; ++k) {
        const int j = j0 + k * 32 + lane;
#pragma unroll
        for (int i = 0; i < W; ++i) v[k].w[i] = 0u;
        if (j < to) {
          const int block = __ldcg(table + j / p.block_size);
          if (block >= 0 && block < p.num_blocks)
            v[k].all = __ldcg(reinterpret_cast<const Words*>(base + block * p.v_block + (j % p.block_size) * p.v_slot));
        }
      }
      unsigned any = 0u;
#pragma unroll
      for (int k = 0; k < AT_ONCE; ++k) {
        uint32_t seen = 0u;
#pragma unroll
        for (int i = 0; i < W; ++i) seen = paged_taint<T>(v[k].w[i], seen);
        odd[k] = __ballot_sync(0xffffffffu, seen != 0u);
        any |= odd[k];
      }
      if (any == 0u) continue;
#pragma unroll
      for (int k = 0; k < AT_ONCE; ++k)
        for (unsigned left = odd[k]; left != 0u; left &= left - 1u) {
          const int from_lane = __ffs(left) - 1, j = j0 + k * 32 + from_lane;
          const bool sees = with && j >= first && j < limit;
#pragma unroll
          for (int i = 0; i < W; ++i) {
            const uint32_t x = __shfl_sync(0xffffffffu, v[k].w[i], from_lane);
            const float a = Pack2<T>::lo(x), b = Pack2<T>::hi(x);
            if (sees && !isfinite(a)) sum[2 * i] += a;
            if (sees && !isfinite(b)) sum[2 * i + 1] += b;
          }
        }
      bool mine_open = false;
#pragma unroll
      for (int i = 0; i < 2 * W; ++i) mine_open |= (nans >> i & 1u) != 0u && !isnan(sum[i]);
      open = __any_sync(0xffffffffu, with && mine_open);
    }
    if (with) {
#pragma unroll
      for (int i = 0; i < W; ++i) {  // a NaN without such a value stays
        const float a = (nans >> (2 * i) & 1u) != 0u && sum[2 * i] != 0.f ? sum[2 * i] : Pack2<T>::lo(o.w[i]);
        const float b = (nans >> (2 * i) & 2u) != 0u && sum[2 * i + 1] != 0.f ? sum[2 * i + 1] : Pack2<T>::hi(o.w[i]);
        o.w[i] = pack_round2<T>(a, b);
      }
      *reinterpret_cast<Words*>(dst) = o.all;
    }
    todo &= ~__ballot_sync(0xffffffffu, with);
  }
}

// 2^x on the special function unit; 0 for -infinity.
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Whether phase `parity` of `bar` has completed, without waiting (try_wait may suspend the thread).
__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(done)
      : "r"(smem_addr(bar)), "r"(parity)
      : "memory");
  return done != 0;
}

// Bounded wait like mbar_wait, for barriers on the critical path: the timer (a read of
// it takes longer than most waits) is asked every 128th poll only.
__device__ __forceinline__ bool mbar_poll(uint64_t* bar, uint32_t parity, uint32_t* status) {
  uint64_t t0 = 0;
  for (uint32_t i = 1; !mbar_try_wait(bar, parity); ++i) {
    if ((i & 127u) == 0) {
      const uint64_t t = global_timer_ns();
      if (t0 == 0) t0 = t;
      if (t - t0 > kWaitLimitNs) {
        flag_error(status, kErrTimeout);
        return false;
      }
    }
  }
  return true;
}

// A count in shared memory that one warp raises and others wait for.
__device__ __forceinline__ void count_store(uint32_t* at, uint32_t n) {
  asm volatile("st.release.cta.shared::cta.u32 [%0], %1;" ::"r"(smem_addr(at)), "r"(n) : "memory");
}
__device__ __forceinline__ bool count_poll(uint32_t* at, uint32_t n, uint32_t* status) {
  uint64_t t0 = 0;
  for (uint32_t i = 1;; ++i) {
    uint32_t now;
    asm volatile("ld.acquire.cta.shared::cta.u32 %0, [%1];" : "=r"(now) : "r"(smem_addr(at)) : "memory");
    if (now >= n) return true;
    if ((i & 127u) == 0) {
      const uint64_t t = global_timer_ns();
      if (t0 == 0) t0 = t;
      if (t - t0 > kWaitLimitNs) {
        flag_error(status, kErrTimeout);
        return false;
      }
    }
  }
}

// 32 bytes at once (one sector).
__device__ __forceinline__ void store32(void* p, const uint32_t (&r)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(r[0]), "r"(r[1]), "r"(r[2]),
               "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}

// The pieces of an item that CTAs c0 .. c1 share are joined in two stages where they are many: runs of
// `by` CTAs first, by the last of each run to arrive, and then their results, by the last of those.
// One CTA that reads all of them is most of the launch otherwise: 70 rows over 32000 keys
// of one head, 95 pieces of 36 KB, 105 us and 48 in two stages; one row over 60000 keys
// of one head, 296 pieces of 0.5 KB, 49 us and 25.
struct PagedJoin {
  int by, x0, x1, runs;  // this CTA's run, and how many there are
  __device__ PagedJoin(int c0, int c1, int cta) {
    const int n = c1 - c0 + 1;
    by = n;
    if (n > 6) {
      by = 3;
      while (by * by < n) ++by;
    }
    x0 = c0 + (cta - c0) / by * by;
    x1 = min(x0 + by - 1, c1);
    runs = (n + by - 1) / by;
  }
};

constexpr int kPagedTickets = 1024;  // words at the start of the workspace, zero between calls
constexpr size_t kPagedWorkspaceBytes = (size_t)64 << 20;
// As many more at its end, for a launch with more CTAs than those have room for.
__device__ __forceinline__ uint32_t* paged_more_tickets(const PagedAttnArgs& p) {
  return reinterpret_cast<uint32_t*>(static_cast<unsigned char*>(p.workspace) + kPagedWorkspaceBytes) - kPagedTickets;
}

}  // namespace mlora
