// Attention over the paged cache for few query rows: decode steps and short drafts.
//
// The G = q_heads / kv_heads query heads of a key head and the request's new
// tokens form one block of rows (row r: token r / G, head r % G; at most 16: a
// tile of the warp-level tensor-core instruction, which more rows would pay for
// again, while csrc/paged_attn_tc.cu's do not: 64 requests x 2000 keys took 182 us
// here and 132 there with 32 and 36 rows). So K and V are read once for all of
// them. What bounds it is that read: R rows are R operations a byte. Everything
// else serves keeping loads in flight:
//   * a producer warp fetches tiles of 64 keys by TMA, one box of a page (the
//     largest power of two of slots that divides the block size, at most 64, by 64
//     columns) a lane, through a ring of stages of K and V; a box behind the keys
//     is a coordinate out of range, which reads zeros and no memory;
//   * four consumer warps take 16 of the 64 keys each and keep their own running
//     maximum, sum and 16 x D output sums over the whole item, with no exchange
//     between warps until its end. K's fragments are all loaded before the
//     products, which run as four chains, and V's are in flight during the
//     softmax: a warp that waited for each in turn took twice as long a tile.
//     Scores, sums and statistics are fp32. For the second product a
//     probability goes in as two terms, its rounding and the rounding's remainder (16 bits of
//     it in bf16, 21 in f16), since one term's 8 or 11 bits would add as much error as the result's own
//     rounding (f16: 1.2 times the whole error; 64 requests to 2048 keys 188 to 193 us
//     with one term, 190 to 206 with two). f16 has few exponents: P and its sum are taken times 2^15
//     (the largest P is 2^15), so that what is subnormal lies below 2^-29 of the largest and
//     not 2^-14: tens of thousands of small ones would be lost together;
//   * head_dims below 64 and between 64 and 128 run as these: the boxes' columns behind
//     them are zeros, and no memory;
//   * key tiles are dealt evenly over two CTAs an SM (paged_sched.cuh), or, for few
//     short requests, an item to a cluster.
// Keys that a row does not see may hold anything: scores are replaced, not added
// to, and since 0 * NaN is NaN the V fragments of keys outside [first, kv) are cleared
// before the product, and infinities and NaN of keys that only some rows see are
// taken out and added to these rows alone. Where the products made NaN of an infinity that
// a row does see, its output is settled after it was stored (paged_settle).
//
// Measured: 64 requests of 33 to 2048 keys, 32 heads of 128: 190 to 197 us, 5.4 to 5.6 TB/s (82 to 85 %
// of the measured copy bandwidth); 4 requests of 20000 to 65536 keys, 8 key heads:
// 115 us, 5.3 TB/s; one request of 777 keys: 6.5 us; 64 requests of 8192 keys with a window of
// 1000, 8 key heads: 60 us, 4.4 TB/s.
#include <climits>

#include "device.h"
#include "kernels.h"
#include "mma.cuh"
#include "paged_sched.cuh"
#include "paged_tma.h"
#include "tc.cuh"

namespace mlora {

constexpr int kDecTile = 64;  // keys a stage
constexpr int kDecJoin = 3;   // joining a piece costs about three tiles
constexpr int kDecItem = 3;   // and so does an item besides its tiles
using DecodeSplit = PagedSplit<kDecJoin, kDecItem>;

struct DecodeArgs {
  CUtensorMap k_map, v_map;
  PagedAttnArgs a;
  int box;     // rows of a TMA box
};

template <int D>
struct DecodeCfg {
  static constexpr int KG = 4;                    // key groups: warps that share 16 rows
  static constexpr int kWarps = KG;
  static constexpr int kThreads = kWarps * 32 + 32;
  static constexpr int kPerSm = 2;
  static constexpr int kSide = kDecTile * D * 2;  // bytes of K (or V) in a stage
  static constexpr int kStages = 96 * 1024 / (2 * kSide);
  static constexpr int kRowF = D + 4;             // floats of a row in the merge buffer
  static constexpr int kMerge = 16 * kRowF * 4;
  static constexpr int kSmem = kStages * 2 * kSide + kMerge + 1024;
};

// One item's description, the same in every warp.
struct DecodeItem {
  int req, head, q0, qn, kv, first, tile0, n;
};

__device__ __forceinline__ void decode_request(const PagedAttnArgs& p, DecodeItem& it, int req, const PagedRequest& r) {
  it.req = req;
  it.q0 = r.q0;
  it.qn = r.qn;
  it.kv = r.kv;
  it.first = paged_first_key(p, r.kv - r.qn);
  it.tile0 = it.first / kDecTile;
  it.n = r.qn > 0 && r.qn * p.group <= kDecodeMaxRows ? max(1, (r.kv + kDecTile - 1) / kDecTile - it.tile0) : 0;
}

constexpr int kFewCtas = 8;    // CTAs of a cluster
constexpr int kFewItems = 16;  // (request, key head)s that clusters are launched for, at most
constexpr int kFewKeys = 4096; // keys that the block tables have room for, at most

template <typename T, int D, bool CLUSTER>
__global__ void __launch_bounds__(DecodeCfg<D>::kThreads, DecodeCfg<D>::kPerSm)
paged_attention_decode_kernel(const __grid_constant__ DecodeArgs args) {
  using C = DecodeCfg<D>;
  constexpr float kUp = Num<T>::is_bf16 ? 0.f : 15.f;  // P is taken times 2^kUp
  constexpr int NS = C::kStages, SIDE = C::kSide, HALF = kDecTile * 128;
  extern __shared__ __align__(1024) unsigned char s_raw[];
  __shared__ __align__(8) uint64_t full[NS], empty[NS];
  __shared__ float s_m[C::kWarps][16], s_l[C::kWarps][16];
  __shared__ int s_last;
  __shared__ PagedPlace s_place;  // of the item that is being joined
  const PagedAttnArgs& p = args.a;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(s_raw) + 1023) & ~uintptr_t(1023));
  float* merge = reinterpret_cast<float*>(smem + NS * 2 * SIDE);
  const int group = p.group;

  if (tid == 0) {
    for (int s = 0; s < NS; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], C::kWarps);
    }
    fence_barrier_init();
  }
  if (warp == C::kWarps && lane == 0) {
    tma_prefetch_map(&args.k_map);
    tma_prefetch_map(&args.v_map);
  }
  pdl_wait();
  pdl_trigger();

  DecodeSplit split;
  DecodeItem it;
  int before, in_req;
  int req;
  PagedRequest found;
  const bool report = CLUSTER ? blockIdx.x % (kFewCtas * p.kv_heads) == 0 : blockIdx.x == 0;
  bool skipped = false;  // a request that is not computed
  auto units = [&](int i, int, int, PagedRequest& r) {
    r = paged_request(p, i, report);
    // rows beyond what the caller said: reported, and where they do not fit the tile not computed
    if (report && r.qn > p.max_q_len) flag_error(p.status, kErrLength);
    DecodeItem x;
    decode_request(p, x, i, r);
    skipped |= r.odd || (r.qn > 0 && x.n == 0);
    return x.n > 0 ? (x.n + kDecItem) * p.kv_heads : 0;
  };
  // CLUSTER: a cluster takes one item, each CTA an eighth of its tiles, and the sums
  // are joined over distributed shared memory, without a search and without the workspace.
  const int rank = blockIdx.x % kFewCtas;
  auto zero_others = [&]() {  // one warp: rows that are nobody's
    if constexpr (CLUSTER) {  // which has asked about its own request only (all of them at the start: 0.2 us more)
      static_assert(kFewItems <= 32, "a lane a request");
      PagedRequest r;
      if (lane < p.requests) units(lane, 0, 1, r);
      skipped = __any_sync(0xffffffffu, skipped);
    }
    if (skipped) paged_zero_uncomputed<T>(p, kDecodeMaxRows);
    else paged_zero_rest<T>(p);
  };
  if constexpr (CLUSTER) {
    const int item = blockIdx.x / kFewCtas;
    req = item / p.kv_heads;
    units(req, 0, 1, found);
    decode_request(p, it, req, found);
    if (it.n == 0) {  // the same in the whole cluster
      if (warp == C::kWarps) zero_others();
      return;
    }
    it.head = item - req * p.kv_heads;
    split.set(0, gridDim.x);
  } else {
    paged_find<C::kThreads, 1>(p.requests, units, split, req, found, before, in_req);
  }
  if constexpr (CLUSTER) __syncthreads();     // the barriers are initialised
  else skipped = __syncthreads_or(skipped);
  PagedCursor<DecodeSplit> cur(split);
  if constexpr (!CLUSTER) {
    if (cur.pos >= cur.end) {
      if (warp == C::kWarps) zero_others();
      return;
    }
    decode_request(p, it, req, found);
    it.head = (cur.pos - before) / (it.n + kDecItem);
    cur.unit = cur.pos - before - it.head * (it.n + kDecItem);
  }
  auto next_item = [&]() {
    if (++it.head == p.kv_heads) {
      it.head = 0;
      PagedRequest r;
      const int i = paged_next(p, it.req, kDecodeMaxRows, r);
      if (i < p.requests) decode_request(p, it, i, r);
    }
  };
  if (!CLUSTER && cur.begin(it.n)) next_item();
  bool begun = false;
  auto take = [&]() {  // this CTA's part of the current item
    if (!CLUSTER) return cur.take(it.n);
    cur.tile = rank * it.n / kFewCtas;
    cur.len = (rank + 1) * it.n / kFewCtas - cur.tile;
    const bool once = !begun;
    begun = true;
    return once;
  };
  auto advance = [&]() { return !CLUSTER && cur.advance(); };
  bool ok = true;

  if (warp == C::kWarps) {  // ---- producer ----
    const int boxes = kDecTile / args.box, jobs = boxes * (D / 64) * 2;
    const int b = lane % boxes, half = (lane / boxes) % (D / 64), side = lane / (boxes * (D / 64));
    int stage = 0, round = 0;
    while (take()) {
      const int32_t* table = p.tables + it.req * p.table_stride;
      for (int k = 0; k < cur.len; ++k) {
        const int j = (it.tile0 + cur.tile + k) * kDecTile + b * args.box;
        int block = (int)p.num_blocks, off = 0;  // out of range: zeros
        if (lane < jobs && j < it.kv && j + args.box > it.first) {
          const int e = __ldcg(table + j / p.block_size);
          off = j % p.block_size;
          if (e >= 0 && e < p.num_blocks) block = e;
          else flag_error(p.status, kErrKvRange);
        }
        if (round > 0) ok = __all_sync(0xffffffffu, ok && mbar_poll(&empty[stage], (round - 1) & 1, p.status));
        if (ok) {
          if (lane == 0) mbar_arrive_expect_tx(&full[stage], 2 * SIDE);
          __syncwarp();
          if (lane < jobs)
            tma_load_4d(smem + stage * 2 * SIDE + side * SIDE + half * HALF + b * args.box * 128,
                        side == 0 ? &args.k_map : &args.v_map, half * 64, off, it.head, block, &full[stage]);
        }
        if (++stage == NS) {
          stage = 0;
          ++round;
        }
      }
      if (advance()) next_item();
    }
    zero_others();
    if constexpr (CLUSTER) {  // with the consumers: sums written, sums read
      for (int i = 0; i < 2; ++i) {
        cluster_arrive_release();
        cluster_wait_acquire();
      }
    }
    return;
  }

  // ---- consumers: 16 rows, 16 keys of each tile a warp ----
  const int kg = warp;
  const float sl = p.scale * 1.4426950408889634f;  // scores in powers of two
  int stage = 0, phase = 0;
  bool ready = false;  // the next stage is known to be there
  uint32_t* tickets = static_cast<uint32_t*>(p.workspace);
  float* parts = reinterpret_cast<float*>(tickets + kPagedTickets);
  constexpr int PART = 16 * (D + 2);  // floats of a piece: sums, maxima, totals
  // Q fragments: rows lane / 4 and + 8, columns (lane % 4) * 2 (+ 8) of each 16
  uint32_t qf[D / 16][4];
  auto load_q = [&](const DecodeItem& x) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = (lane >> 2) + e * 8, t = paged_token(p, r);
      const T* src = static_cast<const T*>(p.q) + (int64_t)(x.q0 + t) * p.q_token +
                     (int64_t)(x.head * group + r - t * group) * p.q_head + (lane & 3) * 2;
      const bool real = r < x.qn * group;
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        qf[k][e] = real && k * 16 < p.dim ? __ldcg(reinterpret_cast<const unsigned int*>(src + k * 16)) : 0u;
        qf[k][2 + e] = real && k * 16 + 8 < p.dim ? __ldcg(reinterpret_cast<const unsigned int*>(src + k * 16 + 8)) : 0u;
      }
    }
  };
  bool more = take();
  if (more) load_q(it);
  while (more) {
    const int rows = it.qn * group;
    int limit[2], floor_[2];  // keys below `limit` and at or above `floor_` are seen
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = (lane >> 2) + e * 8;
      const int pq = it.kv - it.qn + paged_token(p, r);
      limit[e] = r < rows ? pq + 1 : 0;
      floor_[e] = paged_first_key(p, pq);
    }
    float o[D / 8][4];
#pragma unroll
    for (int n = 0; n < D / 8; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    const int all_end = it.kv - it.qn + 1, all_first = paged_first_key(p, it.kv - 1);  // keys that every row sees

    for (int k = 0; k < cur.len; ++k) {
      if (!ready) ok = ok && mbar_poll(&full[stage], phase, p.status);
      const int next = stage + 1 < NS ? stage + 1 : 0;
      ready = mbar_test(&full[next], next == 0 ? phase ^ 1 : phase);  // answered while this tile is worked on
      __syncwarp();
      const int k0 = kg * 16, j0 = (it.tile0 + cur.tile + k) * kDecTile + k0;  // 16 keys
      if (j0 < it.kv && j0 + 16 > it.first) {
        const uint32_t ks = smem_addr(smem + stage * 2 * SIDE), vs = ks + SIDE;
        // All of K's fragments, then the products as four independent chains.
        uint32_t kf[2][D / 32][4];
#pragma unroll
        for (int c = 0; c < D / 32; ++c)  // 32 columns: two k steps
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            const int key = k0 + n * 8 + (lane & 7), chunk = c * 4 + (lane >> 3);
            ldsm_x4(ks + (chunk >> 3) * HALF + key * 128 + (((chunk & 7) ^ (key & 7)) << 4), kf[n][c][0], kf[n][c][1],
                    kf[n][c][2], kf[n][c][3]);
          }
        float s4[2][2][4];
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) s4[n][0][e] = s4[n][1][e] = 0.f;
#pragma unroll
        for (int c = 0; c < D / 32; ++c)
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int n = 0; n < 2; ++n)
              mma_16816<T>(s4[n][h], qf[2 * c + h][0], qf[2 * c + h][1], qf[2 * c + h][2], qf[2 * c + h][3],
                           kf[n][c][2 * h], kf[n][c][2 * h + 1]);
        // V's fragments, in flight during the softmax: keys (lane % 4) * 2 + {0, 1} and + 8
        uint32_t vf[D / 16][4];
        auto load_v = [&]() {
          const int key = k0 + (lane & 15);
#pragma unroll
          for (int n = 0; n < D / 16; ++n) {  // 16 columns of V
            const int chunk = n * 2 + (lane >> 4);
            ldsm_x4_trans(vs + (chunk >> 3) * HALF + key * 128 + (((chunk & 7) ^ (key & 7)) << 4), vf[n][0], vf[n][1],
                          vf[n][2], vf[n][3]);
          }
        };
        load_v();
        float s[2][4];
        const bool edge = j0 + 16 > all_end || j0 < all_first;  // not all seen by all rows
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            s[n][e] = (s4[n][0][e] + s4[n][1][e]) * sl;
            if (edge) {
              const int j = j0 + n * 8 + (lane & 3) * 2 + (e & 1);
              if (j >= limit[e >> 1] || j < floor_[e >> 1]) s[n][e] = -INFINITY;
            }
          }
        uint32_t pf[4], pr[4];
        float fix[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float top = fmaxf(fmaxf(s[0][2 * e], s[0][2 * e + 1]), fmaxf(s[1][2 * e], s[1][2 * e + 1]));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
          const float m_new = fmaxf(m[e], top), ref = m_new == -INFINITY ? 0.f : m_new;
          fix[e] = exp2_fast(m[e] - ref);
          m[e] = m_new;
          const float base = ref - kUp;
          const float p0 = exp2_fast(s[0][2 * e] - base), p1 = exp2_fast(s[0][2 * e + 1] - base);
          const float p2 = exp2_fast(s[1][2 * e] - base), p3 = exp2_fast(s[1][2 * e + 1] - base);
          l[e] = l[e] * fix[e] + ((p0 + p1) + (p2 + p3));
          pf[e] = pack_round2<T>(p0, p1);
          pf[2 + e] = pack_round2<T>(p2, p3);
          pr[e] = pack_round2<T>(p0 - Pack2<T>::lo(pf[e]), p1 - Pack2<T>::hi(pf[e]));
          pr[2 + e] = pack_round2<T>(p2 - Pack2<T>::lo(pf[2 + e]), p3 - Pack2<T>::hi(pf[2 + e]));
        }
        if (__any_sync(0xffffffffu, fix[0] != 1.f || fix[1] != 1.f)) {
#pragma unroll
          for (int n = 0; n < D / 8; ++n) {
            o[n][0] *= fix[0];
            o[n][1] *= fix[0];
            o[n][2] *= fix[1];
            o[n][3] *= fix[1];
          }
        }
        if (j0 + 16 > it.kv || j0 < it.first) {
          const int j = j0 + (lane & 3) * 2;
          auto keep = [&](int x) { return x < it.kv && x >= it.first; };
          const uint32_t clear0 = (keep(j) ? 0xffffu : 0u) | (keep(j + 1) ? 0xffff0000u : 0u);
          const uint32_t clear1 = (keep(j + 8) ? 0xffffu : 0u) | (keep(j + 9) ? 0xffff0000u : 0u);
#pragma unroll
          for (int n = 0; n < D / 16; ++n) {
            vf[n][0] &= clear0;
            vf[n][1] &= clear1;
            vf[n][2] &= clear0;
            vf[n][3] &= clear1;
          }
        }
        if (edge && it.qn > 1) {
          uint32_t any = 0u;
#pragma unroll
          for (int n = 0; n < D / 16; ++n) 
#pragma unroll
            for (int e = 0; e < 4; ++e) any = paged_taint<T>(vf[n][e], any);
          if (__builtin_expect(__any_sync(0xffffffffu, any != 0u), 0)) {
#pragma unroll 1
            for (int i = 0; i < 16; ++i) {
              const int j = j0 + i, row = k0 + i;
#pragma unroll
              for (int n = 0; n < D / 8; ++n) {
                const uint32_t w = *reinterpret_cast<const uint32_t*>(smem + stage * 2 * SIDE + SIDE + (n >> 3) * HALF + row * 128 +
                                                                      (((n & 7) ^ (row & 7)) << 4) + (lane & 3) * 4);
                const float a = Pack2<T>::lo(w), b = Pack2<T>::hi(w);
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                  if (j >= limit[e] || j < floor_[e]) continue;
                  if (!isfinite(a)) o[n][2 * e] += a;
                  if (!isfinite(b)) o[n][2 * e + 1] += b;
                }
              }
            }
            __syncwarp();
#pragma unroll 1
            for (int i = lane; i < 16 * (D / 2); i += 32) {  // out of the stage, whose fragments are loaded again
              const int row = k0 + i / (D / 2), c = i % (D / 2);
              uint32_t* at = reinterpret_cast<uint32_t*>(smem + stage * 2 * SIDE + SIDE + (c >> 5) * HALF + row * 128 +
                                                         ((((c >> 2) & 7) ^ (row & 7)) << 4) + (c & 3) * 4);
              const int j = j0 + row - k0;
              *at = j < it.kv && j >= it.first ? paged_finite<T>(*at) : 0u;
            }
            fence_proxy_async_smem();
            __syncwarp();
            load_v();
          }
        }
#pragma unroll
        for (int n = 0; n < D / 16; ++n) {
          mma_16816<T>(o[2 * n], pf[0], pf[1], pf[2], pf[3], vf[n][0], vf[n][1]);
          mma_16816<T>(o[2 * n + 1], pf[0], pf[1], pf[2], pf[3], vf[n][2], vf[n][3]);
        }
#pragma unroll
        for (int n = 0; n < D / 16; ++n) {
          mma_16816<T>(o[2 * n], pr[0], pr[1], pr[2], pr[3], vf[n][0], vf[n][1]);
          mma_16816<T>(o[2 * n + 1], pr[0], pr[1], pr[2], pr[3], vf[n][2], vf[n][3]);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[stage]);
      stage = next;
      if (stage == 0) phase ^= 1;
    }

    // The next item's Q, in flight while this one is joined.
    const DecodeItem done = it;
    const bool begins = cur.unit == 0, whole = cur.whole(it.n);
    const int item0 = cur.pos - cur.unit;
    if (tid == 0) s_place = {done.req, done.head, done.kv, done.qn};
    more = advance();
    if (more) {
      next_item();
      more = take();
      if (more) load_q(it);
    }

    // ---- join the key groups of each 16 rows: `slots` of them lie side by side in the
    // merge buffer where the rows are few, further ones are added in turn ----
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      l[e] += __shfl_xor_sync(0xffffffffu, l[e], 1);
      l[e] += __shfl_xor_sync(0xffffffffu, l[e], 2);
      if ((lane & 3) == 0) {
        s_m[warp][(lane >> 2) + e * 8] = m[e];
        s_l[warp][(lane >> 2) + e * 8] = l[e];
      }
    }
    const int slots = rows <= 4 ? C::KG : rows <= 8 ? 2 : 1, apart = 16 / (rows <= 4 ? 4 : slots);
    named_barrier(1, C::kWarps * 32);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = (lane >> 2) + e * 8;
      float top = -INFINITY;
#pragma unroll
      for (int g = 0; g < C::KG; ++g) top = fmaxf(top, s_m[g][r]);
      const float own = top == -INFINITY ? 0.f : exp2_fast(m[e] - top);
#pragma unroll
      for (int n = 0; n < D / 8; ++n) {
        o[n][2 * e] *= own;
        o[n][2 * e + 1] *= own;
      }
    }
    for (int g = 0; g < C::KG; g += slots) {
      if (kg >= g && kg < g + slots) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int r = (lane >> 2) + e * 8;
          if (r >= rows) continue;
          float* d = merge + ((kg - g) * apart + r) * C::kRowF + (lane & 3) * 2;
          if (g > 0) {
            float2 u[D / 8];  // all the loads first
#pragma unroll
            for (int n = 0; n < D / 8; ++n) u[n] = *reinterpret_cast<const float2*>(d + n * 8);
#pragma unroll
            for (int n = 0; n < D / 8; ++n) {
              o[n][2 * e] += u[n].x;
              o[n][2 * e + 1] += u[n].y;
            }
          }
#pragma unroll
          for (int n = 0; n < D / 8; ++n)
            *reinterpret_cast<float2*>(d + n * 8) = make_float2(o[n][2 * e], o[n][2 * e + 1]);
        }
      }
      named_barrier(1, C::kWarps * 32);
    }
    auto row_stat = [&](int r, float& top, float& sum) {  // over the key groups of row r
      top = s_m[0][r];
#pragma unroll
      for (int g = 1; g < C::KG; ++g) top = fmaxf(top, s_m[g][r]);
      sum = 0.f;
#pragma unroll
      for (int g = 0; g < C::KG; ++g) sum += top == -INFINITY ? 0.f : s_l[g][r] * exp2_fast(s_m[g][r] - top);
    };
    auto place = [&](int r, int c) {
      const int t = paged_token(p, r);
      return static_cast<T*>(p.out) + (int64_t)(done.q0 + t) * p.out_token +
             (int64_t)(done.head * group + r - t * group) * p.out_head + c;
    };
    auto store = [&](int r, int c, const float* v, float inv) {  // 8 columns of row r; whether they may need settle()
      if (c >= p.dim) return false;
      uint4 u;
      u.x = pack_round2<T>(v[0] * inv, v[1] * inv);
      u.y = pack_round2<T>(v[2] * inv, v[3] * inv);
      u.z = pack_round2<T>(v[4] * inv, v[5] * inv);
      u.w = pack_round2<T>(v[6] * inv, v[7] * inv);
      *reinterpret_cast<uint4*>(place(r, c)) = u;
      return inv == inv && paged_taint<T>(u.w, paged_taint<T>(u.z, paged_taint<T>(u.y, paged_taint<T>(u.x, 0u)))) != 0u;
    };
    // What a lane stored in columns from c of row r where it is not finite, though the row's sum is: the whole warp.
    auto settle = [&](auto words, int r, int c, bool odd) {
      if (__builtin_expect(__any_sync(0xffffffffu, odd), 0)) {
        paged_settle<T, decltype(words)::value>(p, &s_place, r, c, place(r, c), odd);
      }
    };
    // Where the sums go that are not finished here: a piece of the workspace, or for the
    // cluster the ring of stages, which is empty now.
    float* part = CLUSTER ? reinterpret_cast<float*>(smem) : parts + ((long long)blockIdx.x * 2 + (begins ? 1 : 0)) * PART;
    for (int e0 = 0; e0 < rows * (D / 8); e0 += C::kWarps * 32) {
      const int e = e0 + tid, r = e / (D / 8), c = (e % (D / 8)) * 8;
      bool odd = false;
      if (e < rows * (D / 8)) {
        float top, sum;
        row_stat(r, top, sum);
        float4 v0 = *reinterpret_cast<const float4*>(merge + r * C::kRowF + c);
        float4 v1 = *reinterpret_cast<const float4*>(merge + r * C::kRowF + c + 4);
        for (int g = 1; g < slots; ++g) {
          const float4 u0 = *reinterpret_cast<const float4*>(merge + (r + g * apart) * C::kRowF + c);
          const float4 u1 = *reinterpret_cast<const float4*>(merge + (r + g * apart) * C::kRowF + c + 4);
          v0.x += u0.x;
          v0.y += u0.y;
          v0.z += u0.z;
          v0.w += u0.w;
          v1.x += u1.x;
          v1.y += u1.y;
          v1.z += u1.z;
          v1.w += u1.w;
        }
        if (CLUSTER) {
          *reinterpret_cast<float4*>(part + r * D + c) = v0;
          *reinterpret_cast<float4*>(part + r * D + c + 4) = v1;
          if (c == 0) reinterpret_cast<float2*>(part + 16 * D)[r] = make_float2(top, sum);
        } else if (whole) {
          const float v[8] = {v0.x, v0.y, v0.z, v0.w, v1.x, v1.y, v1.z, v1.w};
          odd = store(r, c, v, sum > 0.f || sum != sum ? 1.f / sum : 0.f);
        } else {
          __stcg(reinterpret_cast<float4*>(part + r * D + c), v0);
          __stcg(reinterpret_cast<float4*>(part + r * D + c + 4), v1);
          if (c == 0) __stcg(reinterpret_cast<float2*>(part + 16 * D) + r, make_float2(top, sum));
        }
      }
      if (!CLUSTER) settle(std::integral_constant<int, 4>(), r, c, odd);
    }
    if constexpr (CLUSTER) {
      cluster_arrive_release();
      cluster_wait_acquire();
      const uint32_t base = smem_addr(part);
      const int e = tid * kFewCtas + rank, row = e / (D / 4), c = (e % (D / 4)) * 4;
      static_assert(16 * (D / 4) <= C::kWarps * 32 * kFewCtas, "a thread has one piece of the output");
      bool odd = false;
      if (e < rows * (D / 4) && c < p.dim) {
        float4 u[kFewCtas];
        float2 stat[kFewCtas];
#pragma unroll
        for (int x = 0; x < kFewCtas; ++x) {
          u[x] = ld_dsmem_v4(cluster_map(base + (row * D + c) * 4, x));
          stat[x] = ld_dsmem_v2(cluster_map(base + (16 * D + row * 2) * 4, x));
        }
        float top = stat[0].x, sum = 0.f;
#pragma unroll
        for (int x = 1; x < kFewCtas; ++x) top = fmaxf(top, stat[x].x);
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int x = 0; x < kFewCtas; ++x) {
          const float w = top == -INFINITY ? 0.f : exp2_fast(stat[x].x - top);
          sum = fmaf(stat[x].y, w, sum);
          v.x = fmaf(u[x].x, w, v.x);
          v.y = fmaf(u[x].y, w, v.y);
          v.z = fmaf(u[x].z, w, v.z);
          v.w = fmaf(u[x].w, w, v.w);
        }
        const float inv = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
        const uint2 w = make_uint2(pack_round2<T>(v.x * inv, v.y * inv), pack_round2<T>(v.z * inv, v.w * inv));
        *reinterpret_cast<uint2*>(place(row, c)) = w;
        odd = inv == inv && paged_taint<T>(w.y, paged_taint<T>(w.x, 0u)) != 0u;
      }
      settle(std::integral_constant<int, 2>(), row, c, odd);
      cluster_arrive_release();  // no CTA leaves while another reads its sums
      cluster_wait_acquire();
      return;
    }
    if (!whole) {
      const int c0 = split.first_cta(item0, done.n), c1 = split.last_cta(item0, done.n);
      const PagedJoin run(c0, c1, blockIdx.x);
      auto piece = [&](int c) { return parts + ((long long)c * 2 + (c == c0 ? 1 : 0)) * PART; };
      auto last_of = [&](uint32_t* ticket, int n) {  // whether this CTA is the last of n to get here
        named_barrier(1, C::kWarps * 32);
        if (tid == 0) {
          __threadfence();
          const bool last = atomicAdd(ticket, 1u) == (uint32_t)(n - 1);
          if (last) *ticket = 0u;
          __threadfence();
          s_last = last;
        }
        named_barrier(1, C::kWarps * 32);
        return s_last != 0;
      };
      // Pieces x0, x0 + by, .. x1, to the output or as one piece to x0's place.
      auto join = [&](int x0, int x1, int by, bool final) {
        for (int e0 = 0; e0 < rows * (D / 8); e0 += C::kWarps * 32) {
          const int e = e0 + tid, r = e / (D / 8), c = (e % (D / 8)) * 8;
          const bool real = e < rows * (D / 8);
          float top = -INFINITY, sum = 0.f, v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
          bool odd = false;
          if (real) {
#pragma unroll 8
            for (int x = x0; x <= x1; x += by) {
              const float* src = piece(x);
              const float2 stat = __ldcg(reinterpret_cast<const float2*>(src + 16 * D) + r);
              const float4 v0 = __ldcg(reinterpret_cast<const float4*>(src + r * D + c));
              const float4 v1 = __ldcg(reinterpret_cast<const float4*>(src + r * D + c + 4));
              const float m_new = fmaxf(top, stat.x), ref = m_new == -INFINITY ? 0.f : m_new;
              const float fix = exp2_fast(top - ref), w = exp2_fast(stat.x - ref);
              top = m_new;
              sum = fmaf(sum, fix, stat.y * w);
              v[0] = fmaf(v[0], fix, v0.x * w);
              v[1] = fmaf(v[1], fix, v0.y * w);
              v[2] = fmaf(v[2], fix, v0.z * w);
              v[3] = fmaf(v[3], fix, v0.w * w);
              v[4] = fmaf(v[4], fix, v1.x * w);
              v[5] = fmaf(v[5], fix, v1.y * w);
              v[6] = fmaf(v[6], fix, v1.z * w);
              v[7] = fmaf(v[7], fix, v1.w * w);
            }
            if (final) {
              odd = store(r, c, v, sum > 0.f || sum != sum ? 1.f / sum : 0.f);
            } else {
              __stcg(reinterpret_cast<float4*>(piece(x0) + r * D + c), make_float4(v[0], v[1], v[2], v[3]));
              __stcg(reinterpret_cast<float4*>(piece(x0) + r * D + c + 4), make_float4(v[4], v[5], v[6], v[7]));
            }
          }
          if (final) settle(std::integral_constant<int, 4>(), r, c, odd);
          if (!final) {  // a row's threads are in one turn: 128 is a multiple of D / 8
            named_barrier(1, C::kWarps * 32);
            if (real && c == 0) __stcg(reinterpret_cast<float2*>(piece(x0) + 16 * D) + r, make_float2(top, sum));
          }
        }
      };
      uint32_t* run_ticket = tickets + gridDim.x + run.x0 * 2 + (run.x0 == c0 ? 1 : 0);
      if (run.runs == 1) {
        if (last_of(tickets + c0, c1 - c0 + 1)) join(c0, c1, 1, true);
      } else if (last_of(run_ticket, run.x1 - run.x0 + 1)) {
        join(run.x0, run.x1, 1, false);
        if (last_of(tickets + c0, run.runs)) join(c0, c1, run.by, true);
      }
    }
    named_barrier(1, C::kWarps * 32);  // the merge buffer and s_last are free again
  }
}

namespace {

template <typename T, int D, bool CLUSTER>
cudaError_t launch_decode(const DecodeArgs& a, cudaStream_t st, bool pdl) {
  using C = DecodeCfg<D>;
  auto kern = paged_attention_decode_kernel<T, D, CLUSTER>;
  static SmemLimit limit;
  if (const cudaError_t e = limit.raise(kern, C::kSmem); e != cudaSuccess) return e;
  const int ctas = device_sm_count() * C::kPerSm;
  static_assert(C::kSmem <= 227 * 1024, "shared memory");
  if (ctas * 3 > kPagedTickets ||
      (size_t)ctas * 2 * 16 * (D + 2) * 4 + kPagedTickets * 4 > kPagedWorkspaceBytes)
    return cudaErrorNotSupported;
  if constexpr (!CLUSTER) {
    return launch_kernel(kern, dim3(ctas), dim3(C::kThreads), C::kSmem, st, pdl, a);
  } else {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(a.a.requests * a.a.kv_heads * kFewCtas));
    cfg.blockDim = dim3(C::kThreads);
    cfg.dynamicSmemBytes = C::kSmem;
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = kFewCtas;
    at[0].val.clusterDim.y = 1;
    at[0].val.clusterDim.z = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = pdl ? 1 : 0;
    cfg.attrs = at;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, kern, a);
  }
}

template <typename T, int D>
cudaError_t launch_decode_any(const DecodeArgs& a, cudaStream_t st, bool pdl) {
  // One request of 777 keys, 8 key heads: 6.5 us with clusters, 11.3 without; 4000 keys 12.9 and 18.5. From
  // twice that on an item needs more CTAs than a cluster has. The host knows the lengths' bound only.
  // Without requests there is no item to launch a cluster for: the other kernel's CTAs write the zeros.
  if (a.a.requests > 0 && (long long)a.a.requests * a.a.kv_heads <= kFewItems &&
      (long long)a.a.width * a.a.block_size <= kFewKeys)
    return launch_decode<T, D, true>(a, st, pdl);
  return launch_decode<T, D, false>(a, st, pdl);
}

}  // namespace

cudaError_t launch_paged_attention_decode(const PagedAttnArgs& a, int dtype, cudaStream_t st, bool pdl) {
  if ((dtype != kBF16 && dtype != kF16) || a.dim > 128) return cudaErrorNotSupported;
  // units of work (paged_sched.cuh) in 32 bits
  if ((long long)a.requests * a.kv_heads * ((long long)a.width * a.block_size / kDecTile + 2 + kDecItem) >= INT_MAX)
    return cudaErrorNotSupported;
  DecodeArgs d{};
  d.a = a;
  d.box = paged_box(a.block_size, kDecTile);
  if (d.box < 8 || !paged_maps(a, dtype, d.box, &d.k_map, &d.v_map)) return cudaErrorNotSupported;
  if (dtype == kBF16)
    return a.dim <= 64 ? launch_decode_any<__nv_bfloat16, 64>(d, st, pdl) : launch_decode_any<__nv_bfloat16, 128>(d, st, pdl);
  return a.dim <= 64 ? launch_decode_any<__half, 64>(d, st, pdl) : launch_decode_any<__half, 128>(d, st, pdl);
}

}  // namespace mlora
