// Attention of new tokens over a paged 16-bit cache on the 5th-generation tensor
// cores (function and arguments: paged.cuh).
//
// Work.  A unit is (request, kv head, q-block); a q-block is one (kFew: requests
// of at most 128 query rows) or two tiles of 128 query rows, each holding
// floor(128 / group) tokens x group heads.  Its visible keys are cut into tiles,
// and the tiles of all units, in order, are divided over the workers by the
// host, so a worker streams whole units except at its two ends; the pieces of
// a divided unit are written unnormalised in fp32 and combined by a dependent
// launch in worker order (no atomics: the result does not depend on timing).
//
// A worker is one CTA, or (D 256, two row tiles) a pair of CTAs with one row tile
// each: the pair's products are issued once for 256 rows (cta_group::2), and
// each CTA fetches half of every K and V tile.  One CTA alone would need 63
// bytes per cycle of K and V to keep its tensor pipe busy, and TMA brings an SM
// at most 46 (measured on resident data); it also leaves room for 2.5 tiles of K
// and V instead of 1.25 beside the queries.
//
// Measured (Hq 24 / Hk 4 / D 256, bf16): kFew, 8 x 4 tokens on 24580: 131 us, 6.1
// TB/s (0.94 of the measured copy); 8192 tokens on 17448: 1.95-2.03 ms, 1330-1380
// TFLOP/s (0.98-1.02 of the sustained library rate, at the power cap's clock).
//
// Bounds.  kFew: HBM; the keys stream through shared memory once, 64-key tiles,
// and the products of 128 padded rows take half of the time their bytes do
// (mma.sync on the live rows took more: its operand reads alone filled the
// shared-memory bandwidth that the copies leave).  Else D 256: the tensor pipe;
// D <= 128: the softmax warps, which read each score twice (at D 128 a tile takes
// 4100 cycles, while its products and its 2 x 128 x 128 exponentials, 16 per cycle,
// take 2048 each; 8192 tokens on 17448: 1.21 ms at D 128, 1.10 ms at D 64).
//
// Tile.  Jobs alternate between two score buffers: with one row tile per CTA job j
// is key tile j, with two it is key tile j / 2 of row tile j % 2.  The MMA warp
// issues S(0), S(1), then per job O += P(j) V as soon as P(j) is written and
// S(j + 2), so while the softmax of one job runs the tensor pipe has the other
// job's products.
//   TMEM columns: S[0] [0, 128), S[1] [128, 256), O [256, 512) (one row tile) or
//   O[0] [256, 256 + D), O[1] [384, 384 + D).  P(j) (16 bit) replaces the first
//   half of S(j)'s columns and is the A operand of P V; rows lie on lanes, one
//   query row per softmax thread, so row maxima and sums stay in a thread.
//   S = Q K^T : A = Q, B = K, both shared memory, K-major, 128-byte swizzle.
//   O += P V  : A = P in tensor memory, B = V, MN-major, 128-byte swizzle.
// The running maximum moves only when a score exceeds it by kPgHeadroom (log2
// units); then the thread rescales its row of O in tensor memory.  P is rounded to
// the values' type (the product takes one type), at most 2^-8 (bf16) or 2^-11 of
// each probability and averaged by the sum over keys: the result's error against
// 64 bits is 0.0023 relative (bf16), 0.0017 being its own rounding.  The row sums
// take P as it was before.
//
// Warps: 4 softmax per row tile, one MMA issuer, two TMA producers (K and Q; V)
// that fill one ring of slots in the order the MMAs use them, in boxes of 64
// dims x a power of two of tokens.  Each role is a short loop: unrolled over a
// row or a tile they overran the instruction cache (4.0 against 2.85 ms for 8192
// queries on 17448 keys).  Every wait is bounded; a time-out sets the CTA's abort
// flag and drains.
#pragma once

#include <climits>

#include "paged.cuh"

namespace oscar {

constexpr int kPcRows = 128;   // rows of a row tile
constexpr int kPcCtas = 192;   // workers of a plan
constexpr int kPcMerge = 4;    // warps that combine a row of many pieces

struct PcStart {
  int r, h, qb, t;  // plan index, kv head, q-block, first key tile
};
struct PcPlan {
  int num_req, ctas, tokens;  // workers; tokens per row tile
  int box_tokens;             // tokens per query load: kFew: the most that a request has, else `tokens`
  int req_id[kPgReqs], q_start[kPgReqs], q_len[kPgReqs], seq[kPgReqs];
  PcStart start[kPcCtas];
  int tiles[kPcCtas];  // key tiles of each worker
  int first[kPcCtas];  // tiles before it
};
struct PcSplit {
  int r, h, qb, c0, c1;  // a divided unit and its workers
};
struct PcSplits {
  int n;
  PcSplit unit[kPcCtas];
};

template <int D, bool kFew>
struct PcShape {
  static constexpr bool kPair = D == 256 && !kFew;      // a worker is a pair of CTAs
  static constexpr int kUnit = kFew ? 1 : 2;            // row tiles of a unit
  static constexpr int kM = kPair ? 1 : kUnit;          // row tiles per CTA
  static constexpr int kTile = kFew ? kPgKeys : 128;    // keys per tile
  static constexpr int kPanels = D / 64;                // 64-dim panels
  static constexpr int kKeys = kPair ? 64 : kTile;      // keys of a K tile in this CTA
  static constexpr int kVPanels = kPair ? 2 : kPanels;  // panels of a V tile in this CTA
  static constexpr int kSlot = kKeys * D * 2;           // a K tile or a V tile
  static constexpr int kSlots = kFew ? (D == 256 ? 5 : D == 128 ? 12 : 16) : (D == 64 ? 8 : 5);
  static constexpr int kSoftWarps = 4 * kM;
  static constexpr int kThreads = 32 * (kSoftWarps + 3);
};

template <int D, bool kFew>
struct PcSmem {
  using S = PcShape<D, kFew>;
  uint8_t q[S::kM][S::kPanels][kPcRows * 128];  // [row tile][panel][row][128 bytes], swizzled
  uint8_t ring[S::kSlots][S::kSlot];            // K: [panel][key][128 bytes]; V: [panel][key][128 bytes]
  // full, q_full, p_full: of a pair, the first CTA's are used by both
  unsigned long long full[S::kSlots], empty[S::kSlots];
  unsigned long long q_full, q_empty, s_full[2], p_full[2], o_done[2], tail, end;
  // what this CTA has announced on the barriers above: the latest ring position of each slot (-1: none)
  // and the number of units whose queries it has
  int at[S::kSlots], units;
  uint32_t tmem;
  int abort;
};

OSCAR_DEVINL uint64_t pc_desc(uint32_t addr, uint32_t lbo, uint32_t sbo) {
  return tc::smem_desc(addr, lbo, sbo) | (2ull << 61);  // 128-byte swizzle
}

OSCAR_DEVINL void prefetch_map(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];\n" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory");
}
OSCAR_DEVINL void tma_load_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];\n" ::"r"(
          dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar)
      : "memory");
}

// key tiles that q-block qb of a request sees (at least 1, so that empty rows are written)
template <typename Shape>
__host__ __device__ inline int pc_tiles(int q_len, int seq, int tokens, int qb) {
  const int64_t last = (int64_t)(qb + 1) * tokens * Shape::kUnit;
  const int visible = seq - q_len + (int)(last < q_len ? last : q_len);
  return visible > Shape::kTile ? (visible + Shape::kTile - 1) / Shape::kTile : 1;
}

// Ring position of key tile t's K and V (n tiles in the worker's stream).  S runs two jobs ahead of
// O: with two row tiles K0 V0 K1 V1 .., with one K0 K1 V0 K2 V1 .. K(n-1) V(n-2) V(n-1).
template <int kM>
OSCAR_DEVINL int pc_k_at(int t) {
  return kM == 1 ? (t == 0 ? 0 : 2 * t - 1) : 2 * t;
}
template <int kM>
OSCAR_DEVINL int pc_v_at(int t, int n) {
  return kM == 1 ? (t == n - 1 ? 2 * n - 1 : 2 * t + 2) : 2 * t + 1;
}

// The two CTAs of a pair
OSCAR_DEVINL uint32_t pc_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;\n" : "=r"(r));
  return r;
}
OSCAR_DEVINL uint32_t pc_map(uint32_t addr, uint32_t rank) {  // the same shared address in CTA `rank` of the cluster
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(a) : "r"(addr), "r"(rank));
  return a;
}
OSCAR_DEVINL void pc_cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}
// (kWrites: the arrival publishes this thread's shared-memory writes to the other CTA.  Arrivals for
// tensor memory that tcgen05.wait has completed need no release beyond the CTA, and one at cluster
// scope takes 800 cycles)
template <bool kWrites>
OSCAR_DEVINL void pc_arrive(uint32_t cluster_addr) {
  if constexpr (kWrites)
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];\n" ::"r"(cluster_addr) : "memory");
  else
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];\n" ::"r"(cluster_addr) : "memory");
}
OSCAR_DEVINL void pc_expect(uint32_t cluster_addr, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cluster.b64 _, [%0], %1;\n" ::"r"(cluster_addr),
               "r"(bytes)
               : "memory");
}
template <bool kPair>
OSCAR_DEVINL void pc_commit(uint32_t bar) {  // pair: the barrier of both CTAs
  if constexpr (kPair) {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n" ::"r"(bar),
        "h"((uint16_t)3)
        : "memory");
  } else {
    tc::mma_commit(bar);
  }
}
template <bool kPair>
OSCAR_DEVINL void pc_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  if constexpr (kPair) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
  } else {
    tc::mma_ss(d, a, b, idesc, acc);
  }
}
template <bool kPair>
OSCAR_DEVINL void pc_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  if constexpr (kPair) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n tcgen05.mma.cta_group::2.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
  } else {
    tc::mma_ts(d, a, b, idesc, acc);
  }
}
// TMA loads into this CTA that count on a barrier of either CTA of the pair
template <bool kPair>
OSCAR_DEVINL void pc_load_4d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, int w, uint32_t bar) {
  if constexpr (kPair) {
    asm volatile(
        "cp.async.bulk.tensor.4d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, "
        "%5}], [%6];\n" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar)
        : "memory");
  } else {
    tma_load_4d(dst, map, x, y, z, w, bar);
  }
}
template <bool kPair>
OSCAR_DEVINL void pc_load_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
  if constexpr (kPair) {
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, "
        "%4}], [%5];\n" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar)
        : "memory");
  } else {
    tma_load_3d(dst, map, x, y, z, bar);
  }
}

// Sets the abort flag of the pair's other CTA, whose waits then return soon too
OSCAR_DEVINL void pc_abort(uint32_t cluster_addr) {
  asm volatile("st.shared::cluster.u32 [%0], %1;\n" ::"r"(cluster_addr), "r"(1) : "memory");
}
OSCAR_DEVINL int pc_peek(uint32_t cluster_addr) {
  int v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];\n" : "=r"(v) : "r"(cluster_addr) : "memory");
  return v;
}

// After an abort, by a warp of the CTA that owns `full` and `q_full`, once every producer has stopped:
// waits for the copies that still write shared memory.  A slot is announced again only after its last
// phase was consumed, so at most the phase of the latest position is open; where only one CTA of a pair
// has announced it, the other one's arrival is made up for, so that the phase ends with the bytes.
// (V tiles that are completed by hand count on `tail`, which their producer has drained.)
template <bool kPair, int kSlots, typename Smem>
OSCAR_DEVINL void pc_drain_loads(Smem& sm, int lane) {
  if (lane > kSlots) return;
  const bool is_q = lane == kSlots;
  int* const mine = is_q ? &sm.units : &sm.at[lane];
  const uint32_t bar = is_q ? smem_u32(&sm.q_full) : smem_u32(&sm.full[lane]);
  int n = *reinterpret_cast<volatile int*>(mine);
  if constexpr (kPair) {
    const int theirs = pc_peek(pc_map(smem_u32(mine), 1));
    if (theirs != n) {
      tc::mbar_arrive(bar);
      n = max(n, theirs);
    }
  }
  if (is_q ? n > 0 : n >= 0) pg_drain(bar, (is_q ? n - 1 : n / kSlots) & 1);
}

// The pieces of units of one worker, walked alike by every role.
template <typename Shape>
struct PcWalk {
  const PcPlan& p;
  int r, h, qb, t, left;
  int nt, t_end, piece;  // of the current piece
  OSCAR_DEVINL PcWalk(const PcPlan& plan, int c)
      : p(plan), r(plan.start[c].r), h(plan.start[c].h), qb(plan.start[c].qb), t(plan.start[c].t), left(plan.tiles[c]), piece(0) {
    open();
  }
  OSCAR_DEVINL void open() {
    if (left <= 0) return;
    nt = pc_tiles<Shape>(p.q_len[r], p.seq[r], p.tokens, qb);
    t_end = min(nt, t + left);
  }
  OSCAR_DEVINL bool live() const { return left > 0; }
  OSCAR_DEVINL void next(int hk) {
    left -= t_end - t;
    t = 0;
    ++piece;
    const int per = p.tokens * Shape::kUnit;
    if (++qb >= (p.q_len[r] + per - 1) / per) {
      qb = 0;
      if (++h >= hk) {
        h = 0;
        ++r;
      }
    }
    open();
  }
};

OSCAR_DEVINL float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;\n" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

template <typename T> OSCAR_DEVINL uint32_t pc_pack(float lo, float hi);
template <> OSCAR_DEVINL uint32_t pc_pack<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <> OSCAR_DEVINL uint32_t pc_pack<__half>(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// x[k] of lane 8 g + i <-> x[i] of lane 8 g + k (16-byte pieces), in three exchanges
OSCAR_DEVINL void pc_transpose8(uint32_t (&x)[8][4], int lane) {
#pragma unroll
  for (int bit = 1; bit < 8; bit <<= 1) {
    const bool up = lane & bit;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if (k & bit) continue;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        // the lane keeps the piece whose index has its own bit and sends the other one
        const uint32_t give = up ? x[k][i] : x[k | bit][i];
        const uint32_t got = __shfl_xor_sync(0xffffffffu, give, bit);
        if (up) x[k][i] = got;
        else x[k | bit][i] = got;
      }
    }
  }
}
template <int D, typename T, bool kFew>
__global__ void __launch_bounds__(PcShape<D, kFew>::kThreads, 1)
paged_attn_tc_kernel(const __grid_constant__ PagedArgs a, const __grid_constant__ PcPlan p,
                   const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                   const __grid_constant__ CUtensorMap vmap) {
  using Shape = PcShape<D, kFew>;
  constexpr bool kPair = Shape::kPair;
  constexpr int kM = Shape::kM, kPanels = Shape::kPanels, kSlots = Shape::kSlots, kTile = Shape::kTile;
  constexpr int kMma = Shape::kSoftWarps;
  constexpr int kColO = 256;
  extern __shared__ __align__(1024) uint8_t pc_raw[];
  PcSmem<D, kFew>& sm = *reinterpret_cast<PcSmem<D, kFew>*>(pc_raw);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t rank = kPair ? pc_rank() : 0u;
  const int worker = kPair ? (int)blockIdx.x / 2 : (int)blockIdx.x;
  pdl_release();
  if (tid < 3) prefetch_map(tid == 0 ? &qmap : tid == 1 ? &kmap : &vmap);
  auto full = [&](int i) { return smem_u32(&sm.full[i]); };
  auto empty = [&](int i) { return smem_u32(&sm.empty[i]); };
  // a barrier that the pair's first CTA owns, for arrivals and loads
  auto lead = [&](uint32_t bar) { return kPair ? pc_map(bar, 0) : bar; };
  if (warp == kMma) {
    if (lane == 0) {
      constexpr int kCtas = kPair ? 2 : 1;
      for (int i = 0; i < kSlots; ++i) {
        tc::mbar_init(full(i), kCtas);  // each CTA's producer announces its own bytes
        tc::mbar_init(empty(i), 1);
      }
      for (int i = 0; i < 2; ++i) {
        tc::mbar_init(smem_u32(&sm.s_full[i]), 1);
        tc::mbar_init(smem_u32(&sm.p_full[i]), 4 * kCtas);  // a warp's rows each
        tc::mbar_init(smem_u32(&sm.o_done[i]), 1);
      }
      tc::mbar_init(smem_u32(&sm.q_full), kCtas);
      tc::mbar_init(smem_u32(&sm.q_empty), 1);
      tc::mbar_init(smem_u32(&sm.tail), 1);
      tc::mbar_init(smem_u32(&sm.end), 1);
      for (int i = 0; i < kSlots; ++i) sm.at[i] = -1;
      sm.units = 0;
      sm.abort = 0;
      tc::mbar_fence_init();
    }
    __syncwarp();
    if constexpr (kPair) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;\n" ::"r"(smem_u32(&sm.tmem)) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;\n" ::);
    } else {
      tc::tmem_alloc(smem_u32(&sm.tmem), 512);
      tc::tmem_relinquish();
    }
  }
  if constexpr (kFew) {
    // rows that no query load reaches are zero: their scores and probabilities then are too, and the
    // padded products switch nothing (the copies alone draw 950 of the card's 1000 W)
    for (int i = tid; i < (int)sizeof(sm.q) / 16; i += Shape::kThreads) reinterpret_cast<uint4*>(sm.q)[i] = make_uint4(0, 0, 0, 0);
    tc::fence_async_smem();
  }
  tc::tc_fence_before();
  if constexpr (kPair) pc_cluster_sync();  // the other CTA's barriers are initialised
  else __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = sm.tmem;
  auto wait = [&](uint32_t bar, uint32_t parity) -> bool {  // warp-uniform
    const bool ok = pg_wait(sm.abort, bar, parity, a.tries);
    if (kPair && !ok) pc_abort(pc_map(smem_u32(&sm.abort), rank ^ 1));  // (it cannot end before this warp does)
    return __all_sync(0xffffffffu, ok);
  };
  PcWalk<Shape> w(p, worker);  // (the plan is an argument)
  const int n_tiles = w.left;
  [[maybe_unused]] const int tile0 = p.first[worker];
  pdl_wait();

  if (warp < kMma) {
    // ================= softmax: thread = query row of row tile `wg`
    const int wg = warp / 4, row = tid & 127;
    const int rt = kPair ? (int)rank : wg;  // row tile of the unit
    const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
    const int rows = p.tokens * a.group;  // live rows of a row tile
    int job = kM == 2 ? wg : 0;           // jobs are numbered over the whole CTA
    const float scale = a.scale_log2;
    bool ok = true;
    for (; w.live() && ok; w.next(a.hk)) {
      const int q_len = p.q_len[w.r], seq = p.seq[w.r];
      const int tok = (w.qb * Shape::kUnit + rt) * p.tokens + row / a.group;
      const bool live = row < rows && tok < q_len;
      // visible keys; rows that hold no query are computed as they come and not written
      const int lim = live ? max(0, seq - q_len + tok + 1) : INT_MAX;
      const bool busy = __any_sync(0xffffffffu, live);
      float m = -INFINITY;
      uint64_t l2 = 0;  // two partial sums
      const uint32_t o_col = tmem + lanes + kColO + (kM == 2 ? 128 * wg : 0);
#pragma unroll 1
      for (int t = w.t; t < w.t_end; ++t, job += kM) {
        const int b = job & 1;
        const uint32_t s_col = tmem + lanes + 128 * b;
        if (!wait(smem_u32(&sm.s_full[b]), (job >> 1) & 1)) { ok = false; break; }
        tc::tc_fence_after();
        if (kFew && !busy) {  // no query in this warp's rows: whatever their P is, it stays in them
          if (lane == 0) tc::mbar_arrive(smem_u32(&sm.p_full[b]));
          continue;
        }
        // D 256: the row's scores stay in registers over both passes.  D <= 128 (eleven warps, 168
        // registers): chunks of 32 columns, read twice (103 against 115 us on ragged chunks at D 128;
        // at D 256 2140 against 2025 us on the longest one)
        constexpr int kChunk = kM == 1 ? kTile : 32;
        const int vis = lim - t * kTile;  // keys c < vis are visible
        const bool masked = __any_sync(0xffffffffu, vis < kTile);
        uint32_t s[kChunk];
        auto load_scores = [&](int c0) {
#pragma unroll
          for (int c = 0; c < kChunk; c += 32) tc::tmem_ld32(s_col + c0 + c, s + c);
          tc::tmem_wait_ld();
          if (masked) {
#pragma unroll
            for (int c = 0; c < kChunk; ++c) s[c] = c0 + c < vis ? s[c] : 0xff800000u;
          }
        };
        float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll 1
        for (int c0 = 0; c0 < kTile; c0 += kChunk) {
          load_scores(c0);
#pragma unroll
          for (int c = 0; c < kChunk; c += 8)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              m4[i] = max3(m4[i], __uint_as_float(s[c + 2 * i]), __uint_as_float(s[c + 2 * i + 1]));
        }
        if constexpr (kFew) {
          if (a.scores != nullptr && live) {
            float4* dst = reinterpret_cast<float4*>(a.scores + ((int64_t)(tile0 + job) * a.score_rows + row) * kPgKeys);
#pragma unroll
            for (int c = 0; c < kTile; c += 4)
              dst[c / 4] = make_float4(__uint_as_float(s[c]) * scale, __uint_as_float(s[c + 1]) * scale,
                                       __uint_as_float(s[c + 2]) * scale, __uint_as_float(s[c + 3]) * scale);
          }
        }
        const float mx = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])) * scale;
        const bool grow = mx > m + kPgHeadroom;
        const bool rescale = grow && m != -INFINITY;
        const float alpha = rescale ? pg_exp2(m - mx) : 1.0f;
        if (grow) m = mx;
        if (__any_sync(0xffffffffu, rescale)) {
          // O holds the earlier tiles.  D 256: their last product may still run; with two row
          // tiles S(j) was issued behind it
          if (kM == 1 && !wait(smem_u32(&sm.o_done[b ^ 1]), ((job - 1) >> 1) & 1)) { ok = false; break; }
          tc::tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < D; c += 16) {
            uint32_t o[16];
            tc::tmem_ld16(o_col + c, o);
            tc::tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
            tc::tmem_st16(o_col + c, o);
          }
          l2 = f2_pack(f2_lo(l2) * alpha, f2_hi(l2) * alpha);
        }
        const float base = m == -INFINITY ? 0.0f : -m;
        const uint64_t scale2 = f2_pack(scale, scale), base2 = f2_pack(base, base);
#pragma unroll 1
        for (int c0 = 0; c0 < kTile; c0 += kChunk) {
          // (the columns P overwrites, [c0 / 2, c0 / 2 + 16), have been read)
          if (kChunk < kTile) load_scores(c0);
#pragma unroll
          for (int c = 0; c < kChunk; c += 32) {
            uint32_t pk[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const uint64_t x = f2_fma(f2_pack(__uint_as_float(s[c + 2 * i]), __uint_as_float(s[c + 2 * i + 1])), scale2, base2);
              const float e0 = pg_exp2(f2_lo(x)), e1 = pg_exp2(f2_hi(x));
              l2 = f2_add(l2, f2_pack(e0, e1));
              pk[i] = pc_pack<T>(e0, e1);
            }
            tc::tmem_st16(s_col + (c0 + c) / 2, pk);
          }
        }
        tc::tmem_wait_st();
        tc::tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if constexpr (kPair) pc_arrive<false>(lead(smem_u32(&sm.p_full[b])));
          else tc::mbar_arrive(smem_u32(&sm.p_full[b]));
        }
      }
      if (!ok) break;
      // ---- O of this piece
      // (D 256: the product before the last one first, whose arrival nothing else waits for)
      const int last = job - kM;
      if (kM == 1 && last > 0 && !wait(smem_u32(&sm.o_done[(last - 1) & 1]), ((last - 1) >> 1) & 1)) { ok = false; break; }
      if (!wait(smem_u32(&sm.o_done[last & 1]), (last >> 1) & 1)) { ok = false; break; }
      tc::tc_fence_after();
      const float total = f2_lo(l2) + f2_hi(l2);
      const bool whole = w.t == 0 && w.t_end == w.nt;
      const bool none = m == -INFINITY && total == 0.0f;
      const float inv = none ? 0.0f : 1.0f / total;
      const int head = w.h * a.group + row % a.group;
      const int64_t orow = (int64_t)(p.q_start[w.r] + tok) * a.hq + head;
      const int64_t prow = ((int64_t)(2 * worker + (w.piece == 0 ? 0 : 1)) * Shape::kUnit + rt) * kPcRows + row;
      // 128 bytes of a row at a time lie in one lane; 8 lanes exchange 16-byte pieces so that a store
      // instruction writes whole lines of 4 rows (32 lines of one sector each took 9400 cycles a unit)
      const int64_t row_bytes = D * (whole ? 2 : 4);
      const int64_t my_row = !live ? -1 : (whole ? orow : prow) * row_bytes;
      int64_t to[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) to[k] = __shfl_sync(0xffffffffu, my_row, (lane & 24) + k);
      uint8_t* const base = (whole ? reinterpret_cast<uint8_t*>(a.out) : reinterpret_cast<uint8_t*>(a.part_o)) + 16 * (lane & 7);
      auto store = [&](uint32_t (&x)[8][4], int line) {  // the rows' line-th 128 bytes
        pc_transpose8(x, lane);
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (to[k] >= 0)
            *reinterpret_cast<uint4*>(base + to[k] + 128 * line) = make_uint4(x[k][0], x[k][1], x[k][2], x[k][3]);
      };
      if (busy) {
        uint32_t o[32], x[8][4];
        tc::tmem_ld32(o_col, o);
#pragma unroll 1
        for (int c = 0; c < D; c += 32) {
          tc::tmem_wait_ld();
          if (whole) {
            // 64 columns make 128 bytes: this half's 16-bit values beside the last one's
            const bool second = c & 32;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const uint32_t v = pc_pack<T>(__uint_as_float(o[2 * i]) * inv, __uint_as_float(o[2 * i + 1]) * inv);
              if (second) x[4 + i / 4][i % 4] = v;
              else x[i / 4][i % 4] = v;
            }
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) x[i / 4][i % 4] = o[i];
          }
          if (c + 32 < D) tc::tmem_ld32(o_col + c + 32, o);  // the next columns, during the exchange and the stores
          if (!whole) store(x, c / 32);
          else if (c & 32) store(x, c / 64);
        }
      }
      if (live) {
        if (whole) {
          a.lse[orow] = none ? -INFINITY : (m == -INFINITY ? 0.0f : m) * 0.69314718055994531f + logf(total);
          if (a.stats != nullptr) a.stats[orow] = make_float2(m == -INFINITY ? 0.0f : m, inv);
        } else {
          a.part_ml[prow] = make_float2(m, total);
        }
      }
      tc::tc_fence_before();  // the next unit's first product overwrites O after this thread's next P
    }
  } else if (warp == kMma) {
    // ================= MMA issuer (of a pair: the first CTA's)
    constexpr uint32_t fmt = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
    constexpr int kRows = kPair ? 2 * kPcRows : kPcRows;
    constexpr uint32_t idesc_s = tc::instr_desc(fmt, 0, 0, kRows, kTile);
    constexpr uint32_t idesc_o = tc::instr_desc(fmt, 0, 1, kRows, D);
    const uint64_t dq = pc_desc(smem_u32(sm.q), 16, 1024);
    const uint64_t dk = pc_desc(smem_u32(sm.ring), 16, 1024);
    const uint64_t dv = pc_desc(smem_u32(sm.ring), kTile * 128, 1024);
    constexpr uint64_t kSlotStep = Shape::kSlot >> 4;
    // The warp runs the role converged and elects a lane for each batch of products (run by one
    // thread of a diverged warp the products issue slower: 2580 against 2430 us).  What a step
    // needs beside P is waited for before P where its slot was released by earlier steps, so that
    // both products go out back to back; a new unit's queries come only once the S before it is
    // complete and are waited for after the PV
    // S runs two jobs ahead of O and may belong to the next unit
    PcWalk<Shape> ws = w;                               // unit of the next S
    int unit = 0;                                // its number
    int s_left = (ws.t_end - ws.t) * kM, o_left = s_left;  // jobs left in the units of the next S and O
    bool s_open = false, o_open = false;         // the unit's Q has been waited for; O holds a product of the unit
    const int jobs = rank == 0 ? n_tiles * kM : -2;
#pragma unroll 1
    for (int step = 0; step < jobs + 2; ++step) {
      const int jo = step - 2, js = step;
      const int o_mt = kM == 2 ? jo & 1 : 0, s_mt = kM == 2 ? js & 1 : 0;
      const int v_at = pc_v_at<kM>(kM == 2 ? jo >> 1 : jo, n_tiles), v_slot = v_at % kSlots;
      const int k_at = pc_k_at<kM>(kM == 2 ? js >> 1 : js), k_slot = k_at % kSlots;
      if (jo >= 0 && o_mt == 0 && !wait(full(v_slot), (v_at / kSlots) & 1)) break;
      if (js < jobs && s_open && s_mt == 0) {
        if (!wait(full(k_slot), (k_at / kSlots) & 1)) break;
        tc::tc_fence_after();
      }
      if (jo >= 0) {
        if (!wait(smem_u32(&sm.p_full[jo & 1]), (jo >> 1) & 1)) break;
        tc::tc_fence_after();
        if (tc::elect_one()) {
          const uint64_t vd = dv + (uint64_t)v_slot * kSlotStep;
#pragma unroll
          for (int ks = 0; ks < kTile / 16; ++ks)
            pc_mma_ts<kPair>(tmem + kColO + 128 * o_mt, tmem + 128 * (jo & 1) + 8 * ks, vd + ks * (2048 >> 4), idesc_o,
                             (o_open || ks > 0) ? 1u : 0u);
          if (o_mt == kM - 1) pc_commit<kPair>(empty(v_slot));
          pc_commit<kPair>(smem_u32(&sm.o_done[jo & 1]));
        }
        __syncwarp();
        if (o_mt == kM - 1) o_open = true;
        if (--o_left == 0) {
          w.next(a.hk);
          o_open = false;
          o_left = w.live() ? (w.t_end - w.t) * kM : 0;
        }
      }
      if (js < jobs) {
        if (!s_open) {
          if (!wait(smem_u32(&sm.q_full), unit & 1) || !wait(full(k_slot), (k_at / kSlots) & 1)) break;
          tc::tc_fence_after();
          s_open = true;
        }
        const bool last = --s_left == 0;
        if (tc::elect_one()) {
#pragma unroll
          for (int pn = 0; pn < kPanels; ++pn) {
            const uint64_t qd = dq + (uint64_t)((s_mt * kPanels + pn) * (kPcRows * 128 >> 4));
            const uint64_t kd = dk + (uint64_t)k_slot * kSlotStep + (uint64_t)(pn * (Shape::kKeys * 128 >> 4));
#pragma unroll
            for (int ks = 0; ks < 4; ++ks)
              pc_mma_ss<kPair>(tmem + 128 * (js & 1), qd + 2 * ks, kd + 2 * ks, idesc_s, pn + ks > 0 ? 1u : 0u);
          }
          if (s_mt == kM - 1) pc_commit<kPair>(empty(k_slot));
          pc_commit<kPair>(smem_u32(&sm.s_full[js & 1]));
          if (last) pc_commit<kPair>(smem_u32(&sm.q_empty));
        }
        __syncwarp();
        if (last) {
          ws.next(a.hk);
          ++unit;
          s_open = false;
          s_left = ws.live() ? (ws.t_end - ws.t) * kM : 0;
        }
      }
    }
    // no MMA may be in flight when the tensor memory is freed
    if (rank == 0) {
      if (tc::elect_one()) pc_commit<kPair>(smem_u32(&sm.end));
      __syncwarp();
      wait(smem_u32(&sm.end), 0);
    }
  } else {
    // ================= producers: one warp fetches K (and Q), one V, each in the order of use.
    // Lane i holds the pages of boxes i, i + 32, .. of the next tile, looked up while the tile
    // before it is issued; one elected lane issues (operands uniform over the warp)
    const bool is_k = warp == kMma + 1;
    const CUtensorMap* map = is_k ? &kmap : &vmap;
    const int per = kTile / a.box;  // boxes per tile
    const uint32_t box = (uint32_t)a.box, box_bytes = box * 128u;
    // of a pair's tile: K half of the keys, V half of the dims
    const int box0 = kPair && is_k ? (int)rank * (per / 2) : 0, nbox = kPair && is_k ? per / 2 : per;
    const int pan0 = kPair && !is_k ? (int)rank * Shape::kVPanels : 0, pans = is_k ? kPanels : Shape::kVPanels;
    const uint32_t panel = (uint32_t)nbox * box_bytes;  // bytes of a panel of the slot
    const int32_t* row = nullptr;
    int boxes = 0, unit = 0, t = 0, last_at = -1, tails = 0;
    int blk[kTile / 32];
    auto look_up = [&] {
#pragma unroll
      for (int i = 0; i < kTile / 32; ++i) {
        if (32 * i >= per) break;
        const int j = lane + 32 * i, b = t * per + j;
        blk[i] = j < per && b < boxes ? row[a.page.div((uint32_t)b * box)] : 0;
      }
    };
    bool open = false;
#pragma unroll 1
    for (int tile = 0; tile < n_tiles; ++tile) {
      if (!open) {  // a new piece, with its queries
        t = w.t;
        row = a.table + (int64_t)p.req_id[w.r] * a.table_stride;
        boxes = (p.seq[w.r] + a.box - 1) / a.box;
        look_up();
        open = true;
        if (is_k) {
          if (unit > 0 && !wait(smem_u32(&sm.q_empty), (unit - 1) & 1)) break;
          if (tc::elect_one()) {
            const uint32_t bar = lead(smem_u32(&sm.q_full));
            sm.units = unit + 1;
            const uint32_t bytes = (uint32_t)(kM * kPanels * p.box_tokens * a.group * 128);
            if constexpr (kPair) pc_expect(bar, bytes);
            else tc::mbar_expect_tx(bar, bytes);
#pragma unroll 1
            for (int i = 0; i < kM * kPanels; ++i)
              pc_load_3d<kPair>(smem_u32(sm.q) + i * kPcRows * 128, &qmap, 64 * (i % kPanels), w.h * a.group,
                                p.q_start[w.r] + (w.qb * Shape::kUnit + (kPair ? (int)rank : i / kPanels)) * p.tokens, bar);
          }
          __syncwarp();
          ++unit;
        }
      }
      const int first = t * per, h = w.h, here = min(per, max(0, boxes - first));
      const int have = p.seq[w.r] - t * kTile;  // keys of the request from the tile's first on
      int cur[kTile / 32];
#pragma unroll
      for (int i = 0; i < kTile / 32; ++i) {
        cur[i] = blk[i];
        if (lane + 32 * i < here && (cur[i] < 0 || cur[i] >= a.num_blocks)) {
          flag_error(2u);
          cur[i] = (int)a.num_blocks;  // outside the map: zeros
        }
      }
      if (++t < w.t_end) {
        look_up();
      } else {
        w.next(a.hk);
        open = false;
      }
      const int at = is_k ? pc_k_at<kM>(tile) : pc_v_at<kM>(tile, n_tiles), slot = at % kSlots;
      const int live = max(0, min(nbox, here - box0));
      if (at >= kSlots && !wait(empty(slot), ((at / kSlots) - 1) & 1)) break;
      last_at = at;
      // a V tile past whose end anything may stand (0 * NaN) is completed here before it is announced
      const bool tail = !is_k && have < kTile;
      const uint32_t bar = tail ? smem_u32(&sm.tail) : lead(full(slot));
      const uint32_t bytes = (uint32_t)(live * pans) * box_bytes;
      if (tc::elect_one()) {
        if (!tail) sm.at[slot] = at;
        if (kPair && !tail) pc_expect(bar, bytes);
        else tc::mbar_expect_tx(bar, bytes);
      }
      __syncwarp();
      const uint32_t dst = smem_u32(sm.ring[slot]);
#pragma unroll 1
      for (int i = 0; i < live; ++i) {
        const int j = box0 + i;
        int b = 0;
#pragma unroll
        for (int k = 0; k < kTile / 32; ++k) {
          if (32 * k >= per) break;
          const int v = __shfl_sync(0xffffffffu, cur[k], j & 31);
          if (j >> 5 == k) b = v;
        }
        const int off = (int)a.page.mod((uint32_t)(first + j) * box);
        if (tc::elect_one()) {
#pragma unroll
          for (int pn = 0; pn < kPanels; ++pn)
            if (pn < pans)
              pc_load_4d<kPair>(dst + pn * panel + (uint32_t)i * box_bytes, map, 64 * (pan0 + pn), h, off, b, bar);
        }
      }
      __syncwarp();
      if (tail) {
        if (!wait(bar, tails & 1)) {
          pg_drain(bar, tails & 1);
          break;
        }
        ++tails;
        const int clear = max(have, 0);
        for (int i = lane; i < (kTile - clear) * 8 * pans; i += 32) {
          const int key = clear + i / (8 * pans), c = i % (8 * pans);
          *reinterpret_cast<uint4*>(sm.ring[slot] + (c / 8) * panel + key * 128 + (c % 8) * 16) = make_uint4(0, 0, 0, 0);
        }
        tc::fence_async_smem();
        __syncwarp();
        if (lane == 0) {
          sm.at[slot] = at;
          if constexpr (kPair) pc_arrive<true>(lead(full(slot)));
          else tc::mbar_arrive(full(slot));
        }
      }
    }
    // the releases of the last slots come to both CTAs of a pair: none may come to a CTA that ended
    if constexpr (kPair) {
      for (int i = max(0, n_tiles - 3); i < n_tiles; ++i) {
        const int n = is_k ? pc_k_at<kM>(i) : pc_v_at<kM>(i, n_tiles);
        if (n + kSlots >= 2 * n_tiles && n <= last_at && !wait(empty(n % kSlots), (n / kSlots) & 1)) break;
      }
      if (is_k && unit > 0) wait(smem_u32(&sm.q_empty), (unit - 1) & 1);
    }
  }

  __syncwarp();
  tc::tc_fence_before();
  // every role has issued what it will.  Without an abort all copies and products have been waited
  // for, and neither CTA's barriers, tensor or shared memory are used from here on
  if constexpr (kPair) pc_cluster_sync();
  else __syncthreads();
  // (the second CTA's `end` comes here: its MMA warp issues nothing, and from the kernel's start it
  // would wait for the whole stream, which no limit of a wait suits)
  if (kPair && rank == 1 && warp == kMma) pg_drain(smem_u32(&sm.end), 0);
  __syncwarp();
  if (*reinterpret_cast<volatile int*>(&sm.abort) != 0) {  // (the same for both CTAs of a pair)
    if (warp == kMma) {
      pg_drain(smem_u32(&sm.end), 0);
      __syncwarp();
      if (rank == 0) pc_drain_loads<kPair, kSlots>(sm, lane);
      else __nanosleep(100000);  // the other releases of the products that `end` followed are on their way
    }
    __syncwarp();
    if constexpr (kPair) pc_cluster_sync();  // the first CTA counts the second one's copies
  }
  if (warp == kMma) {
    tc::tc_fence_after();
    if constexpr (kPair) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;\n" ::"r"(tmem) : "memory");
    else tc::tmem_dealloc(tmem, 512);
  }
}

// Combine of the divided units.  W warps a row: one where units have few pieces
// (4 rows a CTA), kPcMerge of them where a row has many (decode of few requests);
// warp w takes pieces w, w + W, .. in worker order, the warps' sums are added in
// warp order.  blockIdx.y: divided unit, blockIdx.x: rows of it.
template <int D, typename T, bool kFew, int W>
__global__ void __launch_bounds__(128) paged_merge_kernel(const __grid_constant__ PagedArgs a,
                                                          const __grid_constant__ PcPlan p,
                                                          const __grid_constant__ PcSplits splits) {
  using Shape = PcShape<D, kFew>;
  constexpr int E = D / 32, kRowsHere = 4 / W;
  __shared__ float part[W > 1 ? W : 1][D], part_l[W > 1 ? W : 1];
  pdl_release();
  const int lane = threadIdx.x & 31, warp = (threadIdx.x >> 5) % W;
  const int idx = blockIdx.x * kRowsHere + (threadIdx.x >> 5) / W;
  const PcSplit& u = splits.unit[blockIdx.y];
  const int mt = idx / kPcRows, row = idx % kPcRows;
  const int tok = (u.qb * Shape::kUnit + mt) * p.tokens + row / a.group;
  pdl_wait();
  if (row >= p.tokens * a.group || tok >= p.q_len[u.r]) return;  // (uniform over the warps of a row)
  // the unit is its first worker's last piece, unless that worker begins with it; the others begin inside it
  const bool inside = p.start[u.c0].r == u.r && p.start[u.c0].h == u.h && p.start[u.c0].qb == u.qb;
  auto at = [&](int c) -> int64_t {
    return ((int64_t)(2 * c + (c > u.c0 || inside ? 0 : 1)) * Shape::kUnit + mt) * kPcRows + row;
  };
  float M = -INFINITY;
  for (int c = u.c0 + lane; c <= u.c1; c += 32) M = fmaxf(M, a.part_ml[at(c)].x);
  M = warp_max(M);
  const float base = M == -INFINITY ? 0.0f : M;
  float total = 0.0f, acc[E];
#pragma unroll
  for (int i = 0; i < E; ++i) acc[i] = 0.0f;
#pragma unroll 4
  for (int c = u.c0 + warp; c <= u.c1; c += W) {
    const int64_t r = at(c);
    const float2 ml = a.part_ml[r];
    const float f = pg_exp2(ml.x - base);  // a piece without visible keys: 2^-inf = 0
    const float* src = a.part_o + r * D + E * lane;
    total = fmaf(f, ml.y, total);
#pragma unroll
    for (int i = 0; i < E; i += 2) {
      const float2 v = *reinterpret_cast<const float2*>(src + i);
      acc[i] = fmaf(f, v.x, acc[i]);
      acc[i + 1] = fmaf(f, v.y, acc[i + 1]);
    }
  }
  if constexpr (W > 1) {
#pragma unroll
    for (int i = 0; i < E; ++i) part[warp][E * lane + i] = acc[i];
    if (lane == 0) part_l[warp] = total;
    __syncthreads();
    if (warp != 0) return;
#pragma unroll
    for (int w = 1; w < W; ++w) {
      total += part_l[w];
#pragma unroll
      for (int i = 0; i < E; ++i) acc[i] += part[w][E * lane + i];
    }
  }
  const bool none = M == -INFINITY && total == 0.0f;
  const float inv = none ? 0.0f : 1.0f / total;
  const int64_t orow = (int64_t)(p.q_start[u.r] + tok) * a.hq + u.h * a.group + row % a.group;
  T* dst = reinterpret_cast<T*>(a.out) + orow * D + E * lane;
#pragma unroll
  for (int i = 0; i < E; i += 2) *reinterpret_cast<uint32_t*>(dst + i) = pc_pack<T>(acc[i] * inv, acc[i + 1] * inv);
  if (lane == 0) {
    a.lse[orow] = none ? -INFINITY : base * 0.69314718055994531f + logf(total);
    if (a.stats != nullptr) a.stats[orow] = make_float2(base, inv);
  }
}

}  // namespace oscar
