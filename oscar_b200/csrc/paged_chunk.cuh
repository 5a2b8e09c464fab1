// Attention of long chunks over a paged 16-bit cache on the 5th-generation
// tensor cores (same function as paged.cuh; requests with many query rows).
//
// Work.  A unit is (request, kv head, q-block); a q-block is kM = 1 (D 256) or 2
// (D 64, 128) tiles of 128 query rows, each holding floor(128 / group) tokens x
// group heads.  Its visible keys are cut into 128-key tiles, and the tiles of
// all units, in order, are divided evenly over the CTAs (one per SM) by the
// host, so a CTA streams whole units except at its two ends; the pieces of a
// divided unit are written unnormalised in fp32 and combined by a dependent
// launch in CTA order.
//
// Tile.  Bound by the tensor pipe at D 256 (per 128 keys 16 + 8 MMAs of N 128
// and N 256) and by the exponentials at D <= 128 (128 x 128 of them per MMA
// tile at 16 per cycle and SM).  Jobs alternate between two score buffers:
// D 256: job j is key tile j of the one row tile; D <= 128: key tile j / 2 of
// row tile j % 2.  The MMA warp issues S(0), S(1), then per job O += P(j) V as
// soon as P(j) is written and S(j + 2), so while the softmax of one job runs the
// tensor pipe has the other job's products.
//   TMEM columns: S[0] [0, 128), S[1] [128, 256), O [256, 512) (D 256) or
//   O[0] [256, 256 + D), O[1] [384, 384 + D).  P(j) (16 bit) replaces the first
//   64 columns of S(j) and is the A operand of P V; rows lie on lanes, one
//   query row per softmax thread, so row maxima and sums stay in a thread.
//   S = Q K^T : A = Q, B = K, both shared memory, K-major, 128-byte swizzle.
//   O += P V  : A = P in tensor memory, B = V, MN-major, 128-byte swizzle.
// The running maximum moves only when a score exceeds it by kPgHeadroom (log2
// units); then the thread rescales its row of O in tensor memory.
// Warps: 4 kM softmax, one MMA issuer, two TMA producers (K and Q; V) that fill one
// ring of slots in the order the MMAs use them, in boxes of 64 dims x a power of
// two of tokens.
// Every wait is bounded; a time-out sets the CTA's abort flag and drains.
#pragma once

#include <climits>

#include "paged.cuh"

namespace oscar {

constexpr int kPcRows = 128;
constexpr int kPcKeys = 128;
constexpr int kPcCtas = 192;  // CTAs of a plan

struct PcStart {
  int r, h, qb, t;  // plan index, kv head, q-block, first key tile
};
struct PcPlan {
  int num_req, ctas, tokens;  // tokens per row tile
  int req_id[kPgReqs], q_start[kPgReqs], q_len[kPgReqs], seq[kPgReqs];
  PcStart start[kPcCtas];
  int tiles[kPcCtas];  // key tiles of each CTA
};
struct PcSplit {
  int r, h, qb, c0, c1;  // a divided unit and its CTAs
};
struct PcSplits {
  int n;
  PcSplit unit[kPcCtas];
};

template <int D>
struct PcShape {
  static constexpr int kM = D == 256 ? 1 : 2;           // row tiles per unit
  static constexpr int kPanels = D / 64;
  static constexpr int kHalves = D == 256 ? 2 : 1;      // slots per K or V tile
  static constexpr int kSlot = kPcKeys * D * 2 / kHalves;
  static constexpr int kSlots = D == 64 ? 8 : 5;
  static constexpr int kSoftWarps = 4 * kM;
  static constexpr int kThreads = 32 * (kSoftWarps + 3);
};

template <int D>
struct PcSmem {
  using S = PcShape<D>;
  uint8_t q[S::kM][S::kPanels][kPcRows * 128];  // [row tile][64-dim panel][row][128 bytes], swizzled
  // K tile: [panel][128 keys][128 bytes]; a slot holds half of the panels at D 256.
  // V tile: the same; at D 256 a slot holds 64 keys: [panel][64 keys][128 bytes]
  uint8_t ring[S::kSlots][S::kSlot];
  unsigned long long full[S::kSlots], empty[S::kSlots];
  unsigned long long q_full, q_empty, s_full[2], p_full[2], o_done[2], end;
  uint32_t tmem;
  int abort;
};

OSCAR_DEVINL uint64_t pc_desc(uint32_t addr, uint32_t lbo, uint32_t sbo) {
  return tc::smem_desc(addr, lbo, sbo) | (2ull << 61);  // 128-byte swizzle
}

OSCAR_DEVINL void tma_load_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];\n" ::"r"(
          dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar)
      : "memory");
}

// key tiles that q-block qb of a request sees (at least 1, so that empty rows are written)
template <int D>
__host__ __device__ inline int pc_tiles(int q_len, int seq, int tokens, int qb) {
  const int last = (qb + 1) * tokens * PcShape<D>::kM;
  const int visible = seq - q_len + (last < q_len ? last : q_len);
  return visible > kPcKeys ? (visible + kPcKeys - 1) / kPcKeys : 1;
}

// Ring position of half hf of key tile t's K and V (n tiles in the CTA's stream).
// D <= 128: K0 V0 K1 V1 ..; D 256: K0 K1 V0 K2 V1 .. K(n-1) V(n-2) V(n-1), two slots each.
template <int D>
OSCAR_DEVINL int pc_k_at(int t, int hf) {
  return D == 256 ? 2 * (t == 0 ? 0 : 2 * t - 1) + hf : 2 * t;
}
template <int D>
OSCAR_DEVINL int pc_v_at(int t, int hf, int n) {
  return D == 256 ? 2 * (t == n - 1 ? 2 * n - 1 : 2 * t + 2) + hf : 2 * t + 1;
}

// The pieces of units of one CTA, walked alike by every role.
template <int D>
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
    nt = pc_tiles<D>(p.q_len[r], p.seq[r], p.tokens, qb);
    t_end = min(nt, t + left);
  }
  OSCAR_DEVINL bool live() const { return left > 0; }
  OSCAR_DEVINL void next(int hk) {
    left -= t_end - t;
    t = 0;
    ++piece;
    const int per = p.tokens * PcShape<D>::kM;
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

OSCAR_DEVINL uint64_t f2_pack(float a, float b) {
  return (uint64_t)__float_as_uint(a) | ((uint64_t)__float_as_uint(b) << 32);
}
OSCAR_DEVINL uint64_t f2_fma(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;\n" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
OSCAR_DEVINL uint64_t f2_add(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;\n" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
OSCAR_DEVINL float f2_lo(uint64_t a) { return __uint_as_float((uint32_t)a); }
OSCAR_DEVINL float f2_hi(uint64_t a) { return __uint_as_float((uint32_t)(a >> 32)); }

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

template <int D, typename T>
__global__ void __launch_bounds__(PcShape<D>::kThreads, 1)
paged_chunk_kernel(const __grid_constant__ PagedArgs a, const __grid_constant__ PcPlan p,
                   const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                   const __grid_constant__ CUtensorMap vmap) {
  using Shape = PcShape<D>;
  constexpr int kM = Shape::kM, kPanels = Shape::kPanels, kHalves = Shape::kHalves, kSlots = Shape::kSlots;
  constexpr int kMma = Shape::kSoftWarps;
  constexpr int kColO = 256;
  extern __shared__ __align__(1024) uint8_t pc_raw[];
  PcSmem<D>& sm = *reinterpret_cast<PcSmem<D>*>(pc_raw);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  pdl_release();
  auto full = [&](int i) { return smem_u32(&sm.full[i]); };
  auto empty = [&](int i) { return smem_u32(&sm.empty[i]); };
  if (warp == kMma) {
    if (lane == 0) {
      for (int i = 0; i < kSlots; ++i) {
        tc::mbar_init(full(i), 1);
        tc::mbar_init(empty(i), 1);
      }
      for (int i = 0; i < 2; ++i) {
        tc::mbar_init(smem_u32(&sm.s_full[i]), 1);
        tc::mbar_init(smem_u32(&sm.p_full[i]), kPcRows);
        tc::mbar_init(smem_u32(&sm.o_done[i]), 1);
      }
      tc::mbar_init(smem_u32(&sm.q_full), 1);
      tc::mbar_init(smem_u32(&sm.q_empty), 1);
      tc::mbar_init(smem_u32(&sm.end), 1);
      sm.abort = 0;
      tc::mbar_fence_init();
    }
    __syncwarp();
    tc::tmem_alloc(smem_u32(&sm.tmem), 512);
    tc::tmem_relinquish();
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = sm.tmem;
  auto wait = [&](uint32_t bar, uint32_t parity) -> bool {  // warp-uniform
    return __all_sync(0xffffffffu, pg_wait(sm.abort, bar, parity));
  };
  pdl_wait();
  PcWalk<D> w(p, blockIdx.x);
  const int n_tiles = w.left;

  if (warp < kMma) {
    // ================= softmax: thread = query row of row tile `wg`
    const int wg = warp / 4, row = tid & 127;
    const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
    const int rows = p.tokens * a.group;  // live rows of a row tile
    int job = kM == 2 ? wg : 0;           // jobs are numbered over the whole CTA
    const float scale = a.scale_log2;
    bool ok = true;
    for (; w.live() && ok; w.next(a.hk)) {
      const int q_len = p.q_len[w.r], seq = p.seq[w.r];
      const int tok = (w.qb * kM + wg) * p.tokens + row / a.group;
      const bool live = row < rows && tok < q_len;
      // visible keys; rows that hold no query are computed as they come and not written
      const int lim = live ? max(0, seq - q_len + tok + 1) : INT_MAX;
      float m = -INFINITY;
      uint64_t l2 = 0;  // two partial sums
      const uint32_t o_col = tmem + lanes + kColO + (kM == 2 ? 128 * wg : 0);
#pragma unroll 1
      for (int t = w.t; t < w.t_end; ++t, job += kM) {
        const int b = job & 1;
        const uint32_t s_col = tmem + lanes + 128 * b;
        if (!wait(smem_u32(&sm.s_full[b]), (job >> 1) & 1)) { ok = false; break; }
        tc::tc_fence_after();
        // Two passes over the scores in chunks of 32 columns, each a short loop: unrolled over
        // the row, the warps of the CTA run out of the instruction cache (see below)
        const int vis = lim - t * kPcKeys;  // keys c < vis are visible
        const bool masked = __any_sync(0xffffffffu, vis < kPcKeys);
        uint32_t s[32];
        float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll 1
        for (int c0 = 0; c0 < kPcKeys; c0 += 32) {
          tc::tmem_ld32(s_col + c0, s);
          tc::tmem_wait_ld();
          if (masked) {
#pragma unroll
            for (int c = 0; c < 32; ++c) s[c] = c0 + c < vis ? s[c] : 0xff800000u;
          }
#pragma unroll
          for (int c = 0; c < 32; c += 8)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              m4[i] = max3(m4[i], __uint_as_float(s[c + 2 * i]), __uint_as_float(s[c + 2 * i + 1]));
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
        for (int c0 = 0; c0 < kPcKeys; c0 += 32) {
          // (the columns P overwrites, [c0 / 2, c0 / 2 + 16), have been read)
          tc::tmem_ld32(s_col + c0, s);
          tc::tmem_wait_ld();
          if (masked) {
#pragma unroll
            for (int c = 0; c < 32; ++c) s[c] = c0 + c < vis ? s[c] : 0xff800000u;
          }
          uint32_t pk[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const uint64_t x = f2_fma(f2_pack(__uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1])), scale2, base2);
            const float e0 = pg_exp2(f2_lo(x)), e1 = pg_exp2(f2_hi(x));
            l2 = f2_add(l2, f2_pack(e0, e1));
            pk[i] = pc_pack<T>(e0, e1);
          }
          tc::tmem_st16(s_col + c0 / 2, pk);
        }
        const int have = seq - t * kPcKeys;
        if (have < kPcKeys) {
          // the last tile: what lies past the sequence may be anything (0 * NaN).  The V slots of
          // the tile have landed before their rows are cleared
          const int first = max(have, 0);
          const int order = kM == 2 ? job >> 1 : job;  // key tile in the CTA's stream
          // (D 256: the product before it is complete, so the slot's earlier use has landed too and
          // the parity below can only mean this one)
          bool there = kM == 2 || job == 0 || wait(smem_u32(&sm.o_done[b ^ 1]), ((job - 1) >> 1) & 1);
#pragma unroll
          for (int hf = 0; hf < kHalves; ++hf) {
            const int at = pc_v_at<D>(order, hf, n_tiles);
            there = there && wait(full(at % kSlots), (at / kSlots) & 1);
            constexpr int kRowsHere = kPcKeys / kHalves;
            uint8_t* v = sm.ring[at % kSlots];
            for (int i = row; i < kRowsHere * (D / 8); i += kPcRows) {
              const int key = i / (D / 8), ch = i % (D / 8);
              if (hf * kRowsHere + key >= first)
                *reinterpret_cast<uint4*>(v + (ch / 8) * (kRowsHere * 128) + key * 128 + (ch % 8) * 16) = make_uint4(0, 0, 0, 0);
            }
          }
          if (!there) { ok = false; break; }
          tc::fence_async_smem();
        }
        tc::tmem_wait_st();
        tc::tc_fence_before();
        tc::mbar_arrive(smem_u32(&sm.p_full[b]));
      }
      if (!ok) break;
      // ---- O of this piece
      const int last = job - kM;
      if (!wait(smem_u32(&sm.o_done[last & 1]), (last >> 1) & 1)) { ok = false; break; }
      tc::tc_fence_after();
      const float total = f2_lo(l2) + f2_hi(l2);
      const bool whole = w.t == 0 && w.t_end == w.nt;
      const bool none = m == -INFINITY && total == 0.0f;
      const float inv = none ? 0.0f : 1.0f / total;
      const int head = w.h * a.group + row % a.group;
      const int64_t orow = (int64_t)(p.q_start[w.r] + tok) * a.hq + head;
      const int64_t prow = ((int64_t)(2 * blockIdx.x + (w.piece == 0 ? 0 : 1)) * kM + wg) * kPcRows + row;
#pragma unroll 1
      for (int c = 0; c < D; c += 32) {
        uint32_t o[32];
        tc::tmem_ld32(o_col + c, o);
        tc::tmem_wait_ld();
        if (!live) continue;
        if (whole) {
          uint4* dst = reinterpret_cast<uint4*>(reinterpret_cast<T*>(a.out) + orow * D + c);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t x[4];
#pragma unroll
            for (int k = 0; k < 4; ++k)
              x[k] = pc_pack<T>(__uint_as_float(o[8 * i + 2 * k]) * inv, __uint_as_float(o[8 * i + 2 * k + 1]) * inv);
            dst[i] = make_uint4(x[0], x[1], x[2], x[3]);
          }
        } else {
          uint4* dst = reinterpret_cast<uint4*>(a.part_o + prow * D + c);
#pragma unroll
          for (int i = 0; i < 8; ++i) dst[i] = make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
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
    // ================= MMA issuer
    constexpr uint32_t fmt = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
    constexpr uint32_t idesc_s = tc::instr_desc(fmt, 0, 0, kPcRows, kPcKeys);
    constexpr uint32_t idesc_o = tc::instr_desc(fmt, 0, 1, kPcRows, D);
    const uint64_t dq = pc_desc(smem_u32(sm.q), 16, 1024);
    const uint64_t dk = pc_desc(smem_u32(sm.ring), 16, 1024);
    const uint64_t dv = pc_desc(smem_u32(sm.ring), (kPcKeys / kHalves) * 128, 1024);
    constexpr uint64_t kSlotStep = Shape::kSlot >> 4;
    // S runs two jobs ahead of O and may belong to the next unit
    PcWalk<D> ws = w;                            // unit of the next S
    int unit = 0;                                // its number
    int s_left = (ws.t_end - ws.t) * kM, o_left = s_left;  // jobs left in the units of the next S and O
    bool s_open = false, o_open = false;         // the unit's Q has been waited for; O holds a product of the unit
    const int jobs = n_tiles * kM;
#pragma unroll 1
    for (int step = 0; step < jobs + 2; ++step) {
      const int jo = step - 2, js = step;
      if (jo >= 0) {
        const int tile = kM == 2 ? jo >> 1 : jo;
        const int mt = kM == 2 ? jo & 1 : 0;
        if (!wait(smem_u32(&sm.p_full[jo & 1]), (jo >> 1) & 1)) break;
        bool there = true;
        if (mt == 0) {
#pragma unroll
          for (int hf = 0; hf < kHalves; ++hf) {
            const int at = pc_v_at<D>(tile, hf, n_tiles);
            there = there && wait(full(at % kSlots), (at / kSlots) & 1);
          }
        }
        if (!there) break;
        tc::tc_fence_after();
        if (tc::elect_one()) {
          constexpr int kStepsPerSlot = kPcKeys / kHalves / 16;
#pragma unroll
          for (int ks = 0; ks < kPcKeys / 16; ++ks) {
            const int at = pc_v_at<D>(tile, ks / kStepsPerSlot, n_tiles);
            const uint64_t vd = dv + (uint64_t)(at % kSlots) * kSlotStep + (uint64_t)((ks % kStepsPerSlot) * (2048 >> 4));
            tc::mma_ts(tmem + kColO + 128 * mt, tmem + 128 * (jo & 1) + 8 * ks, vd, idesc_o, (o_open || ks > 0) ? 1u : 0u);
            if (mt == kM - 1 && (ks + 1) % kStepsPerSlot == 0) tc::mma_commit(empty(at % kSlots));
          }
          tc::mma_commit(smem_u32(&sm.o_done[jo & 1]));
        }
        __syncwarp();
        if (mt == kM - 1) o_open = true;
        if (--o_left == 0) {
          w.next(a.hk);
          o_open = false;
          o_left = w.live() ? (w.t_end - w.t) * kM : 0;
        }
      }
      if (js < jobs) {
        if (!s_open && !wait(smem_u32(&sm.q_full), unit & 1)) break;
        s_open = true;
        const int tile = kM == 2 ? js >> 1 : js;
        const int mt = kM == 2 ? js & 1 : 0;
        bool there = true;
        if (mt == 0) {
#pragma unroll
          for (int hf = 0; hf < kHalves; ++hf) {
            const int at = pc_k_at<D>(tile, hf);
            there = there && wait(full(at % kSlots), (at / kSlots) & 1);
          }
        }
        if (!there) break;
        tc::tc_fence_after();
        const bool last = --s_left == 0;
        if (tc::elect_one()) {
#pragma unroll
          for (int pn = 0; pn < kPanels; ++pn) {
            const int at = pc_k_at<D>(tile, pn * kHalves / kPanels);
            const uint64_t qd = dq + (uint64_t)((mt * kPanels + pn) * (kPcRows * 128 >> 4));
            const uint64_t kd = dk + (uint64_t)(at % kSlots) * kSlotStep +
                                (uint64_t)((pn % (kPanels / kHalves)) * (kPcKeys * 128 >> 4));
#pragma unroll
            for (int ks = 0; ks < 4; ++ks)
              tc::mma_ss(tmem + 128 * (js & 1), qd + 2 * ks, kd + 2 * ks, idesc_s, pn + ks > 0 ? 1u : 0u);
            // a slot is released as soon as its last product is issued
            if (mt == kM - 1 && (pn + 1) % (kPanels / kHalves) == 0) tc::mma_commit(empty(at % kSlots));
          }
          tc::mma_commit(smem_u32(&sm.s_full[js & 1]));
          if (last) tc::mma_commit(smem_u32(&sm.q_empty));
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
    if (tc::elect_one()) tc::mma_commit(smem_u32(&sm.end));
    __syncwarp();
    if (!tc::mbar_wait(smem_u32(&sm.end), 0) && lane == 0) flag_error(16u);
  } else {
    // ================= producers: one warp fetches K (and Q), one V, each in the order of use.
    // Lane i holds the pages of boxes i, i + 32, .. of the next tile, looked up while the tile
    // before it is issued; one elected lane issues (operands uniform over the warp)
    const bool is_k = warp == kMma + 1;
    const CUtensorMap* map = is_k ? &kmap : &vmap;
    const int per = kPcKeys / a.box;  // boxes per tile
    const uint32_t box = (uint32_t)a.box, box_bytes = box * 128u;
    const int32_t* row = nullptr;
    int boxes = 0, unit = 0, t = 0, last_at = -1;
    int blk[kPcKeys / 32];
    auto look_up = [&] {
#pragma unroll
      for (int i = 0; i < kPcKeys / 32; ++i) {
        if (32 * i >= per) break;
        const int j = lane + 32 * i, b = t * per + j;
        blk[i] = j < per && b < boxes ? row[a.page.div((uint32_t)b * box)] : 0;
      }
    };
    bool ok = true, open = false;
#pragma unroll 1
    for (int tile = 0; tile < n_tiles && ok; ++tile) {
      if (!open) {  // a new piece, with its queries
        t = w.t;
        row = a.table + (int64_t)p.req_id[w.r] * a.table_stride;
        boxes = (p.seq[w.r] + a.box - 1) / a.box;
        look_up();
        open = true;
        if (is_k) {
          if (unit > 0 && !wait(smem_u32(&sm.q_empty), (unit - 1) & 1)) break;
          if (tc::elect_one()) {
            const uint32_t bar = smem_u32(&sm.q_full);
            tc::mbar_expect_tx(bar, (uint32_t)(kM * kPanels * p.tokens * a.group * 128));
#pragma unroll 1
            for (int i = 0; i < kM * kPanels; ++i)
              tma_load_3d(smem_u32(sm.q) + i * kPcRows * 128, &qmap, 64 * (i % kPanels), w.h * a.group,
                          p.q_start[w.r] + (w.qb * kM + i / kPanels) * p.tokens, bar);
          }
          __syncwarp();
          ++unit;
        }
      }
      const int first = t * per, h = w.h, here = min(per, max(0, boxes - first));
      int cur[kPcKeys / 32];
#pragma unroll
      for (int i = 0; i < kPcKeys / 32; ++i) {
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
#pragma unroll 1
      for (int hf = 0; hf < kHalves; ++hf) {
        const int at = is_k ? pc_k_at<D>(tile, hf) : pc_v_at<D>(tile, hf, n_tiles), slot = at % kSlots;
        // K: panels [hf * kPanels / kHalves, ..), all boxes; V: all panels, boxes of this key half
        const int pan0 = is_k ? hf * (kPanels / kHalves) : 0, pans = is_k ? kPanels / kHalves : kPanels;
        const int box0 = is_k ? 0 : hf * (per / kHalves), nbox = is_k ? per : per / kHalves;
        const int live = max(0, min(nbox, here - box0));
        const uint32_t panel = (uint32_t)nbox * box_bytes;  // bytes of a panel of the slot
        if (at >= kSlots && !wait(empty(slot), ((at / kSlots) - 1) & 1)) { ok = false; break; }
        last_at = at;
        if (tc::elect_one()) tc::mbar_expect_tx(full(slot), (uint32_t)(live * pans) * box_bytes);
        __syncwarp();
        const uint32_t dst = smem_u32(sm.ring[slot]);
#pragma unroll 1
        for (int i = 0; i < live; ++i) {
          const int j = box0 + i;
          int b = 0;
#pragma unroll
          for (int k = 0; k < kPcKeys / 32; ++k) {
            if (32 * k >= per) break;
            const int v = __shfl_sync(0xffffffffu, cur[k], j & 31);
            if (j >> 5 == k) b = v;
          }
          const int off = (int)a.page.mod((uint32_t)(first + j) * box);
          if (tc::elect_one()) {
#pragma unroll
            for (int pn = 0; pn < kPanels; ++pn)
              if (pn < pans)
                tma_load_4d(dst + pn * panel + (uint32_t)i * box_bytes, map, 64 * (pan0 + pn), h, off, b, full(slot));
          }
        }
        __syncwarp();
      }
    }
    // no copy may still be writing shared memory when the CTA ends.  The MMA warp has waited for
    // all of them unless a wait timed out
    if (*reinterpret_cast<volatile int*>(&sm.abort) != 0) {
      for (int n = max(0, last_at - kSlots + 1); n <= last_at; ++n) tc::mbar_wait(full(n % kSlots), (n / kSlots) & 1);
      if (is_k && unit > 0) tc::mbar_wait(smem_u32(&sm.q_full), (unit - 1) & 1);
    }
  }

  tc::tc_fence_before();
  __syncthreads();
  if (warp == kMma) {
    tc::tc_fence_after();
    tc::tmem_dealloc(tmem, 512);
  }
}

// Combine of the divided units, a warp per query row.
template <int D, typename T>
__global__ void __launch_bounds__(128) paged_chunk_combine_kernel(const __grid_constant__ PagedArgs a,
                                                                  const __grid_constant__ PcPlan p,
                                                                  const __grid_constant__ PcSplits splits) {
  constexpr int kM = PcShape<D>::kM, E = D / 32;
  pdl_release();
  const int lane = threadIdx.x & 31;
  const int idx = blockIdx.x * 4 + (threadIdx.x >> 5);
  const PcSplit& u = splits.unit[idx / (kM * kPcRows)];
  const int mt = idx / kPcRows % kM, row = idx % kPcRows;
  const int tok = (u.qb * kM + mt) * p.tokens + row / a.group;
  pdl_wait();
  if (row >= p.tokens * a.group || tok >= p.q_len[u.r]) return;
  // a divided unit is its CTA's last piece except where the CTA began inside it
  auto at = [&](int c) -> int64_t {
    const bool first = c > u.c0 || (p.start[c].r == u.r && p.start[c].h == u.h && p.start[c].qb == u.qb);
    return ((int64_t)(2 * c + (first ? 0 : 1)) * kM + mt) * kPcRows + row;
  };
  float M = -INFINITY;
  for (int c = u.c0 + lane; c <= u.c1; c += 32) M = fmaxf(M, a.part_ml[at(c)].x);
  M = warp_max(M);
  const float base = M == -INFINITY ? 0.0f : M;
  float total = 0.0f, acc[E];
#pragma unroll
  for (int i = 0; i < E; ++i) acc[i] = 0.0f;
#pragma unroll 2
  for (int c = u.c0; c <= u.c1; ++c) {
    const int64_t r = at(c);
    const float2 ml = a.part_ml[r];
    const float f = pg_exp2(ml.x - base);
    const float* src = a.part_o + r * D + E * lane;
    total = fmaf(f, ml.y, total);
#pragma unroll
    for (int i = 0; i < E; i += 2) {
      const float2 v = *reinterpret_cast<const float2*>(src + i);
      acc[i] = fmaf(f, v.x, acc[i]);
      acc[i + 1] = fmaf(f, v.y, acc[i + 1]);
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
