// Attention over a paged 16-bit cache: arguments, plan and the split-KV kernel
// for requests with few query rows (decode, draft steps), its combine, and the
// keys' accumulated attention weights.
//
//   S = scale Q K^T, row (token i of its request) sees keys [0, seq - q_len + i]
//   O = softmax(S) V,  LSE = log sum exp S
//   weights[slot, h] += sum over observed rows of the group of exp(S - LSE)
//
// Work.  A unit is (request, block of ROWS rows = tokens x heads of the group,
// kv head); its keys are cut into 64-key tiles.  All units' tiles form one
// list, and CTA c of C takes [T c / C, T (c + 1) / C) of it: every SM streams
// the same number of bytes whatever the requests' lengths are.  A unit that
// lies in one CTA's range is finished there; the pieces of a divided unit are
// written unnormalised in fp32 with their maximum and sum, and combined by a
// dependent launch in CTA order (no atomics: the result does not depend on
// timing).
//
// Tile.  Bound by HBM: K and V stream through shared memory once.  One warp
// issues TMA boxes of 64 dims x (the largest power of two that divides the
// page) tokens into a ring of stages; eight warps compute.  For S a warp takes
// 8 of the tile's 64 keys against 16 rows (16 keys and half of the rows when
// there are 32: the Q fragments then still fit the registers), for O it takes
// D / 8 of the dims against all keys, so a row's accumulators are spread over the warps and K
// and V are read from shared memory once.  P goes through shared memory (two
// buffers); its one barrier per tile also carries the vote whether a row's
// maximum grew by more than kPgHeadroom (log2 units): only then do the warps
// exchange maxima and rescale.
#pragma once

#include "tc.cuh"

namespace oscar {

constexpr int kPgKeys = 64;       // keys per tile
constexpr int kPgReqs = 256;      // requests per launch (the plan travels by value)
constexpr int kPgWarps = 8;       // compute warps
constexpr int kPgThreads = 32 * (kPgWarps + 1);
constexpr int kPgCtas = 192;      // CTAs of a plan
constexpr int kPgMerge = 4;       // warps that combine one row
constexpr float kPgHeadroom = 8.0f;

struct PagedPlan {
  int num_req;
  int ctas;             // CTAs that share the tiles
  int64_t total_tiles;
  int req_id[kPgReqs];  // row of the block table
  int q_start[kPgReqs];
  int q_len[kPgReqs];
  int seq[kPgReqs];
  int64_t tile_begin[kPgReqs + 1];
  int64_t cta_begin[kPgCtas + 1];  // first tile of each CTA: total_tiles * c / ctas
};

// Division by the page size without a divide (it sits in the producers' serial path, where
// one costs 150 cycles): q = (mulhi(mul, n) + n) >> shift for n < 2^31, with
// shift = ceil(log2 d), mul = floor(2^32 (2^shift - d) / d) + 1.
struct FastDiv {
  uint32_t d, mul, shift;
  OSCAR_DEVINL uint32_t div(uint32_t n) const { return (__umulhi(mul, n) + n) >> shift; }
  OSCAR_DEVINL uint32_t mod(uint32_t n) const { return n - div(n) * d; }
};

struct PagedArgs {
  const void* q;
  int64_t q_tok, q_head;  // strides in elements
  void* out;              // [n, hq, D] in the queries' type
  float* lse;             // [n, hq]
  float2* stats;          // [n, hq] (maximum in log2 units, 1 / sum), or null
  int hq, hk, group;
  int64_t num_blocks;
  int bs;
  FastDiv page;           // by bs
  int box;                // tokens per TMA box: a power of two that divides the page, at most 64
  const int32_t* table;
  int64_t table_stride;
  float scale_log2;       // scale * log2(e)
  float* part_o;          // [2 * ctas][ROWS][D] unnormalised
  float2* part_ml;        // [2 * ctas][ROWS] (maximum, sum)
  float* scores;          // [tile][ROWS][64] scaled scores in log2 units, or null
  float* weights;         // [num_blocks, hk, bs], or null
  int observe;            // the last `observe` tokens of a request weigh the keys
};

OSCAR_DEVINL int pg_find(const int64_t* begin, int n, int64_t x) {
  int lo = 0, hi = n;  // last i with begin[i] <= x
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (begin[mid] <= x) lo = mid; else hi = mid;
  }
  return lo;
}
OSCAR_DEVINL float pg_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}

OSCAR_DEVINL void tma_load_4d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, int w, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
      "[%6];\n" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar)
      : "memory");
}

// A unit's geometry, the same for every role of a CTA.
struct PagedUnit {
  int r;              // index in the plan
  int row0, nrows;    // rows of the request: token * group + head in group
  int h;
  int64_t begin, end;  // tiles
  int q_start, q_len, seq;
};

template <int ROWS>
OSCAR_DEVINL PagedUnit pg_unit(const PagedPlan& p, const PagedArgs& a, int64_t g) {
  PagedUnit u;
  u.r = pg_find(p.tile_begin, p.num_req, g);
  u.q_start = p.q_start[u.r];
  u.q_len = p.q_len[u.r];
  u.seq = p.seq[u.r];
  const int nt = max(1, (u.seq + kPgKeys - 1) / kPgKeys);
  const int64_t local = g - p.tile_begin[u.r];
  const int unit = (int)(local / nt);
  u.h = unit % a.hk;
  u.row0 = (unit / a.hk) * ROWS;
  u.nrows = min(ROWS, u.q_len * a.group - u.row0);
  u.begin = p.tile_begin[u.r] + (int64_t)unit * nt;
  u.end = u.begin + nt;
  return u;
}

template <int D, int NRT>
struct PagedSmem {
  static constexpr int kTile = kPgKeys * D * 2;
  static constexpr int kStages = D == 256 ? 3 : D == 128 ? 6 : 8;
  uint8_t k[kStages][kTile];  // [64-dim panel][key][128 bytes], 16-byte chunks XOR-swizzled by key % 8 (TMA SWIZZLE_128B)
  uint8_t v[kStages][kTile];
  uint8_t p[2][16 * NRT * 128];  // [row][64 keys], swizzled the same way
  float mx[kPgWarps][16];   // of the warp's 16 rows
  float sum[kPgWarps][16];
  unsigned long long full_k[kStages], full_v[kStages], empty_k[kStages], empty_v[kStages];
  int abort;
};

// 16-byte chunk `c` of 128-byte row `r` under the 128-byte swizzle
OSCAR_DEVINL uint32_t pg_swz(int r, int c) { return (uint32_t)(r * 128 + ((c ^ (r & 7)) << 4)); }

// Bounded wait of a CTA whose roles never leave early: the first time-out sets
// the CTA's abort flag, after which every wait returns soon and the warps run
// to the end through their (always complete) barriers.  A waiting warp suspends
// for up to a millisecond a try: polls take shared-memory cycles from the
// tensor cores' operands (2570 against 2430 us on the longest chunk).
constexpr uint32_t kPgTries = 4096;
OSCAR_DEVINL bool pg_try(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n selp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(ok)
      : "r"(bar), "r"(parity), "r"(1000000u)
      : "memory");
  return ok != 0;
}
OSCAR_DEVINL bool pg_wait(int& abort, uint32_t bar, uint32_t parity) {
  if (tc::mbar_test(bar, parity)) return true;
  for (uint32_t i = 0; i < kPgTries; ++i) {
    if (pg_try(bar, parity)) return true;
    if (*reinterpret_cast<volatile int*>(&abort) != 0) return false;
  }
  *reinterpret_cast<volatile int*>(&abort) = 1;
  flag_error(16u);
  return false;
}

// Producer: one warp.  Lane i holds the block of box (base + i) of the unit, the
// next 32 boxes' blocks are fetched one group ahead; one elected lane issues (lanes
// with operands of their own would be serialised).
template <int D, int ROWS, typename Smem>
OSCAR_DEVINL void pg_produce(Smem& sm, const PagedArgs& a, const PagedPlan& p, const CUtensorMap* kmap,
                             const CUtensorMap* vmap, int64_t g0, int64_t g1, int lane) {
  constexpr int kPanels = D / 64, kSt = Smem::kStages;
  const int per = kPgKeys / a.box;  // boxes per tile
  const uint32_t box_bytes = (uint32_t)a.box * 128u;
  uint32_t it = 0;
  for (int64_t g = g0; g < g1;) {
    const PagedUnit u = pg_unit<ROWS>(p, a, g);
    const int64_t stop = u.end < g1 ? u.end : g1;
    const int32_t* row = a.table + (int64_t)p.req_id[u.r] * a.table_stride;
    const int boxes = (u.seq + a.box - 1) / a.box;  // of the whole request
    const uint32_t box = (uint32_t)a.box;
    auto fetch = [&](int b) -> int { return b < boxes ? row[a.page.div((uint32_t)b * box)] : -1; };
    int base = (int)(g - u.begin) * per;
    int cur = fetch(base + lane), nxt = fetch(base + 32 + lane);
    for (; g < stop; ++g, ++it) {
      const int st = it % kSt;
      const uint32_t phase = (it / kSt) & 1;
      const int first = (int)(g - u.begin) * per;  // first box of the tile
      const int live = max(0, min(per, boxes - first));
      const uint32_t bytes = (uint32_t)live * box_bytes * kPanels;
      const uint32_t fk = smem_u32(&sm.full_k[st]), fv = smem_u32(&sm.full_v[st]);
      if (it >= kSt) {
        const bool k_free = pg_wait(sm.abort, smem_u32(&sm.empty_k[st]), phase ^ 1);
        const bool v_free = pg_wait(sm.abort, smem_u32(&sm.empty_v[st]), phase ^ 1);
        if (!__all_sync(0xffffffffu, k_free && v_free)) {
          g = g1;  // gave up: issue nothing more
          break;
        }
      }
      if (lane == 0) {
        tc::mbar_expect_tx(fk, bytes);
        tc::mbar_expect_tx(fv, bytes);
      }
      __syncwarp();
      for (int j = 0; j < live; ++j) {
        const int b = first + j;
        if (b - base >= 32) {
          base += 32;
          cur = nxt;
          nxt = fetch(base + 32 + lane);
        }
        int blk = __shfl_sync(0xffffffffu, cur, b - base);
        if (blk < 0 || blk >= a.num_blocks) {
          if (lane == 0) flag_error(2u);
          blk = (int)a.num_blocks;  // outside the map: the box is filled with zeros
        }
        const int off = (int)a.page.mod((uint32_t)b * box);
        if (tc::elect_one()) {
          const uint32_t at = (uint32_t)j * box_bytes;
#pragma unroll
          for (int pn = 0; pn < kPanels; ++pn)
            tma_load_4d(smem_u32(sm.k[st]) + pn * (kPgKeys * 128u) + at, kmap, pn * 64, u.h, off, blk, fk);
#pragma unroll
          for (int pn = 0; pn < kPanels; ++pn)
            tma_load_4d(smem_u32(sm.v[st]) + pn * (kPgKeys * 128u) + at, vmap, pn * 64, u.h, off, blk, fv);
        }
      }
    }
  }
  // no copy may still be writing shared memory when the CTA ends
  for (uint32_t t = it > (uint32_t)kSt ? it - kSt : 0; t < it; ++t) {
    tc::mbar_wait(smem_u32(&sm.full_k[t % kSt]), (t / kSt) & 1);
    tc::mbar_wait(smem_u32(&sm.full_v[t % kSt]), (t / kSt) & 1);
  }
}

template <int D, typename T, int NRT>
__global__ void __launch_bounds__(kPgThreads, 1)
paged_split_kernel(const __grid_constant__ PagedArgs a, const __grid_constant__ PagedPlan p,
                   const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap) {
  constexpr int ROWS = 16 * NRT;
  constexpr int kSteps = D / 16;        // MMA k-steps of S
  constexpr int kWarpDims = D / kPgWarps;
  constexpr int kNT = kWarpDims / 8;    // 8-dim output tiles of a warp
  constexpr int kOwn = NRT == 1 ? 2 : 4;  // scores of a thread and row
  using Smem = PagedSmem<D, NRT>;
  extern __shared__ __align__(1024) uint8_t pg_raw[];
  Smem& sm = *reinterpret_cast<Smem*>(pg_raw);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  pdl_release();
  if (tid == 0) {
    for (int i = 0; i < Smem::kStages; ++i) {
      tc::mbar_init(smem_u32(&sm.full_k[i]), 1);
      tc::mbar_init(smem_u32(&sm.full_v[i]), 1);
      tc::mbar_init(smem_u32(&sm.empty_k[i]), kPgWarps);
      tc::mbar_init(smem_u32(&sm.empty_v[i]), kPgWarps);
    }
    sm.abort = 0;
    tc::mbar_fence_init();
  }
  __syncthreads();
  const int64_t g0 = p.cta_begin[blockIdx.x], g1 = p.cta_begin[blockIdx.x + 1];
  pdl_wait();
  if (warp == kPgWarps) {
    pg_produce<D, ROWS>(sm, a, p, &kmap, &vmap, g0, g1, lane);
    return;
  }

  const int qr = lane >> 2, qc = lane & 3;  // row and column pair of a fragment
  // S: 8 keys x 16 rows per warp, or (32 rows) 16 keys x one of the two 16-row tiles
  const int my_rt = NRT == 1 ? 0 : warp / 4;
  const int my_key = NRT == 1 ? 8 * warp : 16 * (warp % 4);
  auto sync_warps = [&] { tc::bar_sync(1, 32 * kPgWarps); };
  uint32_t it = 0;
  for (int64_t g = g0; g < g1;) {
    const PagedUnit u = pg_unit<ROWS>(p, a, g);
    const int64_t stop = u.end < g1 ? u.end : g1;
    const bool whole = g == u.begin && stop == u.end;
    const int64_t seg_first = g;

    // Q fragments of this warp's 16 rows (rows qr, qr + 8) and their visible key counts
    uint32_t qf[kSteps][4];
    int lim[2];
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      const int row = 16 * my_rt + 8 * hf + qr;
      const bool live = row < u.nrows;
      const int rr = u.row0 + row, tok = rr / a.group;
      lim[hf] = live ? max(0, u.seq - u.q_len + tok + 1) : 0;
      const T* src = reinterpret_cast<const T*>(a.q) + (int64_t)(u.q_start + tok) * a.q_tok +
                     (int64_t)(u.h * a.group + rr - tok * a.group) * a.q_head;
#pragma unroll
      for (int ks = 0; ks < kSteps; ++ks)
#pragma unroll
        for (int kh = 0; kh < 2; ++kh)
          qf[ks][2 * kh + hf] = live ? *reinterpret_cast<const uint32_t*>(src + 16 * ks + 8 * kh + 2 * qc) : 0u;
    }
    float o[NRT][kNT][4];
    float m[NRT][2], l[2] = {0.0f, 0.0f};  // l: this warp's rows over its keys
#pragma unroll
    for (int rt = 0; rt < NRT; ++rt) {
#pragma unroll
      for (int n = 0; n < kNT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[rt][n][i] = 0.0f;
      m[rt][0] = m[rt][1] = -INFINITY;
    }
    auto own_max = [&](int hf) { return NRT > 1 && my_rt > 0 ? m[NRT - 1][hf] : m[0][hf]; };

#pragma unroll 1
    for (; g < stop; ++g, ++it) {
      const int st = it % Smem::kStages;
      const uint32_t phase = (it / Smem::kStages) & 1;
      const int key0 = (int)(g - u.begin) * kPgKeys;
      const int buf = it & 1;
      pg_wait(sm.abort, smem_u32(&sm.full_k[st]), phase);
      // ---- S of this warp's rows and keys: two MMA chains (the dims' halves of each
      // 32 for 8 keys, or 2 x 8 keys)
      float s2[2][4];
#pragma unroll
      for (int i = 0; i < 4; ++i) s2[0][i] = s2[1][i] = 0.0f;
      const uint32_t kb = smem_u32(sm.k[st]);
      if constexpr (NRT == 1) {
        const int krow = my_key + (lane & 7), kchunk = lane >> 3;
#pragma unroll
        for (int d0 = 0; d0 < D; d0 += 32) {
          uint32_t b0, b1, b2, b3;
          ldmatrix_x4(kb + (d0 / 64) * (kPgKeys * 128) + pg_swz(krow, (d0 % 64) / 8 + kchunk), b0, b1, b2, b3);
          Mma<T>::run(s2[0], qf[d0 / 16], b0, b1);
          Mma<T>::run(s2[1], qf[d0 / 16 + 1], b2, b3);
        }
      } else {
        const int krow = my_key + (lane & 7) + 8 * (lane >> 4), kchunk = (lane >> 3) & 1;
#pragma unroll
        for (int d0 = 0; d0 < D; d0 += 16) {
          uint32_t b0, b1, b2, b3;
          ldmatrix_x4(kb + (d0 / 64) * (kPgKeys * 128) + pg_swz(krow, (d0 % 64) / 8 + kchunk), b0, b1, b2, b3);
          Mma<T>::run(s2[0], qf[d0 / 16], b0, b1);
          Mma<T>::run(s2[1], qf[d0 / 16], b2, b3);
        }
      }
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(smem_u32(&sm.empty_k[st]));
      float s[2][kOwn];  // [row half][keys 2 qc + e of each 8-key tile]
      float mw[2];
      bool grow = false;
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        float best = -INFINITY;
#pragma unroll
        for (int e = 0; e < kOwn; ++e) {
          const int key = key0 + my_key + 8 * (e >> 1) + 2 * qc + (e & 1);
          float x;
          if constexpr (NRT == 1) x = s2[0][2 * hf + e] + s2[1][2 * hf + e];
          else x = s2[e >> 1][2 * hf + (e & 1)];
          x = key < lim[hf] ? x * a.scale_log2 : -INFINITY;
          s[hf][e] = x;
          best = fmaxf(best, x);
        }
        best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, 1));
        best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, 2));
        mw[hf] = best;
        grow = grow || best > own_max(hf) + kPgHeadroom;
        if (a.scores != nullptr && 16 * my_rt + 8 * hf + qr < u.nrows) {
          float* dst = a.scores + (g * ROWS + 16 * my_rt + 8 * hf + qr) * kPgKeys + my_key + 2 * qc;
#pragma unroll
          for (int e = 0; e < kOwn; e += 2) *reinterpret_cast<float2*>(dst + 4 * e) = make_float2(s[hf][e], s[hf][e + 1]);
        }
      }
      // ---- P of these keys; a vote decides whether the maxima move first
      float pl[2];
      auto write_p = [&] {
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          const float base = own_max(hf) == -INFINITY ? 0.0f : own_max(hf);
          pl[hf] = 0.0f;
#pragma unroll
          for (int e = 0; e < kOwn; e += 2) {
            const float p0 = pg_exp2(s[hf][e] - base), p1 = pg_exp2(s[hf][e + 1] - base);
            pl[hf] += p0 + p1;
            *reinterpret_cast<uint32_t*>(sm.p[buf] + pg_swz(16 * my_rt + 8 * hf + qr, my_key / 8 + e / 2) + 4 * qc) =
                pack2_f32<T>(p0, p1);
          }
        }
      };
      write_p();
      if (tc::bar_or(1, 32 * kPgWarps, grow)) {
        if (qc == 0) {
          sm.mx[warp][qr] = mw[0];
          sm.mx[warp][8 + qr] = mw[1];
        }
        sync_warps();
#pragma unroll
        for (int rt = 0; rt < NRT; ++rt)
#pragma unroll
          for (int hf = 0; hf < 2; ++hf) {
            float best = m[rt][hf];
#pragma unroll
            for (int w = 0; w < kPgWarps / NRT; ++w) best = fmaxf(best, sm.mx[rt * (kPgWarps / NRT) + w][8 * hf + qr]);
            // NaN scores leave the maximum alone and reach O through P
            const float alpha = best == m[rt][hf] ? 1.0f : pg_exp2(m[rt][hf] - best);
            m[rt][hf] = best;
            if (rt == my_rt) l[hf] *= alpha;
#pragma unroll
            for (int n = 0; n < kNT; ++n) {
              o[rt][n][2 * hf] *= alpha;
              o[rt][n][2 * hf + 1] *= alpha;
            }
          }
        write_p();
        sync_warps();
      }
      l[0] += pl[0];
      l[1] += pl[1];
      // ---- O += P V over this warp's dims
      pg_wait(sm.abort, smem_u32(&sm.full_v[st]), phase);
      const int have = u.seq - key0;  // keys of the request in this tile
      if (have < kPgKeys) {
        // the rest of the last page (or what an earlier tile left) may hold anything: 0 * NaN
        const int clear = max(have, 0);
        for (int i = tid; i < (kPgKeys - clear) * (D / 8); i += 32 * kPgWarps) {
          const int row = clear + i / (D / 8), c = i % (D / 8);
          *reinterpret_cast<uint4*>(sm.v[st] + (c / 8) * (kPgKeys * 128) + row * 128 + (c % 8) * 16) = make_uint4(0, 0, 0, 0);
        }
        tc::fence_async_smem();
        sync_warps();
      }
      const uint32_t pb = smem_u32(sm.p[buf]), vb = smem_u32(sm.v[st]);
#pragma unroll
      for (int ks = 0; ks < kPgKeys / 16; ++ks) {
        uint32_t pa[NRT][4];
#pragma unroll
        for (int rt = 0; rt < NRT; ++rt)
          ldmatrix_x4(pb + pg_swz(16 * rt + (lane & 15), 2 * ks + (lane >> 4)), pa[rt][0], pa[rt][1], pa[rt][2], pa[rt][3]);
        if constexpr (kNT >= 2) {
#pragma unroll
          for (int n = 0; n < kNT; n += 2) {
            const int dim = warp * kWarpDims + 8 * n + 8 * (lane >> 4);
            uint32_t b0, b1, b2, b3;
            ldmatrix_x4_trans(vb + (dim / 64) * (kPgKeys * 128) + pg_swz(16 * ks + (lane & 15), (dim % 64) / 8), b0, b1, b2, b3);
#pragma unroll
            for (int rt = 0; rt < NRT; ++rt) {
              Mma<T>::run(o[rt][n], pa[rt], b0, b1);
              Mma<T>::run(o[rt][n + 1], pa[rt], b2, b3);
            }
          }
        } else {
          // 8 dims per warp: the four matrices cover 32 keys, every other k-step loads
          const int dim = warp * kWarpDims;
          uint32_t b0, b1, b2, b3;
          ldmatrix_x4_trans(vb + pg_swz((16 * (ks & ~1) + lane), dim / 8), b0, b1, b2, b3);
#pragma unroll
          for (int rt = 0; rt < NRT; ++rt) Mma<T>::run(o[rt][0], pa[rt], (ks & 1) ? b2 : b0, (ks & 1) ? b3 : b1);
        }
      }
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(smem_u32(&sm.empty_v[st]));
    }

    // ---- the row sums of all warps, then O / l or the piece of a divided unit
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      float v = l[hf];
      v += __shfl_xor_sync(0xffffffffu, v, 1);
      v += __shfl_xor_sync(0xffffffffu, v, 2);
      if (qc == 0) sm.sum[warp][8 * hf + qr] = v;
    }
    sync_warps();
    const int slot = 2 * (int)blockIdx.x + (seg_first == g0 ? 0 : 1);
#pragma unroll
    for (int rt = 0; rt < NRT; ++rt)
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        const int row = 16 * rt + 8 * hf + qr;
        if (row >= u.nrows) continue;
        float total = 0.0f;
#pragma unroll
        for (int w = 0; w < kPgWarps / NRT; ++w) total += sm.sum[rt * (kPgWarps / NRT) + w][8 * hf + qr];
        const float mm = m[rt][hf];
        if (whole) {
          const int rr = u.row0 + row, tok = rr / a.group;
          const int64_t orow = (int64_t)(u.q_start + tok) * a.hq + u.h * a.group + rr - tok * a.group;
          const bool empty = mm == -INFINITY && total == 0.0f;  // a row that sees no key
          const float inv = empty ? 0.0f : 1.0f / total;
          T* dst = reinterpret_cast<T*>(a.out) + orow * D + warp * kWarpDims + 2 * qc;
#pragma unroll
          for (int n = 0; n < kNT; ++n)
            *reinterpret_cast<uint32_t*>(dst + 8 * n) = pack2_f32<T>(o[rt][n][2 * hf] * inv, o[rt][n][2 * hf + 1] * inv);
          if (warp == 0 && qc == 0) {
            a.lse[orow] = empty ? -INFINITY : (mm == -INFINITY ? 0.0f : mm) * 0.69314718055994531f + logf(total);
            if (a.stats != nullptr) a.stats[orow] = make_float2(mm == -INFINITY ? 0.0f : mm, inv);
          }
        } else {
          float* dst = a.part_o + ((int64_t)slot * ROWS + row) * D + warp * kWarpDims + 2 * qc;
#pragma unroll
          for (int n = 0; n < kNT; ++n)
            *reinterpret_cast<float2*>(dst + 8 * n) = make_float2(o[rt][n][2 * hf], o[rt][n][2 * hf + 1]);
          if (warp == 0 && qc == 0) a.part_ml[(int64_t)slot * ROWS + row] = make_float2(mm, total);
        }
      }
    sync_warps();  // the sums are read before the next unit writes them
  }
}

// Combine of the divided units: a CTA of kPgMerge warps per (query token, head)
// row.  O = sum 2^(m_c - M) O_c / sum 2^(m_c - M) l_c; warp w takes pieces w, w + 4, ..
// of the row in CTA order (a lane D / 32 dims), then the warps' sums are added in
// warp order.  Rows of undivided units are done already.
template <int D, typename T, int ROWS>
__global__ void __launch_bounds__(32 * kPgMerge) paged_combine_kernel(const __grid_constant__ PagedArgs a,
                                                                      const __grid_constant__ PagedPlan p) {
  constexpr int E = D / 32;
  __shared__ float part[kPgMerge][D], part_l[kPgMerge];
  pdl_release();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int head = blockIdx.y, h = head / a.group;
  // tokens are numbered from the plan's first one
  const int tok_all = blockIdx.x + p.q_start[0];
  int lo = 0, hi = p.num_req;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (p.q_start[mid] <= tok_all) lo = mid; else hi = mid;
  }
  const int r = lo;
  const int tok = tok_all - p.q_start[r];
  const int rr = tok * a.group + head - h * a.group, row = rr % ROWS;
  const int nt = max(1, (p.seq[r] + kPgKeys - 1) / kPgKeys);
  const int64_t ub = p.tile_begin[r] + ((int64_t)(rr / ROWS) * a.hk + h) * nt;
  const int c0 = pg_find(p.cta_begin, p.ctas, ub), c1 = pg_find(p.cta_begin, p.ctas, ub + nt - 1);
  pdl_wait();
  // (a token of a request that another launch holds, or a row that one CTA finished)
  if (tok >= p.q_len[r] || c0 == c1) return;
  // the unit is the first piece of every CTA that begins inside it, else the last one
  const bool inside = p.cta_begin[c0] >= ub;
  auto piece = [&](int c) -> int64_t { return (int64_t)(2 * c + (c > c0 || inside ? 0 : 1)) * ROWS + row; };
  float M = -INFINITY;
  for (int c = c0 + lane; c <= c1; c += 32) M = fmaxf(M, a.part_ml[piece(c)].x);
  M = warp_max(M);
  const float base = M == -INFINITY ? 0.0f : M;
  float total = 0.0f, acc[E];
#pragma unroll
  for (int i = 0; i < E; ++i) acc[i] = 0.0f;
#pragma unroll 4
  for (int c = c0 + warp; c <= c1; c += kPgMerge) {
    const int64_t at = piece(c);
    const float2 ml = a.part_ml[at];
    const float f = pg_exp2(ml.x - base);  // a piece without visible keys: 2^-inf = 0
    const float* src = a.part_o + at * D + E * lane;
    total = fmaf(f, ml.y, total);
#pragma unroll
    for (int i = 0; i < E; i += 2) {
      const float2 v = *reinterpret_cast<const float2*>(src + i);
      acc[i] = fmaf(f, v.x, acc[i]);
      acc[i + 1] = fmaf(f, v.y, acc[i + 1]);
    }
  }
#pragma unroll
  for (int i = 0; i < E; ++i) part[warp][E * lane + i] = acc[i];
  if (lane == 0) part_l[warp] = total;
  __syncthreads();
  total = 0.0f;
#pragma unroll
  for (int w = 0; w < kPgMerge; ++w) total += part_l[w];
  const bool empty = M == -INFINITY && total == 0.0f;
  const float inv = empty ? 0.0f : 1.0f / total;
  const int64_t orow = (int64_t)tok_all * a.hq + head;
  if (2 * threadIdx.x < D) {
    float2 v = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int w = 0; w < kPgMerge; ++w) {
      v.x += part[w][2 * threadIdx.x];
      v.y += part[w][2 * threadIdx.x + 1];
    }
    reinterpret_cast<uint32_t*>(reinterpret_cast<T*>(a.out) + orow * D)[threadIdx.x] = pack2_f32<T>(v.x * inv, v.y * inv);
  }
  if (threadIdx.x == 0) {
    a.lse[orow] = empty ? -INFINITY : base * 0.69314718055994531f + logf(total);
    if (a.stats != nullptr) a.stats[orow] = make_float2(base, inv);
  }
}

// The keys' attention weights of requests with many query rows: scores are
// recomputed.  CTA = (request, 64-key tile) x kv head, K tile in shared memory;
// warp w takes the observed rows' 16-row blocks w, w + 8, ... that see the tile
// and sums p = exp2(s - m) / l over its rows in registers.
template <int D, typename T>
__global__ void __launch_bounds__(32 * kPgWarps) paged_mass_rows_kernel(const __grid_constant__ PagedArgs a,
                                                                        const __grid_constant__ PagedPlan p,
                                                                        const T* k_cache, int64_t kcb, int64_t kct,
                                                                        int64_t kch) {
  extern __shared__ __align__(1024) uint8_t pg_raw[];
  __shared__ float part[kPgWarps][kPgKeys];
  pdl_release();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  // tile_begin counts 64-key tiles per request here
  const int r = pg_find(p.tile_begin, p.num_req, blockIdx.x), h = blockIdx.y;
  const int key0 = (int)(blockIdx.x - p.tile_begin[r]) * kPgKeys;
  const int q_len = p.q_len[r], seq = p.seq[r];
  const int32_t* row = a.table + (int64_t)p.req_id[r] * a.table_stride;
  pdl_wait();
  for (int i = tid; i < kPgKeys * (D / 8); i += 32 * kPgWarps) {
    const int key = i / (D / 8), c = i % (D / 8);
    uint4 v = make_uint4(0, 0, 0, 0);
    if (key0 + key < seq) {
      const int64_t blk = row[a.page.div(key0 + key)];
      if (blk >= 0 && blk < a.num_blocks)
        v = *reinterpret_cast<const uint4*>(k_cache + blk * kcb + (int64_t)a.page.mod(key0 + key) * kct + h * kch + 8 * c);
    }
    *reinterpret_cast<uint4*>(pg_raw + (c / 8) * (kPgKeys * 128) + pg_swz(key, c % 8)) = v;
  }
  __syncthreads();
  const int qr = lane >> 2, qc = lane & 3;
  // rows that are observed and see at least the tile's first key
  const int tok_first = max(max(0, q_len - a.observe), key0 - (seq - q_len));
  const int row_first = tok_first * a.group, row_end = q_len * a.group;
  float sum[kPgKeys / 8][2];
#pragma unroll
  for (int n = 0; n < kPgKeys / 8; ++n) sum[n][0] = sum[n][1] = 0.0f;
  const uint32_t kb = smem_u32(pg_raw);
#pragma unroll 1
  for (int rb = row_first + 16 * warp; rb < row_end; rb += 16 * kPgWarps) {
    float s[kPgKeys / 8][4];
#pragma unroll
    for (int n = 0; n < kPgKeys / 8; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) s[n][i] = 0.0f;
    const T* src[2];
    float2 st[2];
    int lim[2];
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      const int rr = rb + 8 * hf + qr, tok = rr / a.group;
      const bool live = rr < row_end;
      const int64_t t = p.q_start[r] + (live ? tok : 0);
      const int head = h * a.group + (live ? rr - tok * a.group : 0);
      src[hf] = reinterpret_cast<const T*>(a.q) + t * a.q_tok + head * a.q_head;
      st[hf] = a.stats[t * a.hq + head];
      lim[hf] = live ? seq - q_len + tok + 1 : 0;
    }
#pragma unroll 4
    for (int d0 = 0; d0 < D; d0 += 16) {
      uint32_t qa[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) qa[i] = *reinterpret_cast<const uint32_t*>(src[i & 1] + d0 + 8 * (i >> 1) + 2 * qc);
#pragma unroll
      for (int n = 0; n < kPgKeys / 8; n += 2) {
        uint32_t b0, b1, b2, b3;
        ldmatrix_x4(kb + (d0 / 64) * (kPgKeys * 128) + pg_swz(8 * n + (lane & 7) + 8 * (lane >> 4), (d0 % 64) / 8 + ((lane >> 3) & 1)),
                    b0, b1, b2, b3);
        Mma<T>::run(s[n], qa, b0, b1);
        Mma<T>::run(s[n + 1], qa, b2, b3);
      }
    }
#pragma unroll
    for (int n = 0; n < kPgKeys / 8; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int key = key0 + 8 * n + 2 * qc + (i & 1), hf = i >> 1;
        if (key < lim[hf]) sum[n][i & 1] = fmaf(pg_exp2(fmaf(s[n][i], a.scale_log2, -st[hf].x)), st[hf].y, sum[n][i & 1]);
      }
  }
#pragma unroll
  for (int n = 0; n < kPgKeys / 8; ++n)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float v = sum[n][e];
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
      if (qr == 0) part[warp][8 * n + 2 * qc + e] = v;
    }
  __syncthreads();
  const int key = key0 + tid;
  if (tid >= kPgKeys || key >= seq) return;
  float total = 0.0f;
#pragma unroll
  for (int w = 0; w < kPgWarps; ++w) total += part[w][tid];
  const int64_t blk = row[a.page.div(key)];
  if (blk < 0 || blk >= a.num_blocks) return;  // flagged by the attention pass
  float* w = a.weights + (blk * a.hk + h) * a.bs + a.page.mod(key);
  if (key < seq - q_len)
    atomicAdd(w, total);
  else
    *w = total;
}

// The keys' attention weights from stored scores (few query rows): a thread per
// (key, kv head) sums exp2(s - m) / l over the observed rows.  A key of the
// chunk itself starts from zero, an older one adds to what it has.  Bound by
// reading the scores, 8 rows in flight per thread.
template <int ROWS>
__global__ void __launch_bounds__(kPgKeys) paged_mass_kernel(const __grid_constant__ PagedArgs a,
                                                             const __grid_constant__ PagedPlan p) {
  __shared__ float2 st[ROWS];
  pdl_release();
  const int64_t g = blockIdx.x;
  const PagedUnit u = pg_unit<ROWS>(p, a, g);
  const int key = (int)(g - u.begin) * kPgKeys + threadIdx.x;
  const int page = key < u.seq ? (int)a.page.div(key) : 0;
  pdl_wait();
  const int64_t blk = key < u.seq ? a.table[(int64_t)p.req_id[u.r] * a.table_stride + page] : -1;
  const int first = max(0, u.q_len - a.observe) * a.group;  // first observed row
  for (int i = threadIdx.x; i < u.nrows; i += kPgKeys) {
    const int tok = i / a.group;
    st[i] = a.stats[(int64_t)(u.q_start + tok) * a.hq + u.h * a.group + i - tok * a.group];
  }
  __syncthreads();
  if (blk < 0 || blk >= a.num_blocks) return;  // past the request, or flagged by the attention pass
  float sum = 0.0f;
  const float* s = a.scores + g * ROWS * kPgKeys + threadIdx.x;
#pragma unroll 8
  for (int i = first; i < u.nrows; ++i) sum = fmaf(pg_exp2(s[i * kPgKeys] - st[i].x), st[i].y, sum);
  float* w = a.weights + (blk * a.hk + u.h) * a.bs + (key - page * a.bs);
  if (key < u.seq - u.q_len)
    atomicAdd(w, sum);  // requests may share a page of history
  else
    *w = sum;
}

}  // namespace oscar
