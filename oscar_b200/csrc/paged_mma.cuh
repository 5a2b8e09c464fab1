// Attention of few query rows over a short paged 16-bit cache on mma.sync: the
// same units, pieces and plan as paged_attn.cuh's kFew form (at most 32 live
// rows), for steps whose keys are few.
//
// It has no tensor memory to allocate, no padded rows and a short epilogue, so a
// small step ends sooner (one token on 8192 keys, Hq 24 / Hk 4 / D 256: 11.5
// against 20.5 us); its operand reads fill the shared-memory bandwidth that the
// copies leave, so per 64-key tile it takes longer (8 requests x 24580 keys: 147
// against 131 us).  The two meet near 32 tiles per SM.
//
// Tile.  One warp issues TMA boxes into a ring of stages; eight warps compute.
// For S a warp takes 8 of the tile's 64 keys against 16 rows (16 keys and half of
// the rows when there are 32: the Q fragments then still fit the registers), for
// O it takes D / 8 of the dims against all keys, so a row's accumulators are
// spread over the warps.  P goes through shared memory (two buffers); its one
// barrier per tile also carries the vote whether a row's maximum grew by more
// than kPgHeadroom (log2 units): only then do the warps exchange maxima and
// rescale.
#pragma once

#include "paged_attn.cuh"

namespace oscar {

constexpr int kPgThreads = 32 * (kPgWarps + 1);

template <int D, int NRT>
struct PsSmem {
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

// Producer: one warp.  Lane i holds the block of box (base + i) of the piece, the
// next 32 boxes' blocks are fetched one group ahead; one elected lane issues (lanes
// with operands of their own would be serialised).
template <int D, typename Smem, typename Walk>
OSCAR_DEVINL void ps_produce(Smem& sm, const PagedArgs& a, const PcPlan& p, const CUtensorMap* kmap,
                             const CUtensorMap* vmap, Walk w, int lane) {
  constexpr int kPanels = D / 64, kSt = Smem::kStages;
  const int per = kPgKeys / a.box;  // boxes per tile
  const uint32_t box = (uint32_t)a.box, box_bytes = box * 128u;
  uint32_t it = 0;
  bool ok = true;
  for (; w.live() && ok; w.next(a.hk)) {
    const int32_t* row = a.table + (int64_t)p.req_id[w.r] * a.table_stride;
    const int boxes = (p.seq[w.r] + a.box - 1) / a.box;  // of the whole request
    auto fetch = [&](int b) -> int { return b < boxes ? row[a.page.div((uint32_t)b * box)] : -1; };
    int base = w.t * per;
    int cur = fetch(base + lane), nxt = fetch(base + 32 + lane);
    for (int t = w.t; t < w.t_end; ++t, ++it) {
      const int st = it % kSt;
      const uint32_t phase = (it / kSt) & 1;
      const int first = t * per;  // first box of the tile
      const int live = max(0, min(per, boxes - first));
      const uint32_t bytes = (uint32_t)live * box_bytes * kPanels;
      const uint32_t fk = smem_u32(&sm.full_k[st]), fv = smem_u32(&sm.full_v[st]);
      if (it >= kSt) {
        const bool k_free = pg_wait(sm.abort, smem_u32(&sm.empty_k[st]), phase ^ 1, a.tries);
        const bool v_free = pg_wait(sm.abort, smem_u32(&sm.empty_v[st]), phase ^ 1, a.tries);
        if (!__all_sync(0xffffffffu, k_free && v_free)) {
          ok = false;  // gave up: issue nothing more
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
            tma_load_4d(smem_u32(sm.k[st]) + pn * (kPgKeys * 128u) + at, kmap, pn * 64, w.h, off, blk, fk);
#pragma unroll
          for (int pn = 0; pn < kPanels; ++pn)
            tma_load_4d(smem_u32(sm.v[st]) + pn * (kPgKeys * 128u) + at, vmap, pn * 64, w.h, off, blk, fv);
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
paged_attn_mma_kernel(const __grid_constant__ PagedArgs a, const __grid_constant__ PcPlan p,
                   const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap) {
  constexpr int kSteps = D / 16;        // MMA k-steps of S
  constexpr int kWarpDims = D / kPgWarps;
  constexpr int kNT = kWarpDims / 8;    // 8-dim output tiles of a warp
  constexpr int kOwn = NRT == 1 ? 2 : 4;  // scores of a thread and row
  using Smem = PsSmem<D, NRT>;
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
  using Walk = PcWalk<PcShape<D, true>>;
  Walk w(p, blockIdx.x);
  const int64_t tile0 = p.first[blockIdx.x];
  pdl_wait();
  if (warp == kPgWarps) {
    ps_produce<D>(sm, a, p, &kmap, &vmap, w, lane);
    return;
  }

  const int qr = lane >> 2, qc = lane & 3;  // row and column pair of a fragment
  // S: 8 keys x 16 rows per warp, or (32 rows) 16 keys x one of the two 16-row tiles
  const int my_rt = NRT == 1 ? 0 : warp / 4;
  const int my_key = NRT == 1 ? 8 * warp : 16 * (warp % 4);
  auto sync_warps = [&] { tc::bar_sync(1, 32 * kPgWarps); };
  uint32_t it = 0;
  for (; w.live(); w.next(a.hk)) {
    const int q_start = p.q_start[w.r], q_len = p.q_len[w.r], seq = p.seq[w.r];
    const int nrows = q_len * a.group;  // row: token * group + head in group
    const bool whole = w.t == 0 && w.t_end == w.nt;

    // Q fragments of this warp's 16 rows (rows qr, qr + 8) and their visible key counts
    uint32_t qf[kSteps][4];
    int lim[2];
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      const int row = 16 * my_rt + 8 * hf + qr;
      const bool live = row < nrows;
      const int tok = row / a.group;
      lim[hf] = live ? max(0, seq - q_len + tok + 1) : 0;
      const T* src = reinterpret_cast<const T*>(a.q) + (int64_t)(q_start + tok) * a.q_tok +
                     (int64_t)(w.h * a.group + row - tok * a.group) * a.q_head;
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
    for (int t = w.t; t < w.t_end; ++t, ++it) {
      const int st = it % Smem::kStages;
      const uint32_t phase = (it / Smem::kStages) & 1;
      const int key0 = t * kPgKeys;
      const int buf = it & 1;
      pg_wait(sm.abort, smem_u32(&sm.full_k[st]), phase, a.tries);
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
        if (a.scores != nullptr && 16 * my_rt + 8 * hf + qr < nrows) {
          float* dst = a.scores + ((tile0 + it) * a.score_rows + 16 * my_rt + 8 * hf + qr) * kPgKeys + my_key + 2 * qc;
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
                pc_pack<T>(p0, p1);
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
            for (int v = 0; v < kPgWarps / NRT; ++v) best = fmaxf(best, sm.mx[rt * (kPgWarps / NRT) + v][8 * hf + qr]);
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
      pg_wait(sm.abort, smem_u32(&sm.full_v[st]), phase, a.tries);
      const int have = seq - key0;  // keys of the request in this tile
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
    const int64_t piece = (int64_t)(2 * blockIdx.x + (w.piece == 0 ? 0 : 1)) * kPcRows;
#pragma unroll
    for (int rt = 0; rt < NRT; ++rt)
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        const int row = 16 * rt + 8 * hf + qr;
        if (row >= nrows) continue;
        float total = 0.0f;
#pragma unroll
        for (int v = 0; v < kPgWarps / NRT; ++v) total += sm.sum[rt * (kPgWarps / NRT) + v][8 * hf + qr];
        const float mm = m[rt][hf];
        if (whole) {
          const int tok = row / a.group;
          const int64_t orow = (int64_t)(q_start + tok) * a.hq + w.h * a.group + row - tok * a.group;
          const bool empty = mm == -INFINITY && total == 0.0f;  // a row that sees no key
          const float inv = empty ? 0.0f : 1.0f / total;
          T* dst = reinterpret_cast<T*>(a.out) + orow * D + warp * kWarpDims + 2 * qc;
#pragma unroll
          for (int n = 0; n < kNT; ++n)
            *reinterpret_cast<uint32_t*>(dst + 8 * n) = pc_pack<T>(o[rt][n][2 * hf] * inv, o[rt][n][2 * hf + 1] * inv);
          if (warp == 0 && qc == 0) {
            a.lse[orow] = empty ? -INFINITY : (mm == -INFINITY ? 0.0f : mm) * 0.69314718055994531f + logf(total);
            if (a.stats != nullptr) a.stats[orow] = make_float2(mm == -INFINITY ? 0.0f : mm, inv);
          }
        } else {
          float* dst = a.part_o + (piece + row) * D + warp * kWarpDims + 2 * qc;
#pragma unroll
          for (int n = 0; n < kNT; ++n)
            *reinterpret_cast<float2*>(dst + 8 * n) = make_float2(o[rt][n][2 * hf], o[rt][n][2 * hf + 1]);
          if (warp == 0 && qc == 0) a.part_ml[piece + row] = make_float2(mm, total);
        }
      }
    sync_warps();  // the sums are read before the next unit writes them
  }
}

}  // namespace oscar
