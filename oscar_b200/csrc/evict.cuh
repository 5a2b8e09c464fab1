// Eviction from a 16-bit paged cache by accumulated attention weight.
//
// Per request and kv head, of the positions [0, seq): the first `sink`, the last
// `recent` and, of those between, the keep - sink - recent heaviest (ties to the
// lower position) stay, in order; their K, V and weight slots move to positions
// 0, 1, ... of the destination pages.  The destination may be the request's own
// pages: the j-th kept position is never below j, so moving in ascending order
// never overwrites a slot that is still to be read.
//
// evict_select_kernel (a cluster of 8 CTAs per request and head, each with an eighth
// of the positions) finds the weight of the last key that stays by histograms over
// order-preserving 32-bit keys: each round spreads the range that still holds it,
// [lo, hi], over 256 bins (the keys' own minimum and maximum first, so that
// neighbouring threads rarely count in the same bin) and narrows it to one bin,
// four rounds at most; the CTAs add up each other's bins over distributed shared
// memory (2048 bins and three rounds: those reads cost more than a round saves).
// Then each warp walks its own stretch of the positions twice: it counts its kept
// keys, and after prefix sums over the warps and the CTAs numbers them and writes
// their list; then the list's weights move, coalesced.  Bound by instructions: one
// CTA per request and head took 48 us for 8 x 4 heads of 24580 keys and 26 us for 4
// heads of 9256.  With the copy, 8 x 4 heads of 24580 keys cut to 12288 take 178 us
// (512 threads a CTA: 183), 4 heads of 9256 cut to 4096 take 25 us.  Up to 8 kEvCached
// weights are held in shared memory; a longer request is read again for each round
// and walked piece by piece.
//
// To other pages every row is independent and evict_copy_kernel is bound by bytes.
// In place (evict_move_kernel) a CTA owns a 128-byte slice of one head's K or V
// rows and walks the list in ascending order: it holds 256 rows' slices in
// registers between the read and the write of a step, and the next step's
// reads are already in flight.  A step's chain of loads (list, table, row) and
// the few CTAs of a request (32 with 4 heads at D 256) keep it from the bytes'
// rate: 8 x 24580 keys cut to 12288 take 441 us, one request's 9256 cut to 4096
// 138 us (181 and 30 us to other pages, timed the same way).
#pragma once

#include "paged_attn.cuh"

namespace oscar {

constexpr int kEvReqs = 256;
constexpr int kEvThreads = 1024;
constexpr int kEvCached = 16384;  // weights in a CTA's shared memory
constexpr int kEvCluster = 8;
constexpr int kEvBins = 256;
constexpr int kEvMoveThreads = 256;
constexpr int kEvRows = 4;   // rows per thread and step of the copy
constexpr int kEvWaves = 8;  // rows per thread and step of the in-place move

struct EvictPlan {
  int num_req;
  int req_id[kEvReqs];
  int seq[kEvReqs];
};

struct EvictArgs {
  uint8_t *k, *v;
  int64_t kb, kt, kh, vb, vt, vh;  // cache strides in bytes
  float* weights;                  // [num_blocks, hk, bs]
  int64_t num_blocks;
  int bs, hk;
  FastDiv page;                    // by bs
  int row_bytes;                   // D * 2
  const int32_t *table, *dst;      // dst == table: in place
  int64_t table_stride, dst_stride;
  int keep, sink, recent;
  int32_t* kept;                   // [num_requests, hk, kept_stride], -1 past a head's list
  int kept_stride;
};

// order-preserving key: a < b as floats <=> key(a) < key(b); -0 and 0 are equal, NaN is above every number
OSCAR_DEVINL uint32_t ev_key(float w) {
  if (w != w) return 0xffffffffu;
  const uint32_t b = __float_as_uint(w + 0.0f);
  return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}

// The weight of a position, or null outside the cache.  (The caller flags the error after its loop:
// an atomic inside would keep the loop's loads from overlapping)
OSCAR_DEVINL float* ev_weight(const EvictArgs& a, const int32_t* row, int h, int pos) {
  const int page = (int)a.page.div(pos);
  const int64_t blk = __ldg(row + page);
  if (blk < 0 || blk >= a.num_blocks) return nullptr;
  return a.weights + (blk * a.hk + h) * a.bs + (pos - page * a.bs);
}

OSCAR_DEVINL uint32_t ev_remote(uint32_t addr, uint32_t rank) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];\n" : "=r"(v) : "r"(pc_map(addr, rank)) : "memory");
  return v;
}
OSCAR_DEVINL uint2 ev_remote2(uint32_t addr, uint32_t rank) {  // two words of CTA `rank`'s shared memory
  uint2 v;
  asm volatile("ld.shared::cluster.v2.u32 {%0, %1}, [%2];\n" : "=r"(v.x), "=r"(v.y) : "r"(pc_map(addr, rank)) : "memory");
  return v;
}

__global__ void __launch_bounds__(kEvThreads) evict_select_kernel(const __grid_constant__ EvictArgs a,
                                                                  const __grid_constant__ EvictPlan p) {
  extern __shared__ __align__(16) float ev_w[];
  __shared__ __align__(8) uint32_t bins[kEvBins];
  __shared__ uint32_t warp_sum[2][32];
  // for the other CTAs; two places, since with all keys equal nothing but the walk's own barrier lies
  // between a slow CTA's read of the range and a fast CTA's counts
  __shared__ __align__(8) uint32_t range[2];   // minimum and maximum
  __shared__ __align__(8) uint32_t counts[2];  // kept and equal keys of a piece
  __shared__ uint32_t pick[2];
  pdl_release();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = (int)pc_rank();
  const int r = blockIdx.x / kEvCluster, h = blockIdx.y;
  const int seq = p.seq[r];
  const int32_t* src_row = a.table + (int64_t)p.req_id[r] * a.table_stride;
  const int32_t* dst_row = a.dst + (int64_t)p.req_id[r] * a.dst_stride;
  int32_t* kept = a.kept + ((int64_t)p.req_id[r] * a.hk + h) * a.kept_stride;
  const int n = min(seq, a.keep);
  const bool all = seq <= a.keep;
  constexpr int kPiece = kEvCluster * kEvCached;
  bool bad = false;
  if (tid == 0) range[0] = 0xffffffffu, range[1] = 0u;
  pdl_wait();
  for (int j = n + rank * kEvThreads + tid; j < a.kept_stride; j += kEvCluster * kEvThreads) kept[j] = -1;
  // this CTA's positions of the piece that begins at `first`, and their weights to shared memory
  int from = 0, to = 0;
  auto load = [&](int first) {
    const int end = min(seq, first + kPiece);
    const int per = ((end - first + kEvCluster - 1) / kEvCluster + 31) / 32 * 32;
    from = min(end, first + rank * per);
    to = min(end, from + per);
#pragma unroll 4
    for (int i = from + tid; i < to; i += kEvThreads) {
      const float* w = ev_weight(a, src_row, h, i);
      bad = bad || w == nullptr;
      ev_w[i - from] = w == nullptr ? 0.0f : *w;
    }
    __syncthreads();
  };
  load(0);

  // the key value at which the list is full, and how many of the keys that equal it stay
  const int lo_pos = a.sink, hi_pos = seq - a.recent;
  uint32_t threshold = 0, need = (uint32_t)max(0, a.keep - a.sink - a.recent);
  // calls f(key) for this CTA's keys between sink and recent, in any order
  auto each = [&](auto&& f) {
    for (int first = 0; first < seq; first += kPiece) {
      if (seq > kPiece) {
        __syncthreads();
        load(first);
      }
      const int i0 = max(lo_pos, from), i1 = min(hi_pos, to);
#pragma unroll 4
      for (int i = i0 + tid; i < i1; i += kEvThreads) f(ev_key(ev_w[i - from]));
    }
  };
  if (!all && need > 0) {  // (the same for all CTAs of the cluster)
    uint32_t least = 0xffffffffu, most = 0u;
    each([&](uint32_t key) {
      least = min(least, key);
      most = max(most, key);
    });
    least = __reduce_min_sync(0xffffffffu, least);
    most = __reduce_max_sync(0xffffffffu, most);
    if (lane == 0) {
      atomicMin(&range[0], least);
      atomicMax(&range[1], most);
    }
    pc_cluster_sync();
    const uint2 theirs = ev_remote2(smem_u32(range), lane % kEvCluster);
    uint32_t lo = __reduce_min_sync(0xffffffffu, theirs.x), hi = __reduce_max_sync(0xffffffffu, theirs.y);
    // Every round leaves one bin of at most 1 / 128 of the range, so there are four at most, and all
    // CTAs take the same bin, since they add up the same counts.  (Keys read again from memory that
    // somebody is writing may have too few for `need`: then the lowest bin is as good as any)
#pragma unroll 1
    while (lo < hi) {
      // bins of 2^shift keys, at most 256 of them
      const int shift = max(0, 32 - __clz(hi - lo) - 8);
      for (int i = tid; i < kEvBins; i += kEvThreads) bins[i] = 0;
      if (tid == 0) pick[0] = 0, pick[1] = need;
      __syncthreads();
      each([&](uint32_t key) {
        if (key >= lo && key <= hi) atomicAdd(&bins[(key - lo) >> shift], 1u);
      });
      pc_cluster_sync();
      // count from the top: thread t holds bin 255 - t of all CTAs
      static_assert(kEvBins <= kEvThreads, "a thread per bin");
      const int bin = kEvBins - 1 - tid;
      uint32_t own = 0;
      if (bin >= 0) {
#pragma unroll
        for (int t = 0; t < kEvCluster; ++t) own += ev_remote(smem_u32(&bins[bin]), t);
      }
      uint32_t sum = own;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t x = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += x;
      }
      if (lane == 31) warp_sum[0][warp] = sum;
      __syncthreads();
      uint32_t before = lane < warp ? warp_sum[0][lane] : 0u;
      before = __reduce_add_sync(0xffffffffu, before) + sum - own;
      if (before < need && before + own >= need) pick[0] = bin, pick[1] = need - before;
      __syncthreads();
      lo += pick[0] << shift;
      hi = lo + min(hi - lo, (1u << shift) - 1u);  // (lo + 2^shift may pass 32 bits)
      need = pick[1];
      pc_cluster_sync();  // every CTA has read the bins
    }
    threshold = lo;
  }

  // ordered walk: the kept keys are the fixed ones, those above the threshold and the first `need`
  // that equal it
  uint32_t out = 0, equal = 0;  // kept keys and equal keys of the pieces before
  const bool chooses = !all && a.keep > a.sink + a.recent;
  for (int first = 0; first < seq; first += kPiece) {
    if (seq > kPiece) {
      __syncthreads();
      load(first);
    }
    constexpr int kWarps = kEvThreads / 32;
    const int per = ((to - from + kWarps - 1) / kWarps + 31) / 32 * 32;  // positions of a warp
    const int w0 = min(to, from + warp * per), w1 = min(to, w0 + per);
    auto classify = [&](int i, bool& sure, bool& same) {
      sure = same = false;
      if (i >= w1) return;
      const bool fixed = all || i < lo_pos || i >= hi_pos;
      const uint32_t key = ev_key(ev_w[i - from]);
      sure = fixed || (chooses && key > threshold);
      same = !fixed && chooses && key == threshold;
    };
    uint32_t sures = 0, sames = 0;
    for (int i0 = w0; i0 < w1; i0 += 32) {
      bool sure, same;
      classify(i0 + lane, sure, same);
      sures += __popc(__ballot_sync(0xffffffffu, sure));
      sames += __popc(__ballot_sync(0xffffffffu, same));
    }
    if (lane == 0) warp_sum[0][warp] = sures, warp_sum[1][warp] = sames;
    __syncthreads();
    // before this warp in the CTA: kept keys that do not depend on the rank of equal ones, and equal keys
    uint32_t a_cnt = lane < kWarps ? warp_sum[0][lane] : 0u, e_cnt = lane < kWarps ? warp_sum[1][lane] : 0u;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t x = __shfl_up_sync(0xffffffffu, a_cnt, o), y = __shfl_up_sync(0xffffffffu, e_cnt, o);
      if (lane >= o) a_cnt += x, e_cnt += y;
    }
    const uint32_t a_all = __shfl_sync(0xffffffffu, a_cnt, 31), e_all = __shfl_sync(0xffffffffu, e_cnt, 31);
    if (tid == 0) counts[0] = a_all, counts[1] = e_all;
    pc_cluster_sync();
    // and in the CTAs before this one
    const uint2 theirs = ev_remote2(smem_u32(counts), lane % kEvCluster);
    const uint32_t a_before = __reduce_add_sync(0xffffffffu, lane < rank ? theirs.x : 0u);
    const uint32_t e_before = equal + __reduce_add_sync(0xffffffffu, lane < rank ? theirs.y : 0u);
    const uint32_t a_piece = __reduce_add_sync(0xffffffffu, lane < kEvCluster ? theirs.x : 0u);
    const uint32_t e_piece = __reduce_add_sync(0xffffffffu, lane < kEvCluster ? theirs.y : 0u);
    const uint32_t cta_out = out + a_before + (min(e_before, need) - min(equal, need));
    uint32_t eq = e_before + __shfl_sync(0xffffffffu, e_cnt, warp) - sames;
    uint32_t j0 = cta_out + __shfl_sync(0xffffffffu, a_cnt, warp) - sures + (min(eq, need) - min(e_before, need));
    for (int i0 = w0; i0 < w1; i0 += 32) {
      const int i = i0 + lane;
      bool sure, same;
      classify(i, sure, same);
      const uint32_t sb = __ballot_sync(0xffffffffu, sure), eb = __ballot_sync(0xffffffffu, same);
      const uint32_t below = (1u << lane) - 1u;
      const uint32_t order = eq + __popc(eb & below);  // of an equal key
      const uint32_t j = j0 + __popc(sb & below) + (min(order, need) - min(eq, need));
      if ((sure || (same && order < need)) && (int)j < n) kept[j] = i;
      const uint32_t eq_next = eq + __popc(eb);
      j0 += __popc(sb) + (min(eq_next, need) - min(eq, need));
      eq = eq_next;
    }
    const uint32_t cta_end = min((uint32_t)n, cta_out + a_all + (min(e_before + e_all, need) - min(e_before, need)));
    __syncthreads();  // this CTA's part of the list is written (and all weights of the piece are in shared memory)
#pragma unroll 4
    for (uint32_t j = cta_out + tid; j < cta_end; j += kEvThreads) {
      float* dst = ev_weight(a, dst_row, h, (int)j);
      bad = bad || dst == nullptr;
      if (dst != nullptr) *dst = ev_w[kept[j] - from];
    }
    out = min((uint32_t)n, out + a_piece + (min(equal + e_piece, need) - min(equal, need)));
    equal += e_piece;
    pc_cluster_sync();  // the counts have been read; no CTA ends while another reads its shared memory
  }
  // (as above: places that keys read again have left empty)
  for (int j = (int)out + rank * kEvThreads + tid; j < n; j += kEvCluster * kEvThreads) kept[j] = -1;
  if (bad) flag_error(2u);
}

// To other pages: 16 bytes of a kept row's K and V per lane, 4 rows in flight; the list and the
// block tables of a step are read while the rows of the step before it move.
__global__ void __launch_bounds__(kEvMoveThreads) evict_copy_kernel(const __grid_constant__ EvictArgs a,
                                                                    const __grid_constant__ EvictPlan p) {
  pdl_release();
  const int lanes = a.row_bytes / 16;  // 8, 16 or 32 lanes per row
  const int r = blockIdx.y / a.hk, h = blockIdx.y % a.hk;
  const int n = min(p.seq[r], a.keep);
  const int32_t* src_row = a.table + (int64_t)p.req_id[r] * a.table_stride;
  const int32_t* dst_row = a.dst + (int64_t)p.req_id[r] * a.dst_stride;
  const int32_t* kept = a.kept + ((int64_t)p.req_id[r] * a.hk + h) * a.kept_stride;
  const int c = threadIdx.x % lanes, rows = kEvMoveThreads / lanes, mine = threadIdx.x / lanes;
  const int step = gridDim.x * rows * kEvRows;
  uint8_t* const k = a.k + h * a.kh + 16 * c;
  uint8_t* const v = a.v + h * a.vh + 16 * c;
  pdl_wait();
  struct Move {
    int sb, so, db, dof;  // source and destination block and place; sb < 0: nothing to move
  } m[kEvRows];
  auto look_up = [&](int j0) {
#pragma unroll
    for (int i = 0; i < kEvRows; ++i) {
      const int j = j0 + i * rows + mine;
      m[i].sb = -1;
      if (j >= n) continue;
      const int s = kept[j], sp = (int)a.page.div(max(s, 0)), dp = (int)a.page.div(j);
      const int sb = src_row[sp], db = dst_row[dp];
      // an empty place, or a block that the selection has flagged (one test: the loads stay in flight)
      if (s < 0 || sb < 0 || sb >= a.num_blocks || db < 0 || db >= a.num_blocks) continue;
      m[i] = Move{sb, s - sp * a.bs, db, j - dp * a.bs};
    }
  };
  int j0 = blockIdx.x * rows * kEvRows;
  look_up(j0);
#pragma unroll 1
  for (; j0 < n; j0 += step) {
    uint4 kv[kEvRows], vv[kEvRows];
    int64_t to_k[kEvRows], to_v[kEvRows];
#pragma unroll
    for (int i = 0; i < kEvRows; ++i) {
      to_k[i] = -1;
      if (m[i].sb < 0) continue;
      kv[i] = __ldcs(reinterpret_cast<const uint4*>(k + m[i].sb * a.kb + m[i].so * a.kt));
      vv[i] = __ldcs(reinterpret_cast<const uint4*>(v + m[i].sb * a.vb + m[i].so * a.vt));
      to_k[i] = m[i].db * a.kb + m[i].dof * a.kt;
      to_v[i] = m[i].db * a.vb + m[i].dof * a.vt;
    }
    look_up(j0 + step);
#pragma unroll
    for (int i = 0; i < kEvRows; ++i) {
      if (to_k[i] < 0) continue;
      __stcs(reinterpret_cast<uint4*>(k + to_k[i]), kv[i]);
      __stcs(reinterpret_cast<uint4*>(v + to_v[i]), vv[i]);
    }
  }
}

// In place: CTA = (request, head) x (K | V) x 128-byte slice of the rows.
__global__ void __launch_bounds__(kEvMoveThreads) evict_move_kernel(const __grid_constant__ EvictArgs a,
                                                                    const __grid_constant__ EvictPlan p) {
  constexpr int kRows = kEvMoveThreads / 8;     // rows per wave
  constexpr int kStep = kRows * kEvWaves;
  pdl_release();
  const int r = blockIdx.x / a.hk, h = blockIdx.x % a.hk;
  const int n = min(p.seq[r], a.keep);
  if (p.seq[r] <= a.keep) {  // nothing moves
    pdl_wait();
    return;
  }
  uint8_t* base = blockIdx.y ? a.v : a.k;
  const int64_t sb = blockIdx.y ? a.vb : a.kb, stt = blockIdx.y ? a.vt : a.kt, sh = blockIdx.y ? a.vh : a.kh;
  base += h * sh + 128 * blockIdx.z + 16 * (threadIdx.x % 8);
  const int32_t* row = a.table + (int64_t)p.req_id[r] * a.table_stride;
  const int32_t* kept = a.kept + ((int64_t)p.req_id[r] * a.hk + h) * a.kept_stride;
  pdl_wait();
  auto slot = [&](int pos) -> uint8_t* {
    const int64_t blk = row[a.page.div(pos)];
    return blk < 0 || blk >= a.num_blocks ? nullptr : base + blk * sb + (int64_t)a.page.mod(pos) * stt;
  };
  uint4 x[2][kEvWaves];
  auto read = [&](int j0, uint4 (&y)[kEvWaves]) {
#pragma unroll
    for (int i = 0; i < kEvWaves; ++i) {
      const int j = j0 + i * kRows + threadIdx.x / 8;
      if (j >= n) continue;
      const int s = kept[j];
      const uint8_t* from = s == j || s < 0 ? nullptr : slot(s);
      if (from != nullptr) y[i] = *reinterpret_cast<const uint4*>(from);
    }
  };
  auto write = [&](int j0, const uint4 (&y)[kEvWaves]) {
#pragma unroll
    for (int i = 0; i < kEvWaves; ++i) {
      const int j = j0 + i * kRows + threadIdx.x / 8;
      if (j >= n) continue;
      const int s = kept[j];
      if (s == j || s < 0 || slot(s) == nullptr) continue;
      uint8_t* to = slot(j);
      if (to != nullptr) *reinterpret_cast<uint4*>(to) = y[i];
    }
  };
  // step c's rows go to [c * kStep, (c + 1) * kStep); later steps read at or above (c + 1) * kStep,
  // so only the rows of one step have to be read by all threads before any is written
  read(0, x[0]);
#pragma unroll 1
  for (int j0 = 0; j0 < n; j0 += 2 * kStep) {
    __syncthreads();
    read(j0 + kStep, x[1]);
    write(j0, x[0]);
    __syncthreads();
    read(j0 + 2 * kStep, x[0]);
    write(j0 + kStep, x[1]);
  }
}

}  // namespace oscar
