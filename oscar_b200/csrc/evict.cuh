// Eviction from a 16-bit paged cache by accumulated attention weight.
//
// Per request and kv head, of the positions [0, seq): the first `sink`, the last
// `recent` and, of those between, the keep - sink - recent heaviest (ties to the
// lower position) stay, in order; their K, V and weight slots move to positions
// 0, 1, ... of the destination pages.  The destination may be the request's own
// pages: the j-th kept position is never below j, so moving in ascending order
// never overwrites a slot that is still to be read.
//
// evict_select_kernel (a CTA per request and head) finds the weight of the last
// key that stays by a radix descent over order-preserving 32-bit keys (three
// digits of 11, 11 and 10 bits, counted in shared memory), then walks the
// positions in order, 1024 at a time, numbers the kept ones with a block-wide
// prefix sum, writes their list and moves their weights.  Weights are held in
// shared memory while the request has at most kEvCached keys, else read again
// on each pass (they are then larger than the SM's share of L1 but in L2).
//
// evict_move_kernel moves the rows.  Bound by bytes.  To other pages every row
// is independent.  In place a CTA owns a 128-byte slice of one head's K or V
// rows and walks the list in ascending order: it holds 256 rows' slices in
// registers between the read and the write of a step, and the next step's
// reads are already in flight.
#pragma once

#include "common.cuh"

namespace oscar {

constexpr int kEvReqs = 256;
constexpr int kEvThreads = 1024;
constexpr int kEvCached = 49152;
constexpr int kEvBins = 2048;
constexpr int kEvMoveThreads = 256;
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

OSCAR_DEVINL float* ev_weight(const EvictArgs& a, const int32_t* row, int h, int pos) {
  const int64_t blk = row[pos / a.bs];
  if (blk < 0 || blk >= a.num_blocks) {
    flag_error(2u);
    return nullptr;
  }
  return a.weights + (blk * a.hk + h) * a.bs + pos % a.bs;
}

__global__ void __launch_bounds__(kEvThreads) evict_select_kernel(const __grid_constant__ EvictArgs a,
                                                                  const __grid_constant__ EvictPlan p) {
  extern __shared__ __align__(16) float ev_w[];
  __shared__ uint32_t bins[kEvBins];
  __shared__ uint32_t warp_sum[32];
  __shared__ uint32_t pick[2];
  pdl_release();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int r = blockIdx.x, h = blockIdx.y;
  const int seq = p.seq[r];
  const int32_t* src_row = a.table + (int64_t)p.req_id[r] * a.table_stride;
  const int32_t* dst_row = a.dst + (int64_t)p.req_id[r] * a.dst_stride;
  int32_t* kept = a.kept + ((int64_t)p.req_id[r] * a.hk + h) * a.kept_stride;
  const int n = min(seq, a.keep);
  const bool all = seq <= a.keep;
  const bool cached = seq <= kEvCached;
  pdl_wait();
  for (int j = n + tid; j < a.kept_stride; j += kEvThreads) kept[j] = -1;
  auto global_weight = [&](int pos) -> float {
    const float* w = ev_weight(a, src_row, h, pos);
    return w == nullptr ? 0.0f : *w;
  };
  if (cached) {
#pragma unroll 4
    for (int i = tid; i < seq; i += kEvThreads) ev_w[i] = global_weight(i);
    __syncthreads();
  }
  auto weight = [&](int pos) -> float { return cached ? ev_w[pos] : global_weight(pos); };

  // the key value at which the list is full, and how many of the keys that equal it stay
  const int lo = a.sink, hi = seq - a.recent;
  uint32_t threshold = 0, need = (uint32_t)max(0, a.keep - a.sink - a.recent);
  if (!all && need > 0) {
#pragma unroll 1
    for (int digit = 0; digit < 3; ++digit) {
      const int shift = digit == 0 ? 21 : digit == 1 ? 10 : 0;
      const int width = digit == 2 ? 10 : 11;
      const uint32_t above = digit == 0 ? 0u : 0xffffffffu << (shift + width);
      for (int i = tid; i < kEvBins; i += kEvThreads) bins[i] = 0;
      __syncthreads();
      for (int i0 = lo; i0 < hi; i0 += kEvThreads) {
        const int i = i0 + tid;
        const uint32_t key = i < hi ? ev_key(weight(i)) : 0u;
        const bool in = i < hi && (key & above) == (threshold & above);
        const uint32_t bin = (key >> shift) & ((1u << width) - 1);
        // weights share few exponents: one add per distinct bin of the warp
        const uint32_t who = __match_any_sync(0xffffffffu, in ? bin : 0xffffffffu);
        if (in && (int)(__ffs(who) - 1) == lane) atomicAdd(&bins[bin], (uint32_t)__popc(who));
      }
      __syncthreads();
      // count from the top: thread t holds bins 2 t' and 2 t' + 1 in descending order
      const int b1 = kEvBins - 1 - 2 * tid, b0 = b1 - 1;
      const uint32_t c1 = bins[b1], c0 = bins[b0];
      uint32_t sum = c1 + c0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t x = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += x;
      }
      if (lane == 31) warp_sum[warp] = sum;
      __syncthreads();
      uint32_t before = sum - (c1 + c0);
      for (int w = 0; w < warp; ++w) before += warp_sum[w];
      if (before < need && before + c1 >= need) pick[0] = b1, pick[1] = need - before;
      else if (before + c1 < need && before + c1 + c0 >= need) pick[0] = b0, pick[1] = need - before - c1;
      __syncthreads();
      threshold |= pick[0] << shift;
      need = pick[1];
      __syncthreads();
    }
  }

  // ordered walk
  uint32_t equal_seen = 0, out = 0;
  for (int i0 = 0; i0 < seq; i0 += kEvThreads) {
    const int i = i0 + tid;
    const float w = i < seq ? weight(i) : 0.0f;
    const bool fixed = i < seq && (all || i < lo || i >= hi);
    const bool middle = i < seq && !fixed && a.keep > a.sink + a.recent;
    const uint32_t key = ev_key(w);
    const bool above = middle && key > threshold, equal = middle && key == threshold;
    // prefix of equal keys, then of kept keys: both counts in one 32-bit word (16 bits each)
    auto prefix = [&](uint32_t mine, uint32_t& total) -> uint32_t {
      uint32_t sum = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t x = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += x;
      }
      if (lane == 31) warp_sum[warp] = sum;
      __syncthreads();
      const uint32_t v = warp_sum[lane];
      uint32_t scan = v;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t x = __shfl_up_sync(0xffffffffu, scan, o);
        if (lane >= o) scan += x;
      }
      total = __shfl_sync(0xffffffffu, scan, 31);
      const uint32_t base = warp == 0 ? 0u : __shfl_sync(0xffffffffu, scan, (warp + 31) & 31);
      __syncthreads();
      return base + sum - mine;
    };
    // low half: keys above or fixed; high half: equal ones (at most 1024 of each)
    uint32_t total;
    const uint32_t at = prefix((fixed || above ? 1u : 0u) | (equal ? 0x10000u : 0u), total);
    const uint32_t eq_before = equal_seen + (at >> 16);
    const bool stays = fixed || above || (equal && eq_before < need);
    // kept keys before this one: all fixed / above ones and the equal ones that stay
    const uint32_t j = out + (at & 0xffffu) + (min(eq_before, need) - min(equal_seen, need));
    if (stays && (int)j < n) {
      kept[j] = i;
      float* dst = ev_weight(a, dst_row, h, (int)j);
      if (dst != nullptr) *dst = w;
    }
    const uint32_t eq_after = equal_seen + (total >> 16);
    out += (total & 0xffffu) + (min(eq_after, need) - min(equal_seen, need));
    equal_seen = eq_after;
  }
}

// To other pages: a warp per kept row and K or V, 16 bytes per lane and step.
__global__ void __launch_bounds__(kEvMoveThreads) evict_copy_kernel(const __grid_constant__ EvictArgs a,
                                                                    const __grid_constant__ EvictPlan p) {
  pdl_release();
  const int lanes = a.row_bytes / 16;  // 8, 16 or 32 lanes per row
  const int r = blockIdx.y / a.hk, h = blockIdx.y % a.hk;
  const int n = min(p.seq[r], a.keep);
  const int32_t* src_row = a.table + (int64_t)p.req_id[r] * a.table_stride;
  const int32_t* dst_row = a.dst + (int64_t)p.req_id[r] * a.dst_stride;
  const int32_t* kept = a.kept + ((int64_t)p.req_id[r] * a.hk + h) * a.kept_stride;
  const int c = threadIdx.x % lanes, rows = kEvMoveThreads / lanes;
  pdl_wait();
#pragma unroll 1
  for (int j0 = blockIdx.x * rows * 4; j0 < n; j0 += gridDim.x * rows * 4) {
    uint4 kv[4], vv[4];
    int64_t to_blk[4];
    int to_off[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int j = j0 + i * rows + threadIdx.x / lanes;
      to_blk[i] = -1;
      if (j >= n) continue;
      const int s = kept[j];
      const int64_t sb = src_row[s / a.bs], db = dst_row[j / a.bs];
      if (sb < 0 || sb >= a.num_blocks || db < 0 || db >= a.num_blocks) continue;  // flagged by the selection
      const int so = s % a.bs;
      kv[i] = *reinterpret_cast<const uint4*>(a.k + sb * a.kb + so * a.kt + h * a.kh + 16 * c);
      vv[i] = *reinterpret_cast<const uint4*>(a.v + sb * a.vb + so * a.vt + h * a.vh + 16 * c);
      to_blk[i] = db;
      to_off[i] = j % a.bs;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (to_blk[i] < 0) continue;
      *reinterpret_cast<uint4*>(a.k + to_blk[i] * a.kb + to_off[i] * a.kt + h * a.kh + 16 * c) = kv[i];
      *reinterpret_cast<uint4*>(a.v + to_blk[i] * a.vb + to_off[i] * a.vt + h * a.vh + 16 * c) = vv[i];
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
    const int64_t blk = row[pos / a.bs];
    return blk < 0 || blk >= a.num_blocks ? nullptr : base + blk * sb + (int64_t)(pos % a.bs) * stt;
  };
  uint4 x[2][kEvWaves];
  auto read = [&](int j0, uint4 (&y)[kEvWaves]) {
#pragma unroll
    for (int i = 0; i < kEvWaves; ++i) {
      const int j = j0 + i * kRows + threadIdx.x / 8;
      if (j >= n) continue;
      const int s = kept[j];
      const uint8_t* from = s == j ? nullptr : slot(s);
      if (from != nullptr) y[i] = *reinterpret_cast<const uint4*>(from);
    }
  };
  auto write = [&](int j0, const uint4 (&y)[kEvWaves]) {
#pragma unroll
    for (int i = 0; i < kEvWaves; ++i) {
      const int j = j0 + i * kRows + threadIdx.x / 8;
      if (j >= n) continue;
      const int s = kept[j];
      if (s == j || slot(s) == nullptr) continue;
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
