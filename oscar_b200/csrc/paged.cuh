// Attention over a paged 16-bit cache: the arguments, and the keys' accumulated
// attention weights.  The attention itself is in paged_attn.cuh.
//
//   S = scale Q K^T, row (token i of its request) sees keys [0, seq - q_len + i]
//   O = softmax(S) V,  LSE = log sum exp S
//   weights[slot, h] += sum over observed rows of the group of exp(S - LSE)
//
// Few query rows (decode, draft steps): the attention pass stores its scores
// (4 bytes per row and key against 2 D bytes of a key read again), and a thread
// per key sums them once the rows' maxima and sums are known.  Many rows: the
// scores are computed again, tile by tile of the keys.
#pragma once

#include "tc.cuh"

namespace oscar {

constexpr int kPgKeys = 64;       // keys per tile here and in the attention of few rows
constexpr int kPgReqs = 256;      // requests per launch (the plan travels by value)
constexpr int kPgFewRows = 32;    // query rows up to which scores are stored
constexpr int kPgWarps = 8;
constexpr float kPgHeadroom = 8.0f;

struct KeyPlan {  // the keys of a launch's requests in 64-key tiles
  int num_req;
  int req_id[kPgReqs];  // row of the block table
  int q_start[kPgReqs];
  int q_len[kPgReqs];
  int seq[kPgReqs];
  int tile_begin[kPgReqs + 1];
};

// Division by the page size without a divide (it sits in the producers' serial path, where
// one costs 150 cycles), by the method of Granlund and Montgomery (Division by Invariant
// Integers using Multiplication, 1994): q = (mulhi(mul, n) + n) >> shift for n < 2^31, with
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
  float* part_o;          // [piece][row][D] unnormalised
  float2* part_ml;        // [piece][row] (maximum, sum)
  float* scores;          // [tile][score_rows][64] scaled scores in log2 units, or null
  int score_rows;         // the most query rows of a request
  float* weights;         // [num_blocks, hk, bs], or null
  int observe;            // the last `observe` tokens of a request weigh the keys
  uint32_t tries;         // of a bounded wait
};

OSCAR_DEVINL int pg_find(const int* begin, int n, int x) {
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

// 16-byte chunk `c` of 128-byte row `r` under the 128-byte swizzle
OSCAR_DEVINL uint32_t pg_swz(int r, int c) { return (uint32_t)(r * 128 + ((c ^ (r & 7)) << 4)); }

// Bounded wait of a CTA whose roles never leave early: the first time-out sets
// the CTA's abort flag, after which every wait returns soon and the warps run
// to the end through their (always complete) barriers.  The limit is for one
// step of a pipeline (microseconds): no wait of this kind may span a launch,
// which may take any time.  A waiting warp suspends for up to a millisecond a
// try: polls take shared-memory cycles from the tensor cores' operands (2570
// against 2430 us on the longest chunk).
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
OSCAR_DEVINL bool pg_wait(int& abort, uint32_t bar, uint32_t parity, uint32_t tries) {
  if (tc::mbar_test(bar, parity)) return true;
  for (uint32_t i = 0; i < tries; ++i) {
    if (pg_try(bar, parity)) return true;
    if (*reinterpret_cast<volatile int*>(&abort) != 0) return false;
  }
  *reinterpret_cast<volatile int*>(&abort) = 1;
  flag_error(16u);
  return false;
}

// For what is in flight already and needs no warp to complete (copies, products), whether or not
// the CTA has been aborted: at most a quarter of a second.
constexpr uint32_t kPgDrainTries = 256;
OSCAR_DEVINL bool pg_drain(uint32_t bar, uint32_t parity) {
  for (uint32_t i = 0; i < kPgDrainTries; ++i)
    if (pg_try(bar, parity)) return true;
  flag_error(16u);
  return false;
}

// The keys' attention weights of requests with many query rows: scores are
// recomputed.  CTA = (request, 64-key tile) x kv head, K tile in shared memory;
// warp w takes the observed rows' 16-row blocks w, w + 8, ... that see the tile
// and sums p = exp2(s - m) / l over its rows in registers.  Bound by the latency
// of the query loads, so they are 16 bytes wide (384 rows on 11304 keys, 4 heads,
// D 256: about 50 us; 4-byte loads of the fragments in their own order 85 us).
template <int D, typename T>
__global__ void __launch_bounds__(32 * kPgWarps) paged_mass_rows_kernel(const __grid_constant__ PagedArgs a,
                                                                        const __grid_constant__ KeyPlan p,
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
  constexpr int kLoads = kPgKeys * (D / 8) / (32 * kPgWarps);
  uint4 kv[kLoads];
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const int key = (i * 32 * kPgWarps + tid) / (D / 8), c = tid % (D / 8);
    kv[i] = make_uint4(0, 0, 0, 0);
    if (key0 + key < seq) {
      const int64_t blk = row[a.page.div(key0 + key)];
      if (blk >= 0 && blk < a.num_blocks)
        kv[i] = *reinterpret_cast<const uint4*>(k_cache + blk * kcb + (int64_t)a.page.mod(key0 + key) * kct + h * kch + 8 * c);
    }
  }
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const int key = (i * 32 * kPgWarps + tid) / (D / 8), c = tid % (D / 8);
    *reinterpret_cast<uint4*>(pg_raw + key * (2 * D) + ((c ^ (key & 1) << 2) << 4)) = kv[i];
  }
  __syncthreads();
  const int qr = lane >> 2, qc = lane & 3;
  // rows that are observed and see at least the tile's first key
  const int tok_first = max(max(0, q_len - a.observe), key0 - (seq - q_len));
  const int row_first = tok_first * a.group, row_end = q_len * a.group;
  float sum[kPgKeys / 8][2];
#pragma unroll
  for (int n = 0; n < kPgKeys / 8; ++n) sum[n][0] = sum[n][1] = 0.0f;
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
    // A product's k order is free as long as both operands share it: lane qc holds dims 8 qc .. 8 qc + 7 of
    // each 32, one 16-byte load per row, as k 2 qc, 2 qc + 1, 2 qc + 8, 2 qc + 9 of two steps.
#pragma unroll 4
    for (int d0 = 0; d0 < D; d0 += 32) {
      const uint4 q0 = *reinterpret_cast<const uint4*>(src[0] + d0 + 8 * qc);
      const uint4 q1 = *reinterpret_cast<const uint4*>(src[1] + d0 + 8 * qc);
      const uint32_t qa[4] = {q0.x, q1.x, q0.y, q1.y}, qb[4] = {q0.z, q1.z, q0.w, q1.w};
#pragma unroll
      for (int n = 0; n < kPgKeys / 8; ++n) {
        const uint4 k = *reinterpret_cast<const uint4*>(pg_raw + (8 * n + qr) * (2 * D) + (((d0 / 8 + qc) ^ (qr & 1) << 2) << 4));
        Mma<T>::run(s[n], qa, k.x, k.y);
        Mma<T>::run(s[n], qb, k.z, k.w);
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
// reading the scores, 8 rows in flight per thread (8 x 24580 keys, 24 rows, 4
// heads: 76 MB in 19.5 us).
// (tiles of request r: [head][key tile], numbered as the attention's)
__global__ void __launch_bounds__(kPgKeys) paged_mass_kernel(const __grid_constant__ PagedArgs a,
                                                             const __grid_constant__ KeyPlan p) {
  __shared__ float2 st[kPgFewRows];
  pdl_release();
  const int r = pg_find(p.tile_begin, p.num_req, blockIdx.x);
  const int seq = p.seq[r], q_len = p.q_len[r];
  const int nt = max(1, (seq + kPgKeys - 1) / kPgKeys);
  const int local = blockIdx.x - p.tile_begin[r], h = local / nt;
  const int key = (local - h * nt) * kPgKeys + threadIdx.x, rows = q_len * a.group;
  const int page = key < seq ? (int)a.page.div(key) : 0;
  pdl_wait();
  const int64_t blk = key < seq ? a.table[(int64_t)p.req_id[r] * a.table_stride + page] : -1;
  const int first = max(0, q_len - a.observe) * a.group;  // first observed row
  for (int i = threadIdx.x; i < rows; i += kPgKeys) {
    const int tok = i / a.group;
    st[i] = a.stats[(int64_t)(p.q_start[r] + tok) * a.hq + h * a.group + i - tok * a.group];
  }
  __syncthreads();
  if (blk < 0 || blk >= a.num_blocks) return;  // past the request, or flagged by the attention pass
  float sum = 0.0f;
  const float* s = a.scores + (int64_t)blockIdx.x * a.score_rows * kPgKeys + threadIdx.x;
#pragma unroll 8
  for (int i = first; i < rows; ++i) sum = fmaf(pg_exp2(s[i * kPgKeys] - st[i].x), st[i].y, sum);
  float* w = a.weights + (blk * a.hk + h) * a.bs + (key - page * a.bs);
  if (key < seq - q_len)
    atomicAdd(w, sum);  // requests may share a page of history
  else
    *w = sum;
}

}  // namespace oscar
