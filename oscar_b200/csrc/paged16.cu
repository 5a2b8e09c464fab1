// C ABI of the 16-bit paged attention layer (declarations and contracts:
// include/oscar_b200.h): head norm + rotation + cache write, attention over
// the paged cache with the keys' accumulated weights, eviction by weight.
#include <algorithm>
#include <atomic>
#include <climits>
#include <cmath>

#include "../../include/oscar_b200.h"
#include "evict.cuh"
#include "head_norm.cuh"
#include "host.h"
#include "paged.cuh"
#include "paged_attn.cuh"
#include "paged_mma.cuh"

namespace oscar_host {

int take_paged16_error() {
  unsigned int v = 0, zero = 0;
  if (cudaMemcpyFromSymbol(&v, oscar::g_bounds_error, sizeof(v)) != cudaSuccess) return -OSCAR_ERR_CUDA;
  cudaMemcpyToSymbol(oscar::g_bounds_error, &zero, sizeof(zero));
  return (int)v;
}

}  // namespace oscar_host

namespace {

using oscar_host::cuda_status;
using oscar_host::device_info;
using oscar_host::encode_tiled;
using oscar_host::fail;
using oscar_host::launch_pdl;
using oscar_host::launch_pdl_cluster;

// Positions and tiles are counted in 32 bits, with room for what is added to them: a request's
// cached tokens, its 64-key tiles over all heads and those of a launch, and the tiles of a call's
// query blocks (over 74 pairs of CTAs or more).
constexpr int32_t kMaxLength = 1 << 30;
constexpr int64_t kMaxKeyTiles = (int64_t)1 << 30, kMaxWork = (int64_t)1 << 38;

std::atomic<uint32_t> g_wait_tries{oscar::kPgTries};

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

bool half_dtype(int32_t dtype) { return dtype == OSCAR_DTYPE_BF16 || dtype == OSCAR_DTYPE_F16; }

bool kernel_head_dim(int32_t d) { return d == 64 || d == 128 || d == 256; }

// Are the rows of [n, heads, d] at these strides apart from one another?
bool rows_apart(int64_t n, int64_t heads, int64_t d, int64_t token_stride, int64_t head_stride) {
  if (n < 2) return heads < 2 || head_stride >= d;
  if (heads < 2) return token_stride >= d;
  const bool nested = token_stride >= head_stride;  // heads within a token's stride, or tokens within a head's
  return nested ? head_stride >= d && token_stride >= (heads - 1) * head_stride + d
                : token_stride >= d && head_stride >= (n - 1) * token_stride + d;
}

// One cache of [num_blocks, block_size, hk, D] elements with strides in elements.
int check_cache(const char* what, const void* cache, int64_t num_blocks, int32_t bs, int32_t hk, int32_t d, int64_t sb,
                int64_t st, int64_t sh) {
  if (num_blocks < 0 || num_blocks >= INT_MAX || bs < 1 || hk < 1)
    return fail(OSCAR_ERR_INVALID, "%s: invalid cache geometry", what);
  if (num_blocks > 0 && !cache) return fail(OSCAR_ERR_INVALID, "%s: null cache", what);
  // (a dimension of one element has no stride of its own)
  if (!aligned16(cache) || ((num_blocks > 1 ? sb : 0) | (bs > 1 ? st : 0) | (hk > 1 ? sh : 0)) % 8)
    return fail(OSCAR_ERR_INVALID, "%s: cache rows must be 16-byte aligned", what);
  if ((hk > 1 && sh < d) || (bs > 1 && st < d) || (num_blocks > 1 && sb < d))
    return fail(OSCAR_ERR_INVALID, "%s: cache rows overlap", what);
  return OSCAR_OK;
}

}  // namespace

// ---------------------------------------------------------------------------
namespace {

template <typename T>
void launch_head_norm(const oscar::HeadNormArgs& a, int d, cudaStream_t s) {
  const int heads = a.hq + a.hk + (a.v_cache != nullptr ? a.hk : 0);
  const int groups = (heads + oscar::kHnHeads - 1) / oscar::kHnHeads;
  constexpr int kWarps = oscar::kHnThreads / 32;
  const int64_t tokens = (a.n + 256 / d - 1) / (256 / d);  // warps that hold whole tokens
  // enough warps to fill the SMs (16 each), at most one per group of heads
  const int64_t want = (int64_t)std::max(device_info().sms, 1) * 16;
  const int splits = (int)std::min<int64_t>(groups, std::max<int64_t>(1, (want + tokens - 1) / tokens));
  const dim3 grid((unsigned)((tokens * splits + kWarps - 1) / kWarps)), block(oscar::kHnThreads);
  if (d == 256) launch_pdl(oscar::head_norm_kernel<T, 256>, grid, block, 0, s, a, splits);
  else if (d == 128) launch_pdl(oscar::head_norm_kernel<T, 128>, grid, block, 0, s, a, splits);
  else launch_pdl(oscar::head_norm_kernel<T, 64>, grid, block, 0, s, a, splits);
}

}  // namespace

extern "C" int oscar_qk_norm_rope(const void* q, int64_t q_token_stride, int64_t q_head_stride, const void* k,
                                  int64_t k_token_stride, int64_t k_head_stride, const void* v, int64_t v_token_stride,
                                  int64_t v_head_stride, int32_t dtype, int64_t n_tokens, int32_t num_q_heads,
                                  int32_t num_kv_heads, int32_t head_dim, const void* q_weight, const void* k_weight,
                                  int32_t weight_dtype, float eps, float weight_offset, const void* cos_sin,
                                  int32_t cos_sin_dtype, int64_t cos_sin_stride, int64_t max_positions,
                                  int32_t rot_dim, int32_t interleaved, const int64_t* positions, void* out_q,
                                  int64_t out_q_token_stride, int64_t out_q_head_stride, void* out_k,
                                  int64_t out_k_token_stride, int64_t out_k_head_stride, void* k_cache, void* v_cache,
                                  int64_t num_blocks, int32_t block_size, int64_t k_stride_block,
                                  int64_t k_stride_token, int64_t k_stride_head, int64_t v_stride_block,
                                  int64_t v_stride_token, int64_t v_stride_head, const int64_t* slot_mapping,
                                  void* stream) {
  if (!half_dtype(dtype)) return fail(OSCAR_ERR_UNSUPPORTED, "qk_norm_rope: heads must be bf16 or fp16");
  if (!kernel_head_dim(head_dim))
    return fail(OSCAR_ERR_UNSUPPORTED, "qk_norm_rope: head_dim %d: kernels exist for 64, 128, 256", head_dim);
  if (n_tokens < 0 || num_q_heads < 1 || num_kv_heads < 1 || num_q_heads > 4096 || num_kv_heads > 4096 ||
      max_positions < 1)
    return fail(OSCAR_ERR_INVALID, "qk_norm_rope: invalid geometry");
  if (rot_dim < 16 || rot_dim > head_dim || rot_dim % 16)
    return fail(OSCAR_ERR_INVALID, "qk_norm_rope: rot_dim %d must be a multiple of 16 of at most head_dim", rot_dim);
  if ((weight_dtype != OSCAR_DTYPE_F32 && weight_dtype != dtype) ||
      (cos_sin_dtype != OSCAR_DTYPE_F32 && cos_sin_dtype != dtype))
    return fail(OSCAR_ERR_UNSUPPORTED, "qk_norm_rope: weights and cos / sin must be fp32 or of the heads' type");
  if (!(eps >= 0.0f) || !std::isfinite(eps) || !std::isfinite(weight_offset))
    return fail(OSCAR_ERR_INVALID, "qk_norm_rope: eps must be finite and not negative");
  if ((k_cache == nullptr) != (v_cache == nullptr) || (k_cache == nullptr) != (slot_mapping == nullptr))
    return fail(OSCAR_ERR_INVALID, "qk_norm_rope: caches and slot_mapping come together");
  if (k_cache != nullptr) {
    int st = check_cache("qk_norm_rope", k_cache, num_blocks, block_size, num_kv_heads, head_dim, k_stride_block,
                         k_stride_token, k_stride_head);
    if (!st)
      st = check_cache("qk_norm_rope", v_cache, num_blocks, block_size, num_kv_heads, head_dim, v_stride_block,
                       v_stride_token, v_stride_head);
    if (st) return st;
  }
  if (n_tokens == 0) return OSCAR_OK;
  if (k_cache == nullptr && out_k == nullptr) return fail(OSCAR_ERR_INVALID, "qk_norm_rope: the keys have no destination");
  if (!q || !k || !q_weight || !k_weight || !cos_sin || !positions || !out_q || (k_cache != nullptr && !v))
    return fail(OSCAR_ERR_INVALID, "qk_norm_rope: null pointer");
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(out_q) || !aligned16(out_k) ||
      !aligned16(q_weight) || !aligned16(k_weight) || !aligned16(cos_sin) ||
      (q_token_stride | q_head_stride | k_token_stride | k_head_stride | out_q_token_stride | out_q_head_stride) % 8 ||
      (v != nullptr && (v_token_stride | v_head_stride) % 8) ||
      (out_k != nullptr && (out_k_token_stride | out_k_head_stride) % 8) || cos_sin_stride % 8 || cos_sin_stride < rot_dim)
    return fail(OSCAR_ERR_INVALID, "qk_norm_rope: heads, weights and cos / sin rows must be 16-byte aligned");
  if (!rows_apart(n_tokens, num_q_heads, head_dim, out_q_token_stride, out_q_head_stride) ||
      (out_k != nullptr && !rows_apart(n_tokens, num_kv_heads, head_dim, out_k_token_stride, out_k_head_stride)))
    return fail(OSCAR_ERR_INVALID, "qk_norm_rope: output rows overlap");
  oscar::HeadNormArgs a{};
  a.q = q, a.k = k, a.v = v;
  a.q_tok = q_token_stride, a.q_head = q_head_stride;
  a.k_tok = k_token_stride, a.k_head = k_head_stride;
  a.v_tok = v_token_stride, a.v_head = v_head_stride;
  a.out_q = out_q, a.out_k = out_k;
  a.oq_tok = out_q_token_stride, a.oq_head = out_q_head_stride;
  a.ok_tok = out_k_token_stride, a.ok_head = out_k_head_stride;
  a.wq = q_weight, a.wk = k_weight;
  a.w_f32 = weight_dtype == OSCAR_DTYPE_F32;
  a.eps = eps, a.offset = weight_offset;
  a.cos_sin = cos_sin;
  a.cs_f32 = cos_sin_dtype == OSCAR_DTYPE_F32;
  a.cs_stride = cos_sin_stride, a.max_pos = max_positions;
  a.rot = rot_dim, a.interleaved = interleaved != 0;
  a.positions = positions;
  a.n = n_tokens, a.hq = num_q_heads, a.hk = num_kv_heads;
  a.k_cache = k_cache, a.v_cache = v_cache;
  a.num_blocks = num_blocks, a.bs = block_size;
  a.kcb = k_stride_block, a.kct = k_stride_token, a.kch = k_stride_head;
  a.vcb = v_stride_block, a.vct = v_stride_token, a.vch = v_stride_head;
  a.slots = slot_mapping;
  const int heads = a.hq + 2 * a.hk;
  if (n_tokens > (int64_t)INT_MAX / heads) return fail(OSCAR_ERR_UNSUPPORTED, "qk_norm_rope: too many tokens for one launch");
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == OSCAR_DTYPE_BF16) launch_head_norm<__nv_bfloat16>(a, head_dim, s);
  else launch_head_norm<__half>(a, head_dim, s);
  return cuda_status("head_norm_kernel");
}

// ---------------------------------------------------------------------------
namespace {

// How a request's new tokens are attended.  kFew: at most 32 query rows per kv
// head, one row tile, scores stored where the keys are weighed.  kOne: one row
// tile.  kChunk: q-blocks of two row tiles.
enum PagedClass { kFew = 0, kOne = 1, kChunk = 2, kClasses = 3 };

// Scores that a launch stores at most: its requests are as many as that takes, and one that alone
// passes it has its scores computed again instead (kOne).  8 requests of 4 x 6 rows on 24580 keys
// and 4 heads have 76 MB.
constexpr int64_t kScoreBytes = (int64_t)256 << 20;

inline int64_t key_tiles(int32_t seq, int hk) {
  return std::max<int64_t>(1, ((int64_t)seq + oscar::kPgKeys - 1) / oscar::kPgKeys) * hk;
}
inline int64_t score_bytes(int64_t tiles, int64_t rows) { return tiles * rows * oscar::kPgKeys * (int64_t)sizeof(float); }

inline PagedClass paged_class(int64_t len, int32_t seq, int group, int hk, bool weighted) {
  if (len * group <= oscar::kPgFewRows && !(weighted && score_bytes(key_tiles(seq, hk), len * group) > kScoreBytes)) return kFew;
  return len <= oscar::kPcRows / group ? kOne : kChunk;
}

// kFew runs on mma.sync up to this many 64-key tiles per SM (paged_mma.cuh has both sides)
constexpr int64_t kMmaTiles = 32;

// Workspace of one launch, in this order.
struct PagedSpace {
  int64_t stats, part_ml, part_o, scores;  // bytes
  int64_t total() const { return stats + part_ml + part_o + scores; }
};
inline int64_t round256(int64_t x) { return (x + 255) & ~(int64_t)255; }

// The requests [r0, ..) of a call that fit one launch: at most kPgReqs of one
// class.  Returns the index after the last one looked at.
struct PagedBatch {
  PagedClass cls;
  int64_t tiles;
  int pieces;              // most pieces of a divided unit
  int rows;                // most query rows per kv head of a request
  oscar::PcPlan plan;
  oscar::PcSplits splits;  // its divided units
};

// Divides the tiles of all units over the workers.  A unit costs its tiles and
// kUnitCost more (queries, first products, epilogue: about 9000 cycles against
// 4100 a tile at D 128 and 7000 against 2600 at D 256, from clock traces), so that
// short units are not piled on one worker.
template <typename Shape>
void plan_units(PagedBatch& b, int hk, int sms) {
  constexpr int kUnitCost = 2;
  oscar::PcPlan& p = b.plan;
  const int64_t per = (int64_t)p.tokens * Shape::kUnit;
  int64_t total = 0;
  for (int i = 0; i < p.num_req; ++i)
    for (int qb = 0; qb * per < p.q_len[i]; ++qb)
      total += (int64_t)hk * (kUnitCost + oscar::pc_tiles<Shape>(p.q_len[i], p.seq[i], p.tokens, qb));
  const int workers = std::min(std::max(Shape::kPair ? sms / 2 : sms, 1), oscar::kPcCtas);
  p.ctas = 0;
  b.splits.n = 0;
  b.tiles = 0;
  b.pieces = 1;
  int64_t cost = 0;  // of the units before
  int next = 0;      // the next worker to begin, at cost total * next / workers
  auto begin_of = [&](int w) { return total * w / workers; };
  for (int i = 0; i < p.num_req; ++i)
    for (int h = 0; h < hk; ++h)
      for (int qb = 0; qb * per < p.q_len[i]; ++qb) {
        const int nt = oscar::pc_tiles<Shape>(p.q_len[i], p.seq[i], p.tokens, qb);
        const int holder = p.ctas - 1;  // the worker that reaches the unit, if none begins with it
        int done = 0;                   // tiles of the unit before the current worker
        bool begun = false;             // does a worker begin with the unit's first tile?
        while (next < workers && begin_of(next) < cost + kUnitCost + nt) {
          // a share that begins in a unit's fixed cost begins with its first tile; two that begin
          // at the same tile are one
          const int t = (int)std::max<int64_t>(0, begin_of(next) - cost - kUnitCost);
          ++next;
          if (t < done || (t == done && (begun || done > 0))) continue;
          if (p.ctas > 0) p.tiles[p.ctas - 1] += t - done;
          begun = begun || t == 0;
          done = t;
          p.start[p.ctas] = oscar::PcStart{i, h, qb, t};
          p.first[p.ctas] = (int)(b.tiles + t);
          p.tiles[p.ctas++] = 0;
        }
        p.tiles[p.ctas - 1] += nt - done;
        const int first = begun ? holder + 1 : holder;
        if (p.ctas - 1 > first) b.splits.unit[b.splits.n++] = oscar::PcSplit{i, h, qb, first, p.ctas - 1};
        b.pieces = std::max(b.pieces, p.ctas - first);
        cost += kUnitCost + nt;
        b.tiles += nt;
      }
}

int paged_batch(PagedBatch& b, PagedClass cls, int r0, const int32_t* qsl, const int32_t* seqs, int num, int group,
                int hk, int d, bool weighted, int sms) {
  oscar::PcPlan& p = b.plan;
  b.cls = cls;
  b.rows = 0;
  p.num_req = 0;
  int r = r0;
  int64_t tiles = 0;
  for (; r < num && p.num_req < oscar::kPgReqs; ++r) {
    const int len = qsl[r + 1] - qsl[r];
    if (len == 0 || paged_class(len, seqs[r], group, hk, weighted) != cls) continue;
    tiles += key_tiles(seqs[r], hk);
    const int rows = std::max(b.rows, (int)std::min<int64_t>((int64_t)len * group, INT_MAX));
    if (p.num_req > 0 && (tiles > kMaxKeyTiles || (weighted && cls == kFew && score_bytes(tiles, rows) > kScoreBytes))) break;
    b.rows = rows;
    const int i = p.num_req++;
    p.req_id[i] = r;
    p.q_start[i] = qsl[r];
    p.q_len[i] = len;
    p.seq[i] = seqs[r];
  }
  if (p.num_req == 0) return r;
  p.tokens = p.box_tokens = oscar::kPcRows / group;
  if (cls != kChunk) {
    p.box_tokens = 1;
    for (int i = 0; i < p.num_req; ++i) p.box_tokens = std::max(p.box_tokens, p.q_len[i]);
  }
  if (cls != kChunk) plan_units<oscar::PcShape<256, true>>(b, hk, sms);  // (the plan does not depend on D)
  else if (d == 256) plan_units<oscar::PcShape<256, false>>(b, hk, sms);
  else plan_units<oscar::PcShape<128, false>>(b, hk, sms);  // (64 as 128)
  return r;
}

PagedSpace paged_space(const PagedBatch& b, int64_t n, int hq, int d, bool weighted) {
  PagedSpace s{};
  if (weighted) s.stats = round256(n * hq * (int64_t)sizeof(float2));
  const int64_t pieces = (int64_t)2 * b.plan.ctas * oscar::kPcRows * (b.cls == kChunk ? 2 : 1);
  s.part_ml = round256(pieces * (int64_t)sizeof(float2));
  s.part_o = round256(pieces * d * (int64_t)sizeof(float));
  if (weighted && b.cls == kFew) s.scores = score_bytes(b.tiles, b.rows);
  return s;
}

int check_paged(const int32_t* qsl, const int32_t* seqs, int32_t num_requests, int64_t n_tokens, int32_t hq, int32_t hk) {
  if (hq < 1 || hk < 1 || hq % hk || hq > 4096) return fail(OSCAR_ERR_INVALID, "paged_attention: Hq must be a multiple of Hk");
  if (hq / hk > oscar::kPcRows) return fail(OSCAR_ERR_UNSUPPORTED, "paged_attention: GQA group %d > %d", hq / hk, oscar::kPcRows);
  if (num_requests < 0 || !qsl || (num_requests > 0 && !seqs) || qsl[0] != 0 || qsl[num_requests] != n_tokens)
    return fail(OSCAR_ERR_INVALID, "paged_attention: invalid query layout");
  int64_t work = 0;
  for (int r = 0; r < num_requests; ++r) {
    if (qsl[r] > qsl[r + 1] || seqs[r] < 0)
      return fail(OSCAR_ERR_INVALID, "paged_attention: query starts must not fall and lengths not be negative");
    if (qsl[r] == qsl[r + 1]) continue;
    const int64_t tiles = key_tiles(seqs[r], hk), tokens = oscar::kPcRows / (hq / hk);
    work += tiles * ((qsl[r + 1] - qsl[r] + tokens - 1) / tokens);
    if (seqs[r] > kMaxLength || tiles > kMaxKeyTiles || work > kMaxWork)
      return fail(OSCAR_ERR_UNSUPPORTED, "paged_attention: lengths of request %d too long for one call", r);
  }
  return OSCAR_OK;
}

oscar::FastDiv fast_div(uint32_t d) {
  uint32_t shift = 0;
  while (((uint64_t)1 << shift) < d) ++shift;
  return oscar::FastDiv{d, (uint32_t)((((uint64_t)1 << 32) * (((uint64_t)1 << shift) - d)) / d + 1), shift};
}

// The cache as a 4D map (dims, heads, tokens of a page, pages) in boxes of 64 dims x `box` tokens.
bool paged_map(CUtensorMap* map, const void* base, int dtype, int64_t num_blocks, int bs, int hk, int d, int64_t sb,
               int64_t st, int64_t sh, int box) {
  const auto fn = encode_tiled();
  if (!fn) return false;
  const cuuint64_t dims[4] = {(cuuint64_t)d, (cuuint64_t)hk, (cuuint64_t)bs, (cuuint64_t)num_blocks};
  // a dimension of one element has no stride of its own
  const cuuint64_t strides[3] = {(cuuint64_t)(hk > 1 ? sh : d) * 2, (cuuint64_t)(bs > 1 ? st : d) * 2,
                                 (cuuint64_t)(num_blocks > 1 ? sb : d) * 2};
  const cuuint32_t boxes[4] = {64, 1, (cuuint32_t)box, 1};
  const cuuint32_t step[4] = {1, 1, 1, 1};
  return fn(map, dtype == OSCAR_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
            const_cast<void*>(base), dims, strides, boxes, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) ==
         CUDA_SUCCESS;
}

// The queries as a 3D map (dims, heads, tokens) in boxes of 64 dims x a kv head's group x `tokens`:
// the rows (token, head in group) of a q-block's row tile.
bool query_map(CUtensorMap* map, const void* q, int dtype, int64_t n, int hq, int d, int64_t tok, int64_t head, int group,
               int tokens) {
  const auto fn = encode_tiled();
  if (!fn) return false;
  const cuuint64_t dims[3] = {(cuuint64_t)d, (cuuint64_t)hq, (cuuint64_t)n};
  const cuuint64_t strides[2] = {(cuuint64_t)(hq > 1 ? head : d) * 2, (cuuint64_t)(n > 1 ? tok : d) * 2};
  const cuuint32_t boxes[3] = {64, (cuuint32_t)group, (cuuint32_t)tokens};
  const cuuint32_t step[3] = {1, 1, 1};
  return fn(map, dtype == OSCAR_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
            const_cast<void*>(q), dims, strides, boxes, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// dynamic shared memory above 48 KB has to be asked for once per kernel and device
template <auto Kernel>
void allow_smem(size_t bytes) {
  static thread_local int set_dev = -1;
  int dev = 0;
  cudaGetDevice(&dev);
  if (set_dev == dev) return;
  cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  set_dev = dev;
}

struct PagedCall {
  oscar::PagedArgs args;
  CUtensorMap qmap, kmap, vmap;
  const void* k_cache;
  int64_t kcb, kct, kch;
  cudaStream_t stream;
};

// The keys' weights of a launch's requests, from the scores or computed again
template <int D, typename T>
int launch_mass(const PagedCall& c, const PagedBatch& b) {
  oscar::KeyPlan keys;
  keys.num_req = b.plan.num_req;
  int64_t tiles = 0;
  for (int i = 0; i < b.plan.num_req; ++i) {
    keys.req_id[i] = b.plan.req_id[i];
    keys.q_start[i] = b.plan.q_start[i];
    keys.q_len[i] = b.plan.q_len[i];
    keys.seq[i] = b.plan.seq[i];
    keys.tile_begin[i] = (int)tiles;
    const int64_t nt = ((int64_t)b.plan.seq[i] + oscar::kPgKeys - 1) / oscar::kPgKeys;
    tiles += b.cls == kFew ? std::max<int64_t>(1, nt) * c.args.hk : nt;
  }
  keys.tile_begin[keys.num_req] = (int)tiles;
  if (tiles == 0) return OSCAR_OK;
  if (b.cls == kFew) {
    launch_pdl(oscar::paged_mass_kernel, dim3((unsigned)tiles), dim3(oscar::kPgKeys), 0, c.stream, c.args, keys);
    return cuda_status("paged_mass_kernel");
  }
  launch_pdl(oscar::paged_mass_rows_kernel<D, T>, dim3((unsigned)tiles, (unsigned)c.args.hk), dim3(32 * oscar::kPgWarps),
             (size_t)oscar::kPgKeys * D * 2, c.stream, c.args, keys, reinterpret_cast<const T*>(c.k_cache), c.kcb, c.kct,
             c.kch);
  return cuda_status("paged_mass_rows_kernel");
}

template <int D, typename T, int NRT>
int launch_mma(const PagedCall& c, const PagedBatch& b) {
  constexpr size_t smem = sizeof(oscar::PsSmem<D, NRT>);
  static_assert(smem <= 227 * 1024, "PsSmem exceeds the shared memory of a CTA");
  allow_smem<oscar::paged_attn_mma_kernel<D, T, NRT>>(smem);
  launch_pdl(oscar::paged_attn_mma_kernel<D, T, NRT>, dim3(b.plan.ctas), dim3(oscar::kPgThreads), smem, c.stream, c.args,
             b.plan, c.kmap, c.vmap);
  return cuda_status("paged_attn_mma_kernel");
}

template <int D, typename T, bool kFewRows>
int launch_tc(const PagedCall& c, const PagedBatch& b) {
  using Shape = oscar::PcShape<D, kFewRows>;
  constexpr size_t smem = sizeof(oscar::PcSmem<D, kFewRows>);
  static_assert(smem <= 227 * 1024, "PcSmem exceeds the shared memory of a CTA");
  allow_smem<oscar::paged_attn_tc_kernel<D, T, kFewRows>>(smem);
  launch_pdl_cluster(Shape::kPair ? 2 : 1, oscar::paged_attn_tc_kernel<D, T, kFewRows>,
                     dim3(Shape::kPair ? 2 * b.plan.ctas : b.plan.ctas), dim3(Shape::kThreads), smem, c.stream, c.args,
                     b.plan, c.qmap, c.kmap, c.vmap);
  return cuda_status("paged_attn_tc_kernel");
}

template <int D, typename T, bool kFewRows>
int launch_paged(const PagedCall& c, const PagedBatch& b) {
  using Shape = oscar::PcShape<D, kFewRows>;
  const oscar::PagedArgs& a = c.args;
  const oscar::PcPlan& p = b.plan;
  int st;
  if (b.cls == kFew && b.tiles <= kMmaTiles * device_info().sms)
    st = b.rows <= 16 ? launch_mma<D, T, 1>(c, b) : launch_mma<D, T, 2>(c, b);
  else
    st = launch_tc<D, T, kFewRows>(c, b);
  if (st) return st;
  if (b.splits.n > 0) {
    int rows = Shape::kUnit * oscar::kPcRows;  // of a unit
    if (kFewRows) rows = b.rows;
    // four warps a row from nine pieces on: with one, a row's pieces come one after another (28
    // against 10 us for one request's 24 rows in 37 pieces); below, they would mostly idle
    if (b.pieces > 8)
      launch_pdl(oscar::paged_merge_kernel<D, T, kFewRows, oscar::kPcMerge>, dim3((unsigned)rows, (unsigned)b.splits.n),
                 dim3(128), 0, c.stream, a, p, b.splits);
    else
      launch_pdl(oscar::paged_merge_kernel<D, T, kFewRows, 1>, dim3((unsigned)(rows + 3) / 4, (unsigned)b.splits.n), dim3(128),
                 0, c.stream, a, p, b.splits);
    st = cuda_status("paged_merge_kernel");
    if (st) return st;
  }
  return a.weights == nullptr ? OSCAR_OK : launch_mass<D, T>(c, b);
}

template <typename T>
int launch_paged_d(int d, const PagedCall& c, const PagedBatch& b) {
  if (b.cls == kChunk) {
    if (d == 256) return launch_paged<256, T, false>(c, b);
    if (d == 128) return launch_paged<128, T, false>(c, b);
    return launch_paged<64, T, false>(c, b);
  }
  if (d == 256) return launch_paged<256, T, true>(c, b);
  if (d == 128) return launch_paged<128, T, true>(c, b);
  return launch_paged<64, T, true>(c, b);
}

}  // namespace

extern "C" {

int oscar_set_wait_limit(int tries) {
  if (tries < -1) return fail(OSCAR_ERR_INVALID, "the wait limit must be -1 (default) or a number of tries");
  g_wait_tries.store(tries < 0 ? oscar::kPgTries : (uint32_t)tries);
  return OSCAR_OK;
}

int64_t oscar_paged_attention_workspace(const int32_t* qsl, const int32_t* seqs, int32_t num_requests,
                                        int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
                                        int32_t weighted) {
  if (num_requests < 0 || !qsl || check_paged(qsl, seqs, num_requests, qsl[num_requests], num_q_heads, num_kv_heads) ||
      !kernel_head_dim(head_dim))
    return -1;
  int64_t need = 0;
  PagedBatch b;
  for (int cls = 0; cls < kClasses; ++cls)
    for (int r = 0; r < num_requests;) {
      r = paged_batch(b, (PagedClass)cls, r, qsl, seqs, num_requests, num_q_heads / num_kv_heads, num_kv_heads, head_dim,
                      weighted != 0, device_info().sms);
      if (b.plan.num_req > 0)
        need = std::max(need, paged_space(b, qsl[num_requests], num_q_heads, head_dim, weighted != 0).total());
    }
  return need;
}

int oscar_paged_attention(const void* q, int64_t q_token_stride, int64_t q_head_stride, int32_t dtype,
                          int64_t n_tokens, int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
                          const void* k_cache, const void* v_cache, int64_t num_blocks, int32_t block_size,
                          int64_t k_stride_block, int64_t k_stride_token, int64_t k_stride_head,
                          int64_t v_stride_block, int64_t v_stride_token, int64_t v_stride_head,
                          const int32_t* block_table, int64_t bt_rows, int64_t bt_cols, int64_t bt_stride,
                          const int32_t* qsl, const int32_t* seqs, int32_t num_requests, float scale, float* weights,
                          int32_t observe, void* out, float* lse, void* workspace, int64_t workspace_bytes,
                          void* stream) {
  if (!half_dtype(dtype)) return fail(OSCAR_ERR_UNSUPPORTED, "paged_attention: queries must be bf16 or fp16");
  if (!kernel_head_dim(head_dim))
    return fail(OSCAR_ERR_UNSUPPORTED, "paged_attention: head_dim %d: kernels exist for 64, 128, 256", head_dim);
  int st = check_paged(qsl, seqs, num_requests, n_tokens, num_q_heads, num_kv_heads);
  if (st) return st;
  if (!std::isfinite(scale) || scale <= 0.0f) return fail(OSCAR_ERR_INVALID, "paged_attention: scale must be positive and finite");
  if (weights != nullptr && observe < 1) return fail(OSCAR_ERR_INVALID, "paged_attention: observe must be at least 1");
  st = check_cache("paged_attention", k_cache, num_blocks, block_size, num_kv_heads, head_dim, k_stride_block,
                   k_stride_token, k_stride_head);
  if (!st)
    st = check_cache("paged_attention", v_cache, num_blocks, block_size, num_kv_heads, head_dim, v_stride_block,
                     v_stride_token, v_stride_head);
  if (st) return st;
  bool any = false;
  for (int r = 0; r < num_requests; ++r) {
    if (qsl[r + 1] == qsl[r] || seqs[r] == 0) continue;
    any = true;
    if (((int64_t)seqs[r] + block_size - 1) / block_size > bt_cols)
      return fail(OSCAR_ERR_INVALID, "paged_attention: block table cannot cover the sequence");
  }
  if (bt_rows < num_requests || bt_cols < 0 || bt_stride < bt_cols)
    return fail(OSCAR_ERR_INVALID, "paged_attention: missing request block-table rows");
  if (any && (!block_table || num_blocks < 1))
    return fail(OSCAR_ERR_INVALID, "paged_attention: a sequence needs caches and a block table");
  if (n_tokens == 0) return OSCAR_OK;
  if (!q || !out || !lse) return fail(OSCAR_ERR_INVALID, "paged_attention: null pointer");
  if (!aligned16(q) || (reinterpret_cast<uintptr_t>(out) & 31) || (reinterpret_cast<uintptr_t>(workspace) & 31) ||
      (q_token_stride | q_head_stride) % 8)
    return fail(OSCAR_ERR_INVALID, "paged_attention: query rows must be 16-byte, output and workspace 32-byte aligned");
  if (weights != nullptr) {
    bool again = false;  // are queries read after outputs were written?
    for (int r = 0; r < num_requests; ++r)
      again = again || (qsl[r + 1] > qsl[r] && paged_class(qsl[r + 1] - qsl[r], seqs[r], num_q_heads / num_kv_heads,
                                                           num_kv_heads, true) != kFew);
    const auto q0 = reinterpret_cast<uintptr_t>(q), o0 = reinterpret_cast<uintptr_t>(out);
    const auto q1 = q0 + 2 * ((n_tokens - 1) * q_token_stride + (num_q_heads - 1) * q_head_stride + head_dim);
    if (again && o0 < q1 && q0 < o0 + 2 * n_tokens * num_q_heads * head_dim)
      return fail(OSCAR_ERR_INVALID, "paged_attention: out must not overlap q where the keys are weighed");
  }
  PagedCall c{};
  oscar::PagedArgs& a = c.args;
  a.q = q, a.q_tok = q_token_stride, a.q_head = q_head_stride;
  a.out = out, a.lse = lse;
  a.hq = num_q_heads, a.hk = num_kv_heads, a.group = num_q_heads / num_kv_heads;
  a.num_blocks = num_blocks, a.bs = block_size;
  a.page = fast_div((uint32_t)block_size);
  a.box = std::min(oscar::kPgKeys, block_size & -block_size);
  a.table = block_table, a.table_stride = bt_stride;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.weights = weights;
  a.observe = weights != nullptr ? observe : 0;
  a.tries = g_wait_tries.load(std::memory_order_relaxed);
  c.k_cache = k_cache, c.kcb = k_stride_block, c.kct = k_stride_token, c.kch = k_stride_head;
  c.stream = reinterpret_cast<cudaStream_t>(stream);
  // without any key nothing is loaded: the maps only have to be valid
  const void* kb = any ? k_cache : q;
  const void* vb = any ? v_cache : q;
  const int64_t nb = any ? num_blocks : 1;
  if (!paged_map(&c.kmap, kb, dtype, nb, block_size, num_kv_heads, head_dim, k_stride_block, k_stride_token, k_stride_head, a.box) ||
      !paged_map(&c.vmap, vb, dtype, nb, block_size, num_kv_heads, head_dim, v_stride_block, v_stride_token, v_stride_head, a.box))
    return fail(OSCAR_ERR_INVALID, "paged_attention: the caches' strides do not fit a tensor map");
  PagedBatch b;
  for (int cls = 0; cls < kClasses; ++cls)
    for (int r = 0; r < num_requests;) {
      r = paged_batch(b, (PagedClass)cls, r, qsl, seqs, num_requests, a.group, num_kv_heads, head_dim,
                      weights != nullptr, device_info().sms);
      if (b.plan.num_req == 0) continue;
      if (!query_map(&c.qmap, q, dtype, n_tokens, num_q_heads, head_dim, q_token_stride, q_head_stride, a.group,
                     b.plan.box_tokens))
        return fail(OSCAR_ERR_INVALID, "paged_attention: the queries' strides do not fit a tensor map");
      const PagedSpace space = paged_space(b, n_tokens, num_q_heads, head_dim, weights != nullptr);
      if (workspace_bytes < space.total() || !workspace)
        return fail(OSCAR_ERR_INVALID, "paged_attention: workspace of %lld bytes, %lld needed", (long long)workspace_bytes,
                    (long long)space.total());
      uint8_t* at = reinterpret_cast<uint8_t*>(workspace);
      a.stats = weights != nullptr ? reinterpret_cast<float2*>(at) : nullptr;
      a.part_ml = reinterpret_cast<float2*>(at + space.stats);
      a.part_o = reinterpret_cast<float*>(at + space.stats + space.part_ml);
      a.score_rows = b.rows;
      a.scores = space.scores ? reinterpret_cast<float*>(at + space.stats + space.part_ml + space.part_o) : nullptr;
      st = dtype == OSCAR_DTYPE_BF16 ? launch_paged_d<__nv_bfloat16>(head_dim, c, b)
                                     : launch_paged_d<__half>(head_dim, c, b);
      if (st) return st;
    }
  return OSCAR_OK;
}

// ---------------------------------------------------------------------------
int oscar_evict_cache(void* k_cache, void* v_cache, int32_t head_dim, int64_t num_blocks, int32_t block_size,
                      int32_t num_kv_heads, int64_t k_stride_block, int64_t k_stride_token, int64_t k_stride_head,
                      int64_t v_stride_block, int64_t v_stride_token, int64_t v_stride_head, float* weights,
                      const int32_t* block_table, int64_t bt_rows, int64_t bt_cols, int64_t bt_stride,
                      const int32_t* dst_table, int64_t dst_rows, int64_t dst_cols, int64_t dst_stride,
                      const int32_t* seqs, int32_t num_requests, int32_t keep, int32_t sink, int32_t recent,
                      int32_t* kept, int32_t kept_cols, void* stream) {
  if (!kernel_head_dim(head_dim))
    return fail(OSCAR_ERR_UNSUPPORTED, "evict_cache: head_dim %d: kernels exist for 64, 128, 256", head_dim);
  if (keep < 1 || sink < 0 || recent < 0 || (int64_t)sink + recent > keep)
    return fail(OSCAR_ERR_INVALID, "evict_cache: keep must be at least 1 and hold the sink and recent tokens");
  if (num_requests < 0 || (num_requests > 0 && !seqs) || num_kv_heads < 1 || num_kv_heads > 255)
    return fail(OSCAR_ERR_INVALID, "evict_cache: invalid geometry");
  int st = check_cache("evict_cache", k_cache, num_blocks, block_size, num_kv_heads, head_dim, k_stride_block,
                       k_stride_token, k_stride_head);
  if (!st)
    st = check_cache("evict_cache", v_cache, num_blocks, block_size, num_kv_heads, head_dim, v_stride_block,
                     v_stride_token, v_stride_head);
  if (st) return st;
  const bool in_place = dst_table == nullptr || (dst_table == block_table && dst_stride == bt_stride);
  int most = 0;
  bool any = false;
  for (int r = 0; r < num_requests; ++r) {
    if (seqs[r] < 0) return fail(OSCAR_ERR_INVALID, "evict_cache: lengths must not be negative");
    if (seqs[r] > kMaxLength) return fail(OSCAR_ERR_UNSUPPORTED, "evict_cache: length of request %d too long", r);
    const int n = std::min(seqs[r], keep);
    most = std::max(most, n);
    any = any || n > 0;
    if (((int64_t)seqs[r] + block_size - 1) / block_size > bt_cols)
      return fail(OSCAR_ERR_INVALID, "evict_cache: block table cannot cover the sequence");
    if (!in_place && ((int64_t)n + block_size - 1) / block_size > dst_cols)
      return fail(OSCAR_ERR_INVALID, "evict_cache: destination table cannot cover the kept keys");
  }
  if (bt_rows < num_requests || bt_stride < bt_cols || (!in_place && (dst_rows < num_requests || dst_stride < dst_cols)))
    return fail(OSCAR_ERR_INVALID, "evict_cache: missing request block-table rows");
  if (kept_cols < most) return fail(OSCAR_ERR_INVALID, "evict_cache: the list of kept keys has %d places, %d needed", kept_cols, most);
  if (!any) return OSCAR_OK;
  if (!weights || !block_table || !kept || num_blocks < 1) return fail(OSCAR_ERR_INVALID, "evict_cache: null pointer");
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  oscar::EvictArgs a{};
  a.k = reinterpret_cast<uint8_t*>(k_cache), a.v = reinterpret_cast<uint8_t*>(v_cache);
  a.kb = 2 * k_stride_block, a.kt = 2 * k_stride_token, a.kh = 2 * k_stride_head;
  a.vb = 2 * v_stride_block, a.vt = 2 * v_stride_token, a.vh = 2 * v_stride_head;
  a.weights = weights;
  a.num_blocks = num_blocks, a.bs = block_size, a.hk = num_kv_heads;
  a.page = fast_div((uint32_t)block_size);
  a.row_bytes = 2 * head_dim;
  a.table = block_table, a.table_stride = bt_stride;
  a.dst = in_place ? block_table : dst_table, a.dst_stride = in_place ? bt_stride : dst_stride;
  a.keep = keep, a.sink = sink, a.recent = recent;
  a.kept = kept, a.kept_stride = kept_cols;
  oscar::EvictPlan p;
  for (int r = 0; r < num_requests;) {
    p.num_req = 0;
    int longest = 0, moved = 0;
    for (; r < num_requests && p.num_req < oscar::kEvReqs; ++r) {
      p.req_id[p.num_req] = r;
      p.seq[p.num_req++] = seqs[r];
      longest = std::max(longest, std::min(oscar::kEvCached, (seqs[r] + oscar::kEvCluster - 1) / oscar::kEvCluster + 31));
      moved = std::max(moved, std::min(seqs[r], keep));
    }
    allow_smem<oscar::evict_select_kernel>(oscar::kEvCached * sizeof(float));
    launch_pdl_cluster(oscar::kEvCluster, oscar::evict_select_kernel, dim3(p.num_req * oscar::kEvCluster, num_kv_heads),
                       dim3(oscar::kEvThreads), std::max(16, longest * (int)sizeof(float)), s, a, p);
    st = cuda_status("evict_select_kernel");
    if (st) return st;
    if (moved == 0) continue;
    if (in_place) {
      launch_pdl(oscar::evict_move_kernel, dim3(p.num_req * num_kv_heads, 2, a.row_bytes / 128),
                 dim3(oscar::kEvMoveThreads), 0, s, a, p);
      st = cuda_status("evict_move_kernel");
    } else {
      // about eight CTAs per SM over all heads, each with several steps
      const int rows = oscar::kEvMoveThreads / (a.row_bytes / 16) * oscar::kEvRows;
      const int heads = p.num_req * num_kv_heads, most = (moved + rows - 1) / rows;
      const int want = (8 * std::max(device_info().sms, 1) + heads - 1) / heads;
      launch_pdl(oscar::evict_copy_kernel, dim3(std::min(most, std::max(want, 1)), heads), dim3(oscar::kEvMoveThreads), 0, s,
                 a, p);
      st = cuda_status("evict_copy_kernel");
    }
    if (st) return st;
  }
  return OSCAR_OK;
}

}  // extern "C"
