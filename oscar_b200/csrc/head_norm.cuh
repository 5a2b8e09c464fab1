// Norm of the query and key heads with the position rotation in the same
// pass, and the write of the step's keys and values to a 16-bit paged cache.
//
//   y = x * rsqrt(mean(x^2) + eps) * (w + offset)          (per head, fp32)
//   y[a], y[b] = y[a] cos - y[b] sin, y[b] cos + y[a] sin   (first `rot` dims)
//   pairs (a, b): (i, i + rot/2), or neighbours (2i, 2i + 1) when interleaved
//
// rounded once to the tensor's type.  A vector of D dims lies on D / 8 lanes,
// 16 bytes each, so the mean is a butterfly over those lanes and a pair's
// partner is in the same lane (neighbours) or rot / 16 lanes away at the same
// position (halves): nothing goes through shared memory.  Bound by bytes: each
// vector is read and written once.  A warp walks the heads of one token (of
// 256 / D tokens), kHnHeads at a time with the next ones' loads in flight; the
// token's cos / sin are folded into the query weights, then into the key
// weights.  With few tokens the heads of a token are split over several warps
// (`splits`).  15360 tokens of Hq 24 / Hk 4 / D 256: 99.5 us, 5.1 TB/s, 0.78 of
// the measured copy bandwidth (without the prefetch 106 us; weights folded for
// each four heads 107 us; scalar fp32 instead of pairs 109 us).
#pragma once

#include <type_traits>

#include "common.cuh"

namespace oscar {

constexpr int kHnHeads = 4;      // heads per warp, loads in flight per lane
constexpr int kHnThreads = 128;

struct HeadNormArgs {
  const void *q, *k, *v;                       // v may be null (no cache)
  int64_t q_tok, q_head, k_tok, k_head, v_tok, v_head;  // strides in elements
  void *out_q, *out_k;                         // out_k may be null
  int64_t oq_tok, oq_head, ok_tok, ok_head;
  const void *wq, *wk;                         // [D], fp32 or the tensors' type
  int w_f32;
  float eps, offset;
  const void* cos_sin;                         // [max_pos, rot] (cos, then sin), fp32 or the tensors' type
  int cs_f32;
  int64_t cs_stride, max_pos;
  int rot, interleaved;
  const int64_t* positions;
  int64_t n;
  int hq, hk;
  void *k_cache, *v_cache;                     // may be null
  int64_t num_blocks;
  int bs;
  int64_t kcb, kct, kch, vcb, vct, vch;        // cache strides in elements
  const int64_t* slots;
};

// 16 bytes -> four pairs of fp32
template <typename T>
OSCAR_DEVINL void hn_pairs(const uint4& w, uint64_t (&x)[4]) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (std::is_same<T, __nv_bfloat16>::value) {  // the upper half of an fp32
      x[i] = (uint64_t)(u[i] << 16) | ((uint64_t)(u[i] & 0xffff0000u) << 32);
    } else {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
      x[i] = f2_pack(f.x, f.y);
    }
  }
}
template <typename T>
OSCAR_DEVINL uint4 hn_pack_pairs(const uint64_t (&x)[4]) {
  uint32_t u[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      const __nv_bfloat162 v = __floats2bfloat162_rn(f2_lo(x[i]), f2_hi(x[i]));
      u[i] = *reinterpret_cast<const uint32_t*>(&v);
    } else {
      const __half2 v = __floats2half2_rn(f2_lo(x[i]), f2_hi(x[i]));
      u[i] = *reinterpret_cast<const uint32_t*>(&v);
    }
  }
  return make_uint4(u[0], u[1], u[2], u[3]);
}

// N consecutive values (N * element size <= 32 bytes, naturally aligned) in fp32
template <typename T, int N>
OSCAR_DEVINL void hn_load(const void* base, int64_t at, int f32, float (&x)[N]) {
  if (f32) {
    const float4* p = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(base) + at);
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const float4 v = __ldg(p + i);
      x[4 * i] = v.x, x[4 * i + 1] = v.y, x[4 * i + 2] = v.z, x[4 * i + 3] = v.w;
    }
  } else {
    const uint2* p = reinterpret_cast<const uint2*>(reinterpret_cast<const T*>(base) + at);
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const uint2 v = __ldg(p + i);
      const uint32_t u[2] = {v.x, v.y};
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        T lo, hi;
        *reinterpret_cast<uint16_t*>(&lo) = (uint16_t)(u[j] & 0xffffu);
        *reinterpret_cast<uint16_t*>(&hi) = (uint16_t)(u[j] >> 16);
        x[4 * i + 2 * j] = Elem<T>::to_f32(lo);
        x[4 * i + 2 * j + 1] = Elem<T>::to_f32(hi);
      }
    }
  }
}

template <typename T, int D>
__global__ void __launch_bounds__(kHnThreads, 5) head_norm_kernel(const __grid_constant__ HeadNormArgs a, const int splits) {
  constexpr int L = D / 8;     // lanes per vector
  constexpr int V = 32 / L;    // tokens per warp
  pdl_release();
  const int lane = threadIdx.x & 31;
  const int sub = lane % L, d0 = 8 * sub;
  const int q_groups = (a.hq + kHnHeads - 1) / kHnHeads, k_groups = (a.hk + kHnHeads - 1) / kHnHeads;
  const int groups = q_groups + k_groups * (a.v_cache != nullptr ? 2 : 1);
  const int64_t item = (int64_t)blockIdx.x * (kHnThreads / 32) + (threadIdx.x >> 5);
  const int64_t tok = (item / splits) * V + lane / L;
  const bool live = tok < a.n;
  const bool rotates = d0 < a.rot;
  pdl_wait();
  int64_t pos = live ? a.positions[tok] : 0;
  int64_t slot = live && a.slots != nullptr ? a.slots[tok] : -1;
  const bool known = pos >= 0 && pos < a.max_pos;
  if (!known) {
    if (sub == 0 && live) flag_error(64u);
    pos = 0;
    slot = -1;
  }
  if (slot >= a.num_blocks * a.bs) {
    if (sub == 0) flag_error(1u);
    slot = -1;
  }
  // cos / sin of the lane's dims: 8 pairs (halves; the lane holds one side) or 4 (neighbours).
  // With the partner's value p: x cos - p sin, or x cos + p sin on the upper side
  float c[8], s[8];
  const int half = a.rot >> 1;
  const bool upper = !a.interleaved && d0 >= half;  // the lane holds the second member of its pairs
#pragma unroll
  for (int j = 0; j < 8; ++j) c[j] = 1.0f, s[j] = 0.0f;
  if (rotates) {
    const int64_t row = pos * a.cs_stride;
    if (a.interleaved) {
      float c4[4], s4[4];
      hn_load<T, 4>(a.cos_sin, row + d0 / 2, a.cs_f32, c4);
      hn_load<T, 4>(a.cos_sin, row + half + d0 / 2, a.cs_f32, s4);
#pragma unroll
      for (int i = 0; i < 4; ++i) c[2 * i] = c[2 * i + 1] = c4[i], s[2 * i] = -s4[i], s[2 * i + 1] = s4[i];
    } else {
      hn_load<T, 8>(a.cos_sin, row + (upper ? d0 - half : d0), a.cs_f32, c);
      hn_load<T, 8>(a.cos_sin, row + half + (upper ? d0 - half : d0), a.cs_f32, s);
      if (!upper) {
#pragma unroll
        for (int j = 0; j < 8; ++j) s[j] = -s[j];
      }
    }
  }
  // the lane with the partners (halves), and where their weights are
  const int partner = rotates && !a.interleaved ? (upper ? lane - a.rot / 16 : lane + a.rot / 16) : lane;
  const int p0 = d0 + 8 * (partner - lane);
  int64_t k_at = 0, v_at = 0;  // the token's cache rows
  if (slot >= 0) {
    const int64_t blk = slot <= 0x7fffffff ? (int64_t)((uint32_t)slot / (uint32_t)a.bs) : slot / a.bs;
    const int64_t off = slot - blk * a.bs;
    k_at = blk * a.kcb + off * a.kct + d0;
    v_at = blk * a.vcb + off * a.vct + d0;
  }
  const bool writes = live && known;
  // folded: y = (x w' + p wp') r, w' = (w + offset) cos, wp' = (w of the partner + offset) (+-sin)
  uint64_t w[4], wp[4];
  int folded = -1;  // the kind they are for
  struct Group {  // kind 0: queries, 1: keys, 2: values (uniform over the warp)
    int kind, h0, heads;
  };
  auto group = [&](int g) -> Group {
    if (g < q_groups) return {0, g * kHnHeads, a.hq};
    if (g < q_groups + k_groups) return {1, (g - q_groups) * kHnHeads, a.hk};
    return {2, (g - q_groups - k_groups) * kHnHeads, a.hk};
  };
  auto fetch = [&](int g, uint4 (&raw)[kHnHeads]) {
    const Group u = group(g);
    const int64_t head = u.kind == 0 ? a.q_head : u.kind == 1 ? a.k_head : a.v_head;
    const T* src = u.kind == 0   ? reinterpret_cast<const T*>(a.q) + tok * a.q_tok
                   : u.kind == 1 ? reinterpret_cast<const T*>(a.k) + tok * a.k_tok
                                 : reinterpret_cast<const T*>(a.v) + tok * a.v_tok;
    src += u.h0 * head + d0;
#pragma unroll
    for (int i = 0; i < kHnHeads; ++i) {
      raw[i] = make_uint4(0, 0, 0, 0);
      if (live && g < groups && u.h0 + i < u.heads) raw[i] = __ldcs(reinterpret_cast<const uint4*>(src + i * head));
    }
  };
  int g = (int)(item % splits);
  uint4 next[kHnHeads];
  fetch(g, next);
#pragma unroll 1
  for (; g < groups; g += splits) {
    const Group u = group(g);
    const int kind = u.kind, h0 = u.h0, heads = u.heads;
    uint4 raw[kHnHeads];
#pragma unroll
    for (int i = 0; i < kHnHeads; ++i) raw[i] = next[i];
    fetch(g + splits, next);
    if (kind == 2) {  // value heads: straight to the cache
#pragma unroll
      for (int i = 0; i < kHnHeads; ++i)
        if (slot >= 0 && h0 + i < heads)
          *reinterpret_cast<uint4*>(reinterpret_cast<T*>(a.v_cache) + v_at + (h0 + i) * a.vch) = raw[i];
      continue;
    }
    if (kind != folded) {
      folded = kind;
      float u[8], v[8];
      const void* weight = kind == 0 ? a.wq : a.wk;
      hn_load<T, 8>(weight, d0, a.w_f32, u);
      hn_load<T, 8>(weight, p0, a.w_f32, v);
#pragma unroll
      for (int j = 0; j < 8; j += 2) {
        w[j / 2] = f2_pack((u[j] + a.offset) * c[j], (u[j + 1] + a.offset) * c[j + 1]);
        wp[j / 2] = a.interleaved ? f2_pack((v[j + 1] + a.offset) * s[j], (v[j] + a.offset) * s[j + 1])
                                  : f2_pack((v[j] + a.offset) * s[j], (v[j + 1] + a.offset) * s[j + 1]);
      }
    }
    T* out = kind == 0 ? reinterpret_cast<T*>(a.out_q) + tok * a.oq_tok
             : a.out_k != nullptr ? reinterpret_cast<T*>(a.out_k) + tok * a.ok_tok : nullptr;
    const int64_t out_head = kind == 0 ? a.oq_head : a.ok_head;
#pragma unroll
    for (int i = 0; i < kHnHeads; ++i) {
      const int h = h0 + i;
      if (h >= heads) break;  // uniform over the warp
      uint64_t x[4], y[4];
      hn_pairs<T>(raw[i], x);
      uint64_t s2 = f2_mul(x[0], x[0]);
#pragma unroll
      for (int j = 1; j < 4; ++j) s2 = f2_fma(x[j], x[j], s2);
      float ss = f2_lo(s2) + f2_hi(s2);
#pragma unroll
      for (int o = L / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      const float r = rsqrtf(ss * (1.0f / D) + a.eps);
      const uint64_t r2 = f2_pack(r, r);
      uint64_t p[4];
      if (a.interleaved) {
#pragma unroll
        for (int j = 0; j < 4; ++j) p[j] = f2_pack(f2_hi(x[j]), f2_lo(x[j]));
      } else {
        // the partners as they came: four exchanges instead of eight
        uint4 other;
        other.x = __shfl_sync(0xffffffffu, raw[i].x, partner);
        other.y = __shfl_sync(0xffffffffu, raw[i].y, partner);
        other.z = __shfl_sync(0xffffffffu, raw[i].z, partner);
        other.w = __shfl_sync(0xffffffffu, raw[i].w, partner);
        hn_pairs<T>(other, p);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) y[j] = f2_mul(f2_fma(p[j], wp[j], f2_mul(x[j], w[j])), r2);
      const uint4 packed = hn_pack_pairs<T>(y);
      if (writes && out != nullptr) *reinterpret_cast<uint4*>(out + h * out_head + d0) = packed;
      if (kind == 1 && slot >= 0) *reinterpret_cast<uint4*>(reinterpret_cast<T*>(a.k_cache) + k_at + h * a.kch) = packed;
    }
  }
}

}  // namespace oscar
