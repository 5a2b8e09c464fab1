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
// token's cos / sin and the weights stay in registers.  With few tokens the
// heads of a token are split over several warps (`splits`).
#pragma once

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

template <typename T>
OSCAR_DEVINL void hn_unpack(const uint4& w, float (&x)[8]) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    T lo, hi;
    *reinterpret_cast<uint16_t*>(&lo) = (uint16_t)(u[i] & 0xffffu);
    *reinterpret_cast<uint16_t*>(&hi) = (uint16_t)(u[i] >> 16);
    x[2 * i] = Elem<T>::to_f32(lo);
    x[2 * i + 1] = Elem<T>::to_f32(hi);
  }
}

template <typename T>
OSCAR_DEVINL uint4 hn_pack(const float (&x)[8]) {
  return make_uint4(pack2_f32<T>(x[0], x[1]), pack2_f32<T>(x[2], x[3]), pack2_f32<T>(x[4], x[5]),
                    pack2_f32<T>(x[6], x[7]));
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
__global__ void __launch_bounds__(kHnThreads) head_norm_kernel(const __grid_constant__ HeadNormArgs a, const int splits) {
  constexpr int L = D / 8;     // lanes per vector
  constexpr int V = 32 / L;    // tokens per warp
  pdl_release();
  const int lane = threadIdx.x & 31;
  const int sub = lane % L, d0 = 8 * sub;
  const int heads = a.hq + a.hk + (a.v_cache != nullptr ? a.hk : 0);
  const int groups = (heads + kHnHeads - 1) / kHnHeads;
  const int64_t item = (int64_t)blockIdx.x * (kHnThreads / 32) + (threadIdx.x >> 5);
  const int64_t tok = (item / splits) * V + lane / L;
  const bool live = tok < a.n;
  const bool rotates = d0 < a.rot;
  pdl_wait();
  int64_t pos = live ? a.positions[tok] : 0;
  int64_t slot = live && a.slots != nullptr ? a.slots[tok] : -1;
  const T *q = nullptr, *k = nullptr, *v = nullptr;
  if (live) {
    q = reinterpret_cast<const T*>(a.q) + tok * a.q_tok + d0;
    k = reinterpret_cast<const T*>(a.k) + tok * a.k_tok + d0;
    if (a.v_cache != nullptr) v = reinterpret_cast<const T*>(a.v) + tok * a.v_tok + d0;
  }
  auto fetch = [&](int g, uint4 (&raw)[kHnHeads]) {
#pragma unroll
    for (int i = 0; i < kHnHeads; ++i) {
      const int h = g * kHnHeads + i;
      raw[i] = make_uint4(0, 0, 0, 0);
      if (live && h < heads) {
        const T* src = h < a.hq ? q + h * a.q_head : h < a.hq + a.hk ? k + (h - a.hq) * a.k_head : v + (h - a.hq - a.hk) * a.v_head;
        raw[i] = __ldcs(reinterpret_cast<const uint4*>(src));
      }
    }
  };
  int g = (int)(item % splits);
  uint4 raw[kHnHeads];
  fetch(g, raw);
  // the weights of the lane's dims, with the offset
  float wq[8], wk[8];
  hn_load<T, 8>(a.wq, d0, a.w_f32, wq);
  hn_load<T, 8>(a.wk, d0, a.w_f32, wk);
#pragma unroll
  for (int j = 0; j < 8; ++j) wq[j] += a.offset, wk[j] += a.offset;
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
  float c[8], s[8];
  const int half = a.rot >> 1;
  const bool upper = !a.interleaved && d0 >= half;  // the lane holds the second member of its pairs
  if (rotates) {
    const int64_t row = pos * a.cs_stride;
    if (a.interleaved) {
      float c4[4], s4[4];
      hn_load<T, 4>(a.cos_sin, row + d0 / 2, a.cs_f32, c4);
      hn_load<T, 4>(a.cos_sin, row + half + d0 / 2, a.cs_f32, s4);
#pragma unroll
      for (int i = 0; i < 4; ++i) c[i] = c4[i], s[i] = s4[i];
    } else {
      hn_load<T, 8>(a.cos_sin, row + (upper ? d0 - half : d0), a.cs_f32, c);
      hn_load<T, 8>(a.cos_sin, row + half + (upper ? d0 - half : d0), a.cs_f32, s);
      if (!upper) {
#pragma unroll
        for (int j = 0; j < 8; ++j) s[j] = -s[j];
      }
    }
  }
  const int partner = (upper ? lane - a.rot / 16 : lane + a.rot / 16) & 31;
  T *ck = nullptr, *cv = nullptr;  // the token's cache rows
  if (slot >= 0) {
    const int64_t blk = slot <= 0x7fffffff ? (int64_t)((uint32_t)slot / (uint32_t)a.bs) : slot / a.bs;
    const int64_t off = slot - blk * a.bs;
    ck = reinterpret_cast<T*>(a.k_cache) + blk * a.kcb + off * a.kct + d0;
    cv = reinterpret_cast<T*>(a.v_cache) + blk * a.vcb + off * a.vct + d0;
  }
  T* oq = reinterpret_cast<T*>(a.out_q) + tok * a.oq_tok + d0;
  T* ok = a.out_k == nullptr ? nullptr : reinterpret_cast<T*>(a.out_k) + tok * a.ok_tok + d0;
  const bool writes = live && known;
#pragma unroll 1
  for (; g < groups; g += splits) {
    uint4 next[kHnHeads];
    fetch(g + splits, next);  // (past the heads: nothing is loaded)
#pragma unroll
    for (int i = 0; i < kHnHeads; ++i) {
      const int h = g * kHnHeads + i;
      if (h >= heads) break;  // uniform over the warp
      const int kv = h - a.hq;
      if (kv >= a.hk) {  // a value head: straight to the cache
        if (cv != nullptr) *reinterpret_cast<uint4*>(cv + (kv - a.hk) * a.vch) = raw[i];
        continue;
      }
      float x[8];
      hn_unpack<T>(raw[i], x);
      float ss = 0.0f;
#pragma unroll
      for (int j = 0; j < 8; ++j) ss = fmaf(x[j], x[j], ss);
#pragma unroll
      for (int o = L / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      const float r = rsqrtf(ss * (1.0f / D) + a.eps);
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = x[j] * r * (kv < 0 ? wq[j] : wk[j]);
      if (a.interleaved) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float u = x[2 * j], w = x[2 * j + 1];
          if (rotates) x[2 * j] = u * c[j] - w * s[j], x[2 * j + 1] = w * c[j] + u * s[j];
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float other = __shfl_sync(0xffffffffu, x[j], partner);
          if (rotates) x[j] = x[j] * c[j] + other * s[j];
        }
      }
      const uint4 y = hn_pack<T>(x);
      if (kv < 0) {
        if (writes) *reinterpret_cast<uint4*>(oq + h * a.oq_head) = y;
      } else {
        if (writes && ok != nullptr) *reinterpret_cast<uint4*>(ok + kv * a.ok_head) = y;
        if (ck != nullptr) *reinterpret_cast<uint4*>(ck + kv * a.kch) = y;
      }
    }
#pragma unroll
    for (int i = 0; i < kHnHeads; ++i) raw[i] = next[i];
  }
}

}  // namespace oscar
