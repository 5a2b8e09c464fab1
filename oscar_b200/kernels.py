"""Kernel-level API over the C ABI (torch tensors in, device work out).

Mirrors the reference's kernel entry points for the hot path:
  * ``oscar_store``       kernels/store_kernel.py:54-102 / :247-279 (+ clip of backend.py:140-146)
  * ``staging_invalidate`` backend.py:172-176
  * ``staging_write``     backend.py:513-555
  * ``slab_attention``    kernels/slab_attention.py:376-476 (semantics of
                          kernels/streaming_attention.py:134-196)
  * ``slab_attention_shard`` one history shard of slab_attention.py:458-475
                          (split-KV across GPUs)
  * ``merge_slab``        kernels/slab_attention.py:341-373

and has the attention step of a 16-bit paged layer (the MTP draft layers,
which the reference leaves to the engine): ``qk_norm_rope``,
``paged_attention`` and ``evict_cache``.

Layout problems raise ValueError with the reference's messages; every call
is asynchronous on the current CUDA stream and never synchronises the host.
There is no CPU path: CPU tensors raise.
"""
from __future__ import annotations

import numpy as np
import torch

from . import _native
from ._native import check
from .format import check_d

# bound on the attention workspace (split partials, then the continuation pre-pass tiles:
# ceil(seq / 64) x Hk x 64 KiB per request); the allocation is what a call needs, up to this
DEFAULT_WORKSPACE_BYTES = 512 * 1024 * 1024

_DTYPES = {torch.float32: _native.DTYPE_F32, torch.bfloat16: _native.DTYPE_BF16, torch.float16: _native.DTYPE_F16}


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


# the current stream's handle without a Stream object (0.1 instead of 2.3 us a call) where torch offers it
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


def _stream(device: torch.device) -> int:
    return _raw_stream(torch.cuda.current_device() if device.index is None else device.index)


def _require_cuda(*tensors: torch.Tensor | None) -> torch.device:
    dev = None
    for t in tensors:
        if t is None:
            continue
        if t.device.type != "cuda":
            raise ValueError("OSCAR B200 kernels require CUDA tensors (there is no CPU path)")
        if dev is None:
            dev = t.device
        elif t.device != dev:
            raise ValueError("all tensors must be on the same CUDA device")
    if dev is None:
        raise ValueError("no tensor given")
    return dev


def _byte_view(cache: torch.Tensor) -> torch.Tensor:
    c8 = cache.view(torch.uint8)
    if c8.ndim != 4 or not c8.is_contiguous():
        raise ValueError("OSCAR requires contiguous [blocks, tokens, heads, bytes] caches")
    return c8


def _clip_ok(r: float) -> float:
    r = float(r)
    if not 0.0 <= r <= 1.0:
        raise ValueError("OSCAR clip ratios must be finite and in [0, 1]")
    return r


# ---------------------------------------------------------------------------
def oscar_store(k_rot: torch.Tensor, v_rot: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                slot_mapping: torch.Tensor, k_clip_ratio: float = 0.0, v_clip_ratio: float = 0.0) -> None:
    """Clip, INT2-quantize, pack and scatter rotated K/V [N, Hk, D] into the
    paged caches in place; slot < 0 is skipped.  Bit-exact with
    oscar_store_ref for identical rotated fp32 input (clip ratios 0)."""
    dev = _require_cuda(k_rot, v_rot, k_cache, v_cache, slot_mapping)
    if k_rot.shape != v_rot.shape or k_rot.ndim != 3:
        raise ValueError("k_rot/v_rot must be [N, H, D] with equal shapes")
    n, h, d = k_rot.shape
    check_d(d)
    k8, v8 = _byte_view(k_cache), _byte_view(v_cache)
    if k8.shape[:3] != v8.shape[:3] or k8.shape[2] != h:
        raise ValueError("cache geometry does not match [N, H, D] input")
    k_rot = k_rot.to(torch.float32).contiguous()
    v_rot = v_rot.to(torch.float32).contiguous()
    slots = slot_mapping.to(device=dev, dtype=torch.int64).contiguous()
    if slots.numel() < n:
        raise ValueError("slot_mapping shorter than the token count")
    check(_native.lib().oscar_store_int2(
        k_rot.data_ptr(), v_rot.data_ptr(), n, h, d, _clip_ok(k_clip_ratio), _clip_ok(v_clip_ratio),
        k8.data_ptr(), v8.data_ptr(), k8.shape[0], k8.shape[1], *k8.stride()[:3], *v8.stride()[:3],
        slots.data_ptr(), _stream(dev)))


def oscar_store_ref(k_rot, v_rot, k_cache, v_cache, slot_mapping) -> None:
    """Name-compatible alias of kernels/store_kernel.py:54 (runs on the GPU)."""
    oscar_store(k_rot, v_rot, k_cache, v_cache, slot_mapping)


# ---------------------------------------------------------------------------
def staging_invalidate(slot_mapping: torch.Tensor, owner: torch.Tensor, block_size: int) -> None:
    """owner[seat(slot)] = -1 for every slot >= 0 (backend.py:172-176)."""
    dev = _require_cuda(slot_mapping, owner)
    if owner.dtype != torch.int64 or owner.ndim != 2 or not owner.is_contiguous():
        raise ValueError("owner must be a contiguous int64 [rows, block_size] tensor")
    slots = slot_mapping.to(device=dev, dtype=torch.int64).contiguous()
    check(_native.lib().oscar_staging_invalidate(slots.data_ptr(), slots.numel(), owner.data_ptr(),
                                                 owner.shape[0], int(block_size), _stream(dev)))


def staging_write(k_rot: torch.Tensor, v_rot: torch.Tensor, slot_mapping: torch.Tensor, qsl: torch.Tensor,
                  seqs: torch.Tensor, sink_eff: int, recent_tokens: int, stage_k: torch.Tensor,
                  stage_v: torch.Tensor, owner: torch.Tensor, seat_winner: torch.Tensor, epoch: int) -> None:
    """Sink/recent staging write of rotated, unclipped fp32 K/V [N, Hk, D]
    (backend.py:513-555).  qsl/seqs are device int32 tensors [B+1], [B]."""
    dev = _require_cuda(k_rot, v_rot, slot_mapping, qsl, seqs, stage_k, stage_v, owner, seat_winner)
    n, h, d = k_rot.shape
    rows, bs = owner.shape
    if stage_k.shape != (rows, bs, h, d) or stage_v.shape != stage_k.shape:
        raise ValueError("Invalid streaming staging geometry")
    if seat_winner.numel() != rows * bs or seat_winner.dtype != torch.int64:
        raise ValueError("seat_winner must be int64 [rows * block_size]")
    for t in (stage_k, stage_v, owner, seat_winner):
        if not t.is_contiguous():
            raise ValueError("Streaming staging tensors must be contiguous")
    k_rot = k_rot.to(torch.float32).contiguous()
    v_rot = v_rot.to(torch.float32).contiguous()
    slots = slot_mapping.to(device=dev, dtype=torch.int64).contiguous()
    qsl = qsl.to(device=dev, dtype=torch.int32).contiguous()
    seqs = seqs.to(device=dev, dtype=torch.int32).contiguous()
    check(_native.lib().oscar_staging_write(
        k_rot.data_ptr(), v_rot.data_ptr(), n, h, d, slots.data_ptr(), qsl.data_ptr(), seqs.data_ptr(),
        seqs.numel(), int(sink_eff), int(recent_tokens), stage_k.data_ptr(), stage_v.data_ptr(), owner.data_ptr(),
        rows, bs, seat_winner.data_ptr(), int(epoch) & 0xFFFFFFFF, _stream(dev)))


WRITE_STEP_MAX_TOKENS = 256
WRITE_STEP_MAX_REQUESTS = 256


def write_step(k_rot: torch.Tensor, v_rot: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
               slot_mapping: torch.Tensor, k_clip_ratio: float, v_clip_ratio: float, qsl: torch.Tensor,
               seqs: torch.Tensor, sink_eff: int, recent_tokens: int, stage_k: torch.Tensor, stage_v: torch.Tensor,
               owner: torch.Tensor) -> None:
    """oscar_store + staging_write of the same tokens in one launch (at most
    WRITE_STEP_MAX_TOKENS tokens and WRITE_STEP_MAX_REQUESTS requests): the
    write side of a decode step with the staging window on.  Needs no seat
    scratch and no epoch, so it can be captured in a CUDA graph."""
    dev = _require_cuda(k_rot, v_rot, k_cache, v_cache, slot_mapping, qsl, seqs, stage_k, stage_v, owner)
    if k_rot.shape != v_rot.shape or k_rot.ndim != 3:
        raise ValueError("k_rot/v_rot must be [N, H, D] with equal shapes")
    n, h, d = k_rot.shape
    check_d(d)
    k8, v8 = _byte_view(k_cache), _byte_view(v_cache)
    if k8.shape[:3] != v8.shape[:3] or k8.shape[2] != h:
        raise ValueError("cache geometry does not match [N, H, D] input")
    rows, bs = owner.shape
    if stage_k.shape != (rows, bs, h, d) or stage_v.shape != stage_k.shape or bs != k8.shape[1]:
        raise ValueError("Invalid streaming staging geometry")
    for t in (stage_k, stage_v, owner):
        if not t.is_contiguous():
            raise ValueError("Streaming staging tensors must be contiguous")
    k_rot = k_rot.to(torch.float32).contiguous()
    v_rot = v_rot.to(torch.float32).contiguous()
    slots = slot_mapping.to(device=dev, dtype=torch.int64).contiguous()
    qsl = qsl.to(device=dev, dtype=torch.int32).contiguous()
    seqs = seqs.to(device=dev, dtype=torch.int32).contiguous()
    if slots.numel() < n:
        raise ValueError("slot_mapping shorter than the token count")
    check(_native.lib().oscar_write_step(
        k_rot.data_ptr(), v_rot.data_ptr(), n, h, d, _clip_ok(k_clip_ratio), _clip_ok(v_clip_ratio),
        k8.data_ptr(), v8.data_ptr(), k8.shape[0], k8.shape[1], *k8.stride()[:3], *v8.stride()[:3],
        slots.data_ptr(), qsl.data_ptr(), seqs.data_ptr(), seqs.numel(), int(sink_eff), int(recent_tokens),
        stage_k.data_ptr(), stage_v.data_ptr(), owner.data_ptr(), rows, _stream(dev)))


def staging_write_noalloc(k_rot: torch.Tensor, v_rot: torch.Tensor, slot_mapping: torch.Tensor, qsl: torch.Tensor,
                          seqs: torch.Tensor, sink_eff: int, recent_tokens: int, stage_k: torch.Tensor,
                          stage_v: torch.Tensor, owner: torch.Tensor) -> None:
    """staging_write with the library's built-in seat scratch, cleared on every
    call instead of tagged by a host epoch: no caller scratch and no host state,
    so it can be captured in a CUDA graph and replayed with new slots."""
    dev = _require_cuda(k_rot, v_rot, slot_mapping, qsl, seqs, stage_k, stage_v, owner)
    n, h, d = k_rot.shape
    rows, bs = owner.shape
    if stage_k.shape != (rows, bs, h, d) or stage_v.shape != stage_k.shape:
        raise ValueError("Invalid streaming staging geometry")
    for t in (stage_k, stage_v, owner):
        if not t.is_contiguous():
            raise ValueError("Streaming staging tensors must be contiguous")
    for t in (k_rot, v_rot, slot_mapping, qsl, seqs):
        if not t.is_contiguous():
            raise ValueError("staging_write_noalloc: inputs must be contiguous")
    if k_rot.dtype != torch.float32 or v_rot.dtype != torch.float32 or slot_mapping.dtype != torch.int64 \
            or qsl.dtype != torch.int32 or seqs.dtype != torch.int32:
        raise ValueError("staging_write_noalloc: fp32 rows, int64 slots and int32 qsl / seqs expected")
    check(_native.lib().oscar_staging_write_noalloc(
        k_rot.data_ptr(), v_rot.data_ptr(), n, h, d, slot_mapping.data_ptr(), qsl.data_ptr(), seqs.data_ptr(),
        seqs.numel(), int(sink_eff), int(recent_tokens), stage_k.data_ptr(), stage_v.data_ptr(), owner.data_ptr(),
        rows, bs, _stream(dev)))


# ---------------------------------------------------------------------------
def _validate_tensors(q, k, v, kc, vc, bt, qsl, seqs, stage):
    """streaming_attention._validate_tensors (streaming_attention.py:32-65)."""
    if q.ndim != 3 or kc.ndim != 4 or kc.shape != vc.shape or kc.shape[3] != q.shape[2]:
        raise ValueError("Streaming attention requires [tokens,heads,D] queries and native 4-D caches")
    if not kc.is_contiguous() or not vc.is_contiguous():
        raise ValueError("Streaming caches must be contiguous")
    if (k is None) != (v is None):
        raise ValueError("Both new K and V must be supplied together")
    if k is not None and (k.shape != v.shape or k.shape != (q.shape[0], kc.shape[2], q.shape[2])
                          or k.dtype != q.dtype or v.dtype != q.dtype):
        raise ValueError("Current K/V must match query tokens, dtype and KV geometry")
    if bt.ndim != 2 or bt.shape[0] < len(seqs):
        raise ValueError("Missing request block-table rows")
    for a, b, seq in zip(qsl, qsl[1:], seqs):
        prefix = seq - (b - a) if k is not None else seq
        if b > a and -(-prefix // kc.shape[1]) > bt.shape[1]:
            raise ValueError("Block table cannot cover the history")
    if stage is not None:
        sk, sv, owner = stage
        shape = (owner.shape[0], kc.shape[1], kc.shape[2], q.shape[2])
        if owner.shape != shape[:2] or sk.shape != shape or sv.shape != shape or shape[0] < 1:
            raise ValueError("Invalid streaming staging geometry")
        if not all(t.is_contiguous() for t in stage):
            raise ValueError("Streaming staging tensors must be contiguous")


def slab_attention(q, k_new, v_new, kc, vc, table, qsl, seqs, scale, stage=None, *,
                   workspace_bytes: int = DEFAULT_WORKSPACE_BYTES, chunk_tokens: int | None = None):
    """Exact attention of rotated queries over paged INT2 history (+ staged
    fp32 overrides) and the causal current chunk.  Returns (out [n, Hq, D]
    fp32, lse [n, Hq] fp32 natural log).  ``qsl``/``seqs`` are host lists.

    ``workspace_bytes`` bounds the workspace: split-KV partials, then (head dim
    256, q-blocks of 128 rows) the keys' tiles written once by a pre-pass.  Any
    value is valid; a smaller one only lowers parallelism or makes each
    attention CTA dequantise its own tiles.  ``chunk_tokens`` is accepted for
    signature compatibility: the fused kernel never materialises a slab."""
    del chunk_tokens
    qsl = [int(x) for x in qsl]
    seqs = [int(x) for x in seqs]
    if (q.ndim != 3 or kc.ndim != 4 or q.shape[1] < 1 or kc.shape[2] < 1 or len(qsl) != len(seqs) + 1
            or not qsl or qsl[0] != 0 or qsl[-1] != q.shape[0] or q.shape[1] % kc.shape[2]):
        raise ValueError("Invalid slab query layout")
    if any(a > b or seq < 0 or (k_new is not None and seq < b - a) for a, b, seq in zip(qsl, qsl[1:], seqs)):
        raise ValueError("Sequence length must cover its query chunk")
    _validate_tensors(q, k_new, v_new, kc, vc, table, qsl, seqs, stage)
    dev = _require_cuda(q, k_new, v_new, kc, vc, table, *(stage or ()))
    out_dtype = q.dtype
    if q.dtype == torch.float32:
        # fp32 queries: fp16 tensor-core operands (history is fp16-exact on this path)
        q = q.half()
        k_new = None if k_new is None else k_new.half()
        v_new = None if v_new is None else v_new.half()
    if q.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError(f"unsupported query dtype {out_dtype}")
    n, hq, d = q.shape
    hk = kc.shape[2]
    q = q.contiguous()
    k_new = None if k_new is None else k_new.contiguous()
    v_new = None if v_new is None else v_new.contiguous()
    table = table.to(device=dev, dtype=torch.int32).contiguous()
    k8, v8 = _byte_view(kc), _byte_view(vc)
    sk = sv = owner = None
    rows = 0
    if stage is not None:
        sk, sv, owner = stage
        if sk.dtype != torch.float32 or sv.dtype != torch.float32 or owner.dtype != torch.int64:
            raise ValueError("staging arena must be fp32 K/V and int64 owner tags")
        rows = owner.shape[0]
    out = torch.empty(n, hq, d, dtype=torch.float32, device=dev)
    lse = torch.empty(n, hq, dtype=torch.float32, device=dev)
    if n == 0:
        return out, lse
    lib = _native.lib()
    qsl_a = np.ascontiguousarray(qsl, dtype=np.int32)
    seqs_a = np.ascontiguousarray(seqs, dtype=np.int32)
    qsl_p, seqs_p = qsl_a.ctypes.data, seqs_a.ctypes.data
    need = lib.oscar_slab_attention_workspace(qsl_p, seqs_p, len(seqs), int(k_new is not None), hq, hk, d)
    ws_bytes = max(0, min(int(need), int(workspace_bytes)))
    ws = torch.empty(max(ws_bytes, 16), dtype=torch.uint8, device=dev)
    dtype = _DTYPES[q.dtype]
    check(lib.oscar_slab_attention(
        q.data_ptr(), _ptr(k_new), _ptr(v_new), dtype, n, hq, hk, d,
        k8.data_ptr(), v8.data_ptr(), k8.shape[0], k8.shape[1], *k8.stride()[:3], *v8.stride()[:3],
        table.data_ptr(), table.shape[0], table.stride(0), qsl_p, seqs_p, len(seqs), float(scale),
        _ptr(sk), _ptr(sv), _ptr(owner), rows, out.data_ptr(), lse.data_ptr(), ws.data_ptr(), ws_bytes,
        _stream(dev)))
    return out, lse


def slab_attention_shard(q, kc, vc, table, qsl, history_lens, scale, stage=None, *,
                         workspace_bytes: int = DEFAULT_WORKSPACE_BYTES):
    """Partial attention of rotated queries over one shard of the paged
    history: request r's keys [0, history_lens[r]) through table row r, all of
    them visible to all of its queries, no current chunk.  Returns (out, lse)
    like ``slab_attention``; shards of one history are combined with
    ``merge_slab`` (the split-KV merge of slab_attention.py:458-475 across
    GPUs).  Decode-sized steps at head dim 256 only (the tensor-core decode
    kernel or the CUDA-core decode kernel); other layouts raise ValueError."""
    qsl = [int(x) for x in qsl]
    hist = [int(x) for x in history_lens]
    if (q.ndim != 3 or kc.ndim != 4 or q.shape[1] < 1 or kc.shape[2] < 1 or len(qsl) != len(hist) + 1
            or not qsl or qsl[0] != 0 or qsl[-1] != q.shape[0] or q.shape[1] % kc.shape[2]):
        raise ValueError("Invalid slab query layout")
    if any(a > b or h < 0 for a, b, h in zip(qsl, qsl[1:], hist)):
        raise ValueError("Sequence length must cover its query chunk")
    _validate_tensors(q, None, None, kc, vc, table, qsl, hist, stage)
    dev = _require_cuda(q, kc, vc, table, *(stage or ()))
    if q.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError(f"unsupported query dtype {q.dtype}")
    n, hq, d = q.shape
    hk = kc.shape[2]
    q = q.contiguous()
    table = table.to(device=dev, dtype=torch.int32).contiguous()
    k8, v8 = _byte_view(kc), _byte_view(vc)
    sk = sv = owner = None
    rows = 0
    if stage is not None:
        sk, sv, owner = stage
        if sk.dtype != torch.float32 or sv.dtype != torch.float32 or owner.dtype != torch.int64:
            raise ValueError("staging arena must be fp32 K/V and int64 owner tags")
        rows = owner.shape[0]
    out = torch.empty(n, hq, d, dtype=torch.float32, device=dev)
    lse = torch.empty(n, hq, dtype=torch.float32, device=dev)
    if n == 0:
        return out, lse
    lib = _native.lib()
    qsl_a = np.ascontiguousarray(qsl, dtype=np.int32)
    hist_a = np.ascontiguousarray(hist, dtype=np.int32)
    # the shard's plan is the one of a step with the history as prefix and the
    # queries as its chunk
    seqs_a = np.ascontiguousarray([h + b - a for h, a, b in zip(hist, qsl, qsl[1:])], dtype=np.int32)
    need = lib.oscar_slab_attention_workspace(qsl_a.ctypes.data, seqs_a.ctypes.data, len(hist), 1, hq, hk, d)
    ws_bytes = max(0, min(int(need), int(workspace_bytes)))
    ws = torch.empty(max(ws_bytes, 16), dtype=torch.uint8, device=dev)
    check(lib.oscar_slab_attention_shard(
        q.data_ptr(), _DTYPES[q.dtype], n, hq, hk, d,
        k8.data_ptr(), v8.data_ptr(), k8.shape[0], k8.shape[1], *k8.stride()[:3], *v8.stride()[:3],
        table.data_ptr(), table.shape[0], table.stride(0), qsl_a.ctypes.data, hist_a.ctypes.data, len(hist),
        float(scale), _ptr(sk), _ptr(sv), _ptr(owner), rows, out.data_ptr(), lse.data_ptr(), ws.data_ptr(), ws_bytes,
        _stream(dev)))
    return out, lse


def decode_step_scratch_bytes(n: int, hq: int, hk: int, d: int, workspace_bytes: int) -> int:
    """Scratch of decode_layer_step for up to n tokens: the rotated rows and
    the attention output, then `workspace_bytes` of attention workspace."""
    fixed = int(_native.lib().oscar_decode_layer_step_scratch(n, hq, hk, d, _native.DTYPE_BF16))
    if fixed < 0:
        raise ValueError("decode_layer_step: invalid geometry")
    return fixed + max(0, int(workspace_bytes))


def decode_layer_step(q, k, v, token_strides, n, hq, hk, d, rot_k, rot_v, rot_vt, k_clip_ratio, v_clip_ratio,
                      k_cache, v_cache, slot_mapping, qsl_dev, seqs_dev, table, qsl, seqs, sink_eff, recent_tokens,
                      scale, stage_k, stage_v, owner, out, scratch) -> None:
    """One decode-sized layer step in one native call (oscar_decode_layer_step):
    rotations, clip + INT2 store + staging write, rotated attention, output
    rotation into ``out``.  The backend's fast path: the caller has checked
    the layouts (heads contiguous per token, ``token_strides`` = the token
    row strides of q, k, v, out in elements; int64 slots, int32 device qsl /
    seqs and block table, host lists ``qsl`` / ``seqs``); the C side checks
    sizes and alignment and raises through ``check``."""
    lib = _native.lib()
    k8, v8 = k_cache.view(torch.uint8), v_cache.view(torch.uint8)
    qsl_a = np.asarray(qsl, dtype=np.int32)
    seqs_a = np.asarray(seqs, dtype=np.int32)
    kst, vst = k8.stride(), v8.stride()
    check(lib.oscar_decode_layer_step(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), _DTYPES[q.dtype], token_strides[0], token_strides[1],
        token_strides[2], n, hq, hk, d, rot_k.data_ptr(), rot_v.data_ptr(), rot_vt.data_ptr(), _clip_ok(k_clip_ratio),
        _clip_ok(v_clip_ratio), k8.data_ptr(), v8.data_ptr(), k8.shape[0], k8.shape[1], kst[0], kst[1], kst[2],
        vst[0], vst[1], vst[2], slot_mapping.data_ptr(), qsl_dev.data_ptr(), seqs_dev.data_ptr(), table.data_ptr(),
        table.shape[0], table.stride(0), qsl_a.ctypes.data, seqs_a.ctypes.data, len(seqs), int(sink_eff),
        int(recent_tokens), float(scale), stage_k.data_ptr(), stage_v.data_ptr(), owner.data_ptr(), owner.shape[0],
        out.data_ptr(), token_strides[3], scratch.data_ptr(), scratch.numel(), _stream(q.device)))


def merge_slab(output, lse, part, part_lse, start, ids) -> None:
    """In-place LSE merge of part into output[start:start+n] (or output[ids])."""
    dev = _require_cuda(output, lse, part, part_lse, ids)
    n, hq, d = part.shape
    if output.dtype != torch.float32 or lse.dtype != torch.float32 or not output.is_contiguous() or not lse.is_contiguous():
        raise ValueError("output/lse must be contiguous fp32")
    if part.dtype not in _DTYPES:
        raise ValueError(f"unsupported partial dtype {part.dtype}")
    part = part.contiguous()
    part_lse = part_lse.to(torch.float32).contiguous()
    ids_t = None if ids is None else ids.to(device=dev, dtype=torch.int32).contiguous()
    if output.shape[1:] != part.shape[1:] or lse.shape != output.shape[:2] or part_lse.shape != part.shape[:2]:
        raise ValueError("merge: output/lse/part geometry mismatch")
    check(_native.lib().oscar_merge_slab(output.data_ptr(), lse.data_ptr(), output.shape[0], part.data_ptr(),
                                         _DTYPES[part.dtype],
                                         part_lse.data_ptr(), n, hq, d, int(start), _ptr(ids_t), _stream(dev)))


# ---------------------------------------------------------------------------
# the 16-bit paged layer
_HALF = {torch.bfloat16: _native.DTYPE_BF16, torch.float16: _native.DTYPE_F16}


def _cuda_index(first: torch.Tensor, *others: torch.Tensor | None) -> int:
    """The one CUDA device of the tensors (as _require_cuda, for calls whose host time counts)."""
    index = first.get_device()
    for t in others:
        if t is not None and t.get_device() != index:
            _require_cuda(first, *others)
    if index < 0:
        _require_cuda(first)
    return index


# the library launches on the current device, which therefore has to be the tensors'
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def _rows16(t: torch.Tensor, stride: tuple) -> torch.Tensor:
    """[n, heads, D] with contiguous, 16-byte aligned head vectors (a copy of t where its layout has none)."""
    if stride[2] != 1 or (stride[0] | stride[1]) % 8 or t.data_ptr() % 16:
        return t.clone(memory_format=torch.contiguous_format)
    return t


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Do the memory ranges of two tensors meet?"""
    if a.numel() == 0 or b.numel() == 0:
        return False
    first, last = ([t.data_ptr() for t in (a, b)],
                   [t.data_ptr() + t.element_size() * sum((n - 1) * s for n, s in zip(t.shape, t.stride())) for t in (a, b)])
    return first[0] <= last[1] and first[1] <= last[0]


def _cache16(name: str, k_cache: torch.Tensor, v_cache: torch.Tensor, dtype, hk: int, d: int) -> tuple:
    """Strides of the two caches, [blocks, tokens, hk, d] of `dtype` with contiguous rows."""
    shape, ks, vs = k_cache.shape, k_cache.stride(), v_cache.stride()
    if len(shape) != 4 or shape != v_cache.shape or shape[2] != hk or shape[3] != d:
        raise ValueError(f"{name}: caches must be [blocks, tokens, {hk}, {d}] and alike")
    if k_cache.dtype != dtype or v_cache.dtype != dtype:
        raise ValueError(f"{name}: the caches must have the heads' type {dtype}, got {k_cache.dtype} and {v_cache.dtype}")
    if ks[3] != 1 or vs[3] != 1:
        raise ValueError(f"{name}: cache rows must be contiguous in the last dim")
    return ks, vs


def _host_ints(values) -> np.ndarray:
    if type(values) is np.ndarray and values.dtype == np.int32 and values.flags.c_contiguous:
        return values
    if isinstance(values, torch.Tensor):
        values = values.cpu().numpy()
    out = np.ascontiguousarray(values, dtype=np.int32)
    if isinstance(values, np.ndarray) and not np.array_equal(out, values):  # (numpy wraps and cuts without a word)
        raise ValueError("query starts and lengths must be whole numbers of 32 bits")
    return out


def _table32(name: str, table: torch.Tensor) -> tuple:
    """The block table as int32 rows apart from one another, and their stride."""
    if table.ndim != 2:
        raise ValueError(f"{name}: the block table must be [requests, pages]")
    if table.dtype != torch.int32:
        table = table.to(torch.int32)
    (rows, cols), (stride, step) = table.shape, table.stride()
    if rows < 2:
        stride = cols  # one row has no stride of its own
    if (step != 1 and cols > 1) or stride < cols:  # (an expanded row among them)
        return table.clone(memory_format=torch.contiguous_format), cols
    return table, stride


def _long(t: torch.Tensor) -> torch.Tensor:
    return t if t.dtype == torch.int64 and t.is_contiguous() else t.to(torch.int64).contiguous()


def qk_norm_rope(q, k, v, q_weight, k_weight, eps, cos_sin, positions, *, weight_offset: float = 0.0,
                 interleaved: bool = False, k_cache=None, v_cache=None, slot_mapping=None, out_q=None, out_k=None):
    """RMS norm of every query and key head, position rotation and (with
    caches) the write of the step's keys and values to a 16-bit paged cache,
    in one pass.

    q [n, Hq, D], k / v [n, Hk, D] (bf16 or fp16; views of a fused projection
    are fine); weights [D] and ``cos_sin`` [max_positions, rot] (cosines, then
    sines) in fp32 or the heads' type (what is not 16-byte aligned is copied
    first); ``positions`` [n].  ``weight_offset``
    1 is the zero-centred weight (1 + w).  Pairs (i, i + rot/2) rotate, or
    neighbours (2i, 2i + 1) with ``interleaved``.  Without caches the keys come
    back (v is not needed); with them k and v go to ``slot_mapping`` (slots
    < 0 are skipped) and the keys come back only into a given ``out_k``.
    Returns (out_q, out_k)."""
    q_shape, k_shape, dtype = q.shape, k.shape, q.dtype
    if len(q_shape) != 3 or len(k_shape) != 3 or k_shape[0] != q_shape[0] or k_shape[2] != q_shape[2] or k.dtype != dtype:
        raise ValueError("qk_norm_rope: q [n, Hq, D] and k [n, Hk, D] of one type are needed")
    code = _HALF.get(dtype)
    if code is None:
        raise ValueError(f"qk_norm_rope: unsupported type {dtype}")
    n, hq, d = q_shape
    hk = k_shape[1]
    write = k_cache is not None
    if write != (v_cache is not None) or write != (slot_mapping is not None) or (write and v is None):
        raise ValueError("qk_norm_rope: v, caches and slot_mapping come together")
    index = _cuda_index(q, k, v, q_weight, k_weight, cos_sin, positions, k_cache, v_cache, slot_mapping, out_q, out_k)
    if index != _current_device():
        with torch.cuda.device(index):
            return qk_norm_rope(q, k, v, q_weight, k_weight, eps, cos_sin, positions, weight_offset=weight_offset,
                                interleaved=interleaved, k_cache=k_cache, v_cache=v_cache, slot_mapping=slot_mapping,
                                out_q=out_q, out_k=out_k)
    w_dtype, cs_dtype, cs_shape = q_weight.dtype, cos_sin.dtype, cos_sin.shape
    if q_weight.shape != (d,) or k_weight.shape != (d,) or w_dtype != k_weight.dtype:
        raise ValueError(f"qk_norm_rope: the weights must be two [{d}] tensors of one type")
    if len(cs_shape) != 2 or positions.shape != (n,):
        raise ValueError("qk_norm_rope: cos_sin [max_positions, rot] and positions [n] are needed")
    if (w_dtype != torch.float32 and w_dtype != dtype) or (cs_dtype != torch.float32 and cs_dtype != dtype):
        raise ValueError("qk_norm_rope: weights and cos_sin must be fp32 or of the heads' type")
    qt, kt, ct = q.stride(), k.stride(), cos_sin.stride()
    q, k = _rows16(q, qt), _rows16(k, kt)
    qt, kt = q.stride(), k.stride()
    q_weight, k_weight, positions = q_weight.contiguous(), k_weight.contiguous(), _long(positions)
    wq_p, wk_p, cs_p = q_weight.data_ptr(), k_weight.data_ptr(), cos_sin.data_ptr()
    if (wq_p | wk_p) % 16:
        q_weight, k_weight = q_weight.clone(), k_weight.clone()
        wq_p, wk_p = q_weight.data_ptr(), k_weight.data_ptr()
    if ct[1] != 1 or ct[0] % 8 or ct[0] < cs_shape[1] or cs_p % 16:
        cos_sin = cos_sin.clone(memory_format=torch.contiguous_format)
        ct, cs_p = cos_sin.stride(), cos_sin.data_ptr()
    if out_q is None:
        out_q = q.new_empty(q_shape)  # (a third less host time than torch.empty)
    elif out_q.shape != q_shape or out_q.dtype != dtype or out_q.stride(2) != 1:
        raise ValueError(f"qk_norm_rope: out_q must be {list(q_shape)} rows of {dtype}")
    if out_k is None:
        if not write:
            out_k = q.new_empty(k_shape)
    elif out_k.shape != k_shape or out_k.dtype != dtype or out_k.stride(2) != 1:
        raise ValueError(f"qk_norm_rope: out_k must be {list(k_shape)} rows of {dtype}")
    nb = bs = 1
    ks = vs = vt = (0, 0, 0)
    kc_p = vc_p = v_p = slots_p = ok_p = None
    if write:
        if v.shape != k_shape or v.dtype != dtype:
            raise ValueError("qk_norm_rope: v must match k")
        v = _rows16(v, v.stride())
        vt = v.stride()
        ks, vs = _cache16("qk_norm_rope", k_cache, v_cache, dtype, hk, d)
        nb, bs = k_cache.shape[:2]
        slot_mapping = _long(slot_mapping)
        if slot_mapping.numel() < n:
            raise ValueError("slot_mapping shorter than the token count")
        kc_p, vc_p, v_p, slots_p = k_cache.data_ptr(), v_cache.data_ptr(), v.data_ptr(), slot_mapping.data_ptr()
    oq, ok = out_q.stride(), (0, 0)
    if out_k is not None:
        ok, ok_p = out_k.stride(), out_k.data_ptr()
    check(_native.lib().oscar_qk_norm_rope(
        q.data_ptr(), qt[0], qt[1], k.data_ptr(), kt[0], kt[1], v_p, vt[0], vt[1], code, n, hq, hk, d,
        wq_p, wk_p, _DTYPES[w_dtype], eps, weight_offset, cs_p,
        _DTYPES[cs_dtype], ct[0], cs_shape[0], cs_shape[1], 1 if interleaved else 0, positions.data_ptr(),
        out_q.data_ptr(), oq[0], oq[1], ok_p, ok[0], ok[1], kc_p, vc_p, nb, bs, ks[0], ks[1], ks[2], vs[0], vs[1], vs[2],
        slots_p, _raw_stream(index)))
    return out_q, out_k


def paged_attention(q, k_cache, v_cache, table, qsl, seqs, scale, *, weights=None, observe: int | None = None, out=None):
    """Attention of each request's new tokens (one or thousands) over a paged
    16-bit cache that already holds them: query i of request r sees keys
    [0, seqs[r] - q_len + i].  Returns (out [n, Hq, D] in q's type, lse [n, Hq]
    fp32 natural log); a row that sees no key is 0 with lse -inf.

    q [n, Hq, D]; caches [blocks, tokens, Hk, D] of q's type (strided views
    are fine); ``table`` [requests, pages]; ``qsl`` / ``seqs`` are host lists
    or int32 arrays as in ``slab_attention``; ``out`` may be q.

    ``weights`` [blocks, Hk, tokens] fp32 accumulates the attention weight of
    every cached key, summed over the heads of its group and the last
    ``observe`` tokens of each request (None: all): keys older than the chunk
    add it to what they have, the chunk's own keys start from it."""
    q_shape, c_shape, dtype = q.shape, k_cache.shape, q.dtype
    if len(q_shape) != 3 or len(c_shape) != 4 or c_shape[2] < 1 or q_shape[1] % c_shape[2]:
        raise ValueError("paged_attention: q [n, Hq, D] with Hq a multiple of the caches' heads is needed")
    code = _HALF.get(dtype)
    if code is None:
        raise ValueError(f"paged_attention: unsupported query type {dtype}")
    n, hq, d = q_shape
    nb, bs, hk = c_shape[:3]
    index = _cuda_index(q, k_cache, v_cache, table, weights, out)
    if index != _current_device():
        with torch.cuda.device(index):
            return paged_attention(q, k_cache, v_cache, table, qsl, seqs, scale, weights=weights, observe=observe, out=out)
    ks, vs = _cache16("paged_attention", k_cache, v_cache, dtype, hk, d)
    qsl_a, seqs_a = _host_ints(qsl), _host_ints(seqs)
    if qsl_a.ndim != 1 or seqs_a.ndim != 1 or qsl_a.size != seqs_a.size + 1 or qsl_a[0] != 0 or qsl_a[-1] != n:
        raise ValueError("paged_attention: invalid query layout")
    table, ts = _table32("paged_attention", table)
    if weights is not None and (weights.shape != (nb, hk, bs) or weights.dtype != torch.float32
                                or not weights.is_contiguous()):
        raise ValueError(f"paged_attention: weights must be contiguous fp32 [{nb}, {hk}, {bs}]")
    if observe is not None and (weights is None or int(observe) < 1):
        raise ValueError("paged_attention: observe needs weights and at least one token")
    q = _rows16(q, q.stride())
    if out is None:
        out = q.new_empty(q_shape)
    elif out.shape != q_shape or out.dtype != dtype or not out.is_contiguous() or out.data_ptr() % 32:
        raise ValueError(f"paged_attention: out must be contiguous, 32-byte aligned {list(q_shape)} of {dtype}")
    elif _overlap(q, out) and (weights is not None or q.data_ptr() != out.data_ptr() or q.stride() != out.stride()):
        q = q.clone()  # the keys' weights read the queries again; other overlaps are other rows'
    lse = q.new_empty((n, hq), dtype=torch.float32)
    lib = _native.lib()
    qsl_p, seqs_p, b = qsl_a.ctypes.data, seqs_a.ctypes.data, seqs_a.size
    need = lib.oscar_paged_attention_workspace(qsl_p, seqs_p, b, hq, hk, d, 0 if weights is None else 1)
    if need < 0:
        check(_native.ERR_INVALID)
    ws = q.new_empty(max(need, 16), dtype=torch.uint8)
    qs, (rows, cols) = q.stride(), table.shape
    check(lib.oscar_paged_attention(
        q.data_ptr(), qs[0], qs[1], code, n, hq, hk, d, k_cache.data_ptr(), v_cache.data_ptr(), nb, bs, ks[0], ks[1],
        ks[2], vs[0], vs[1], vs[2], table.data_ptr(), rows, cols, ts, qsl_p, seqs_p, b, scale,
        None if weights is None else weights.data_ptr(), 0x7FFFFFFF if observe is None else min(int(observe), 0x7FFFFFFF),
        out.data_ptr(), lse.data_ptr(), ws.data_ptr(), need, _raw_stream(index)))
    return out, lse


def evict_cache(k_cache, v_cache, weights, table, seqs, keep: int, *, sink: int = 0, recent: int = 0, dst_table=None):
    """Cuts every request with more than ``keep`` cached tokens down to
    ``keep``, per kv head: the first ``sink``, the last ``recent`` and the
    heaviest of the others by ``weights`` [blocks, Hk, tokens] stay in order
    (ties: the lower position).  Their K, V and weight slots move to the front
    of the request's pages, or to the pages of ``dst_table`` (for pages shared
    with other requests, which must not be overwritten; ``table`` itself: the
    request's own).  ``seqs``: host list.
    Returns the kept positions [requests, Hk, min(keep, max(seqs))] int32 (-1
    past a request's list); the new lengths are min(seqs, keep)."""
    shape, dtype = k_cache.shape, k_cache.dtype
    if len(shape) != 4:
        raise ValueError("evict_cache: caches must be [blocks, tokens, heads, D]")
    nb, bs, hk, d = shape
    if dtype not in _HALF:
        raise ValueError(f"evict_cache: unsupported cache type {dtype}")
    index = _cuda_index(k_cache, v_cache, weights, table, dst_table)
    if index != _current_device():
        with torch.cuda.device(index):
            return evict_cache(k_cache, v_cache, weights, table, seqs, keep, sink=sink, recent=recent, dst_table=dst_table)
    ks, vs = _cache16("evict_cache", k_cache, v_cache, dtype, hk, d)
    if weights.shape != (nb, hk, bs) or weights.dtype != torch.float32 or not weights.is_contiguous():
        raise ValueError(f"evict_cache: weights must be contiguous fp32 [{nb}, {hk}, {bs}]")
    seqs_a = _host_ints(seqs)
    if seqs_a.ndim != 1:
        raise ValueError("evict_cache: seqs must be a list of lengths")
    source, (table, ts) = table, _table32("evict_cache", table)
    rows, cols = table.shape
    dst_p, dst_rows, dst_cols, dst_stride = None, 0, 0, 0
    if dst_table is not None and (dst_table.data_ptr() != source.data_ptr() or dst_table.stride() != source.stride()):
        dst, dst_stride = _table32("evict_cache", dst_table)
        dst_p, (dst_rows, dst_cols) = dst.data_ptr(), dst.shape
    keep, sink, recent = int(keep), int(sink), int(recent)
    if keep < 1 or sink < 0 or recent < 0 or sink + recent > keep:
        raise ValueError("evict_cache: keep must be at least 1 and hold the sink and recent tokens")
    longest = int(seqs_a.max(initial=0))
    if keep > longest:  # nothing goes, and the numbers may pass 32 bits
        keep, sink, recent = max(longest, 1), 0, 0
    places = min(keep, longest)
    kept = k_cache.new_empty((seqs_a.size, hk, places), dtype=torch.int32)
    check(_native.lib().oscar_evict_cache(
        k_cache.data_ptr(), v_cache.data_ptr(), d, nb, bs, hk, ks[0], ks[1], ks[2], vs[0], vs[1], vs[2],
        weights.data_ptr(), table.data_ptr(), rows, cols, ts, dst_p, dst_rows, dst_cols, dst_stride,
        seqs_a.ctypes.data, seqs_a.size, keep, sink, recent, kept.data_ptr(), places, _raw_stream(index)))
    return kept


_PATHS = {"auto": 0, "tile": 1, "decode": 2, "tensor": 3}


def rotate_rows(x: torch.Tensor, rot: torch.Tensor, *, transpose: bool = False, out: torch.Tensor | None = None,
                out_f32: torch.Tensor | None = None, out_dtype: torch.dtype | None = None):
    """y = x @ R (or x @ R^T) over the last dim of x in fp32 (the per-layer
    rotations of backend.py:238-246).  x: [..., D] (fp32/bf16/fp16, rows with a
    uniform stride); writes `out` (given, or new of `out_dtype`) and/or
    `out_f32`, both [..., D] views with uniform row strides.  Returns (out, out_f32)."""
    d = x.shape[-1]
    if rot.shape != (d, d) or rot.dtype != torch.float32:
        raise ValueError(f"rotation must be fp32 [{d}, {d}], got {tuple(rot.shape)} {rot.dtype}")
    rot = rot.contiguous()
    x2 = x.reshape(-1, d)
    if x2.stride(-1) != 1 or (x2.shape[0] > 1 and x2.stride(0) % 8) or x2.data_ptr() % 16:
        x2 = x2.clone(memory_format=torch.contiguous_format)
    rows = x2.shape[0]
    if out is None and out_f32 is None:
        out = torch.empty(x.shape, dtype=out_dtype or x.dtype, device=x.device)
    o2 = None if out is None else out.view(-1, d)
    f2 = None if out_f32 is None else out_f32.view(-1, d)
    for t in (x2, o2, f2):
        if t is not None and rows > 1 and t.stride(-1) != 1:
            raise ValueError("rotate_rows: rows must be contiguous in the last dim")
    dev = _require_cuda(x, rot)
    check(_native.lib().oscar_rotate_rows(
        _ptr(x2), _DTYPES[x2.dtype], rows, x2.stride(0), d, _ptr(rot), 1 if transpose else 0,
        _ptr(o2), _DTYPES[o2.dtype] if o2 is not None else 0, o2.stride(0) if o2 is not None else 0,
        _ptr(f2), f2.stride(0) if f2 is not None else 0, _stream(dev)))
    return out, out_f32


def rotate_rows_many(jobs) -> None:
    """Several rotate_rows calls in one launch.  ``jobs``: up to four
    ``(x, rot, out, out_f32)`` tuples (x @ R, no transpose) whose x share one
    dtype and D and whose ``out`` tensors share one dtype; each output is
    preallocated ([..., D] rows with uniform strides) or None."""
    if not jobs:
        return
    if len(jobs) > 4:
        raise ValueError("rotate_rows_many: at most 4 jobs per launch")
    dev = _require_cuda(*[t for job in jobs for t in job])
    d = jobs[0][0].shape[-1]
    x_dt = jobs[0][0].dtype
    out_dt = next((o.dtype for _, _, o, _ in jobs if o is not None), torch.float32)
    segs = (_native.RotateSeg * len(jobs))()
    keep = []
    for i, (x, rot, out, out_f32) in enumerate(jobs):
        if x.shape[-1] != d or x.dtype != x_dt or (out is not None and out.dtype != out_dt):
            raise ValueError("rotate_rows_many: jobs must share x dtype, D and out dtype")
        if rot.shape != (d, d) or rot.dtype != torch.float32:
            raise ValueError(f"rotation must be fp32 [{d}, {d}], got {tuple(rot.shape)} {rot.dtype}")
        rot = rot.contiguous()
        keep.append(rot)
        x2 = x.reshape(-1, d)
        if x2.stride(-1) != 1 or (x2.shape[0] > 1 and x2.stride(0) % 8) or x2.data_ptr() % 16:
            x2 = x2.clone(memory_format=torch.contiguous_format)
        o2 = None if out is None else out.view(-1, d)
        f2 = None if out_f32 is None else out_f32.view(-1, d)
        for t in (o2, f2):
            if t is not None and t.shape[0] > 1 and t.stride(-1) != 1:
                raise ValueError("rotate_rows_many: rows must be contiguous in the last dim")
        keep.append(x2)
        segs[i] = _native.RotateSeg(_ptr(x2), x2.shape[0], x2.stride(0), _ptr(rot), 0,
                                    _ptr(o2), o2.stride(0) if o2 is not None else 0,
                                    _ptr(f2), f2.stride(0) if f2 is not None else 0)
    check(_native.lib().oscar_rotate_rows_batch(segs, len(jobs), _DTYPES[x_dt], d, _DTYPES[out_dt], _stream(dev)))


def set_attention_path(path: str) -> None:
    """Kernel family for slab_attention: "auto" (tensor-core decode kernel,
    else the mma.sync decode kernel, else the tile kernel, whichever is
    eligible first), "tensor" or "decode" (that decode kernel where eligible,
    else the tile kernel) or "tile" (tile kernel only).  All compute the same
    function."""
    check(_native.lib().oscar_set_attention_path(_PATHS[path]))


_ROT_PATHS = {"auto": 0, "fma": 1, "tensor": 2, "fma_big": 3}


def set_rotation_path(path: str) -> None:
    """Rotation kernel for rotate_rows / rotate_rows_many and the layer step:
    "auto" (per tensor, by its own size: tcgen05 kind::tf32 with split
    precision for fp32 tensors of at least 2560 rows -- the output rotation --,
    register-tiled fp32 FMAs for 16-bit ones of at least 6144 rows -- the
    k / v / q rotations of long chunks; 64-row tiles below 16384 rows, 128-row
    tiles from there --, 16-row FMA tiles for the rest), "fma" (16-row FMA
    tiles), "tensor" or "fma_big" (register-tiled FMAs, D 128 or 256).  All
    compute x @ R to within a few fp32 ulps."""
    check(_native.lib().oscar_set_rotation_path(_ROT_PATHS[path]))


def set_wait_limit(tries: int = -1) -> None:
    """Limit of one bounded wait of the paged_attention kernels in tries of up
    to a millisecond (-1: the default).  A wait that runs out latches device
    error 16 and ends the launch early (debug)."""
    check(_native.lib().oscar_set_wait_limit(int(tries)))


def device_error(device=None) -> int:
    """Synchronise and return/clear the kernels' bounds-violation flag (debug)."""
    dev = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    return int(_native.lib().oscar_device_error(_stream(dev)))
