"""The attention step of a layer whose cache holds plain bf16 / fp16 keys and
values -- the MTP draft layers beside the INT2 ones, in the pool of
:mod:`oscar_b200.mtp_shadow` or any paged pool of that form.

:class:`DraftLayer` runs the whole step on the device: norm of the query and
key heads with the position rotation and the cache write
(``kernels.qk_norm_rope``), attention over the paged cache with the keys'
accumulated weights (``kernels.paged_attention``), and, on request, eviction of
the lightest keys (``kernels.evict_cache``).  A draft layer's evicted key can
cost an accepted draft token, never a wrong output token, so its pool may be
bounded where the target's may not.

``python -m oscar_b200.draft`` runs a prompt, draft steps and an eviction on
random data and prints the time of each.
"""
from __future__ import annotations

import torch

from . import kernels


class DraftLayer:
    """One 16-bit paged attention layer.

    ``kv_cache``: the pair (K, V) of [blocks, tokens, Hk, D] caches (views of one
    pool are fine).  ``q_weight`` / ``k_weight`` [D], ``cos_sin`` [positions, rot]:
    as ``kernels.qk_norm_rope``.  ``keep``: cached tokens per request that
    :meth:`evict` leaves (None: weights are not kept); ``sink`` / ``recent``: of
    these, the first and last ones that always stay; ``observe``: the last
    tokens of a step that weigh the keys (None: all).

    Memory beside the caches: with ``keep`` 4 bytes per cache slot and head for
    the weights, and during a step the queries' copy, the output and a
    workspace of at most 320 MiB and 8 bytes per token and query head."""

    def __init__(self, num_heads: int, kv_cache, q_weight, k_weight, cos_sin, *, eps: float = 1e-6,
                 weight_offset: float = 0.0, interleaved: bool = False, scale: float | None = None,
                 keep: int | None = None, sink: int = 64, recent: int = 256, observe: int | None = None):
        self.k_cache, self.v_cache = kv_cache[0], kv_cache[1]
        blocks, tokens, hk, d = self.k_cache.shape
        if num_heads % hk:
            raise ValueError("DraftLayer: Hq must be a multiple of the caches' heads")
        if keep is not None and not 0 <= sink + recent <= keep:
            raise ValueError("DraftLayer: keep must hold the sink and recent tokens")
        self.num_heads, self.scale = num_heads, d**-0.5 if scale is None else float(scale)
        self.norm = (q_weight, k_weight, float(eps), cos_sin)
        self.weight_offset, self.interleaved = float(weight_offset), bool(interleaved)
        self.keep, self.sink, self.recent, self.observe = keep, sink, recent, observe
        self.weights = None
        if keep is not None:
            self.weights = torch.zeros(blocks, hk, tokens, dtype=torch.float32, device=self.k_cache.device)

    def forward(self, q, k, v, positions, slot_mapping, table, qsl, seqs, out=None):
        """One step: q [n, Hq, D], k / v [n, Hk, D] as projected, ``positions`` [n]
        of the tokens in their requests, ``slot_mapping`` [n] their cache slots,
        ``qsl`` / ``seqs`` host lists (``seqs``: cached tokens, the step's among
        them -- after an eviction fewer than positions).  Returns (out [n, Hq, D],
        lse [n, Hq])."""
        q_weight, k_weight, eps, cos_sin = self.norm
        q, _ = kernels.qk_norm_rope(q, k, v, q_weight, k_weight, eps, cos_sin, positions, weight_offset=self.weight_offset,
                                    interleaved=self.interleaved, k_cache=self.k_cache, v_cache=self.v_cache,
                                    slot_mapping=slot_mapping)
        return kernels.paged_attention(q, self.k_cache, self.v_cache, table, qsl, seqs, self.scale, weights=self.weights,
                                       observe=self.observe if self.weights is not None else None, out=out)

    def evict(self, table, seqs, dst_table=None):
        """Cuts every request with more than ``keep`` cached tokens down to them,
        in its own pages or into ``dst_table``'s (which then replace them).
        Returns (cached lengths, kept positions)."""
        if self.keep is None:
            raise ValueError("DraftLayer: the layer keeps no weights (keep is None)")
        kept = kernels.evict_cache(self.k_cache, self.v_cache, self.weights, table, seqs, self.keep, sink=self.sink,
                                   recent=self.recent, dst_table=dst_table)
        return [min(int(s), self.keep) for s in seqs], kept


def slots_of(table: torch.Tensor, lens, seqs, tokens: int) -> torch.Tensor:
    """Cache slots of the last ``lens[r]`` of ``seqs[r]`` cached tokens of each
    request, pages of ``tokens`` tokens (the engine's slot_mapping)."""
    parts = []
    for r, (m, seq) in enumerate(zip(lens, seqs)):
        p = torch.arange(seq - m, seq, device=table.device)
        parts.append(table[r].long()[p // tokens] * tokens + p % tokens)
    return torch.cat(parts) if parts else torch.zeros(0, dtype=torch.int64, device=table.device)


def main() -> None:
    import argparse

    ap = argparse.ArgumentParser(description="A draft layer's prompt, steps and eviction on random data")
    ap.add_argument("--requests", type=int, default=8)
    ap.add_argument("--prompt", type=int, default=2048)
    ap.add_argument("--steps", type=int, default=8)
    ap.add_argument("--draft-tokens", type=int, default=4)
    ap.add_argument("--keep", type=int, default=1024)
    args = ap.parse_args()
    dev = torch.device("cuda", torch.cuda.current_device())
    hq, hk, d, page, rot, n = 24, 4, 256, 128, 64, args.requests
    gen = torch.Generator(device=dev).manual_seed(0)
    width = -(-(args.prompt + 2 * args.steps * args.draft_tokens) // page)
    pool = torch.zeros(2, n * width, page, hk, d, dtype=torch.bfloat16, device=dev)
    table = torch.randperm(n * width, generator=gen, device=dev).to(torch.int32).view(n, width)
    angle = torch.arange(65536, device=dev)[:, None] / 1e6 ** (torch.arange(0, rot, 2, device=dev) / rot)
    weight = torch.zeros(d, device=dev)
    layer = DraftLayer(hq, pool, weight, weight, torch.cat([angle.cos(), angle.sin()], 1), weight_offset=1.0, keep=args.keep)

    def step(m, cached, position):
        qkv = torch.randn(n * m, hq + 2 * hk, d, generator=gen, device=dev).to(torch.bfloat16)
        cached = [c + m for c in cached]
        positions = (torch.arange(m, device=dev) + position).repeat(n)
        slots = slots_of(table, [m] * n, cached, page)
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        layer.forward(qkv[:, :hq], qkv[:, hq:hq + hk], qkv[:, hq + hk:], positions, slots, table,
                      [m * i for i in range(n + 1)], cached)
        b.record()
        b.synchronize()
        return cached, position + m, a.elapsed_time(b) * 1e3

    cached, position, us = step(args.prompt, [0] * n, 0)
    print(f"prompt: {n} x {args.prompt} tokens, {us:.0f} us (first call)")
    for phase in ("full cache", "after eviction"):
        for _ in range(args.steps):
            cached, position, us = step(args.draft_tokens, cached, position)
        print(f"{phase}: {cached[0]} cached tokens per request, {us:.0f} us per step of {n} x {args.draft_tokens} tokens")
        if phase == "full cache":
            cached, _ = layer.evict(table, cached)
    if kernels.device_error(dev):
        raise RuntimeError("a kernel flagged an index out of range")


if __name__ == "__main__":
    main()
