"""Cases, inputs and plain forms of the operators of a 16-bit paged attention layer.

The operators (``oscar_b200.kernels``):
  * ``qk_norm_rope``    norm of the query and key heads, position rotation and cache write
  * ``paged_attention`` attention of new tokens over a paged 16-bit cache, with the keys'
                        accumulated attention weights on request
  * ``evict_cache``     keeps each head's heaviest keys and moves them together

``own`` false: elementary torch operations in 32 bits, rounded once; true: the
framework's kernels.  ``exact`` is the definition in 64 bits, written apart.
"""
import math
import random

import numpy as np
import torch

own = False

EPS = 1e-6
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


def _lognormal(n, seed, lo=1024, hi=32768):
    r = random.Random(seed)
    return [int(min(max(math.exp(r.gauss(math.log(4096), 1.0)), lo), hi)) for _ in range(n)]


def _text(values):
    return ",".join(str(v) for v in values)


def _ints(text):
    return [int(v) for v in text.split(",")]


def listed():
    layer = dict(hq=24, hk=4, d=256, page=128, dtype="bf16")
    return [
        # one draft step of 8 requests with 4 tokens each: latency counts
        dict(name="rope_step", op="rope", tokens=32, rot=64, interleaved=False, offset=1.0, write=True, **layer),
        # a long prompt chunk of the same layer
        dict(name="rope_chunk", op="rope", tokens=15360, rot=64, interleaved=False, offset=1.0, write=True, **layer),
        # fp16, whole-head rotation of neighbouring dims, an odd token count; keys handed on (the INT2 path stores them)
        dict(name="rope_odd", op="rope", tokens=1237, rot=128, interleaved=True, offset=0.0, write=False, hq=16, hk=2, d=128,
             page=16, dtype="f16"),
        # one request, one token: the smallest attention call
        dict(name="attn_one", op="attn", seqs="8192", lens="1", observe=-1, **layer),
        # 8 long requests, 4 draft tokens each
        dict(name="attn_mtp", op="attn", seqs=_text([24580] * 8), lens=_text([4] * 8), observe=-1, **layer),
        # 64 requests of mixed lengths, 1 to 4 tokens each
        dict(name="attn_mixed", op="attn", seqs=_text(_lognormal(64, 5)), lens=_text([1 + (i * 7) % 4 for i in range(64)]),
             observe=-1, **layer),
        # a long chunk on cached history
        dict(name="attn_chunk", op="attn", seqs="17448", lens="8192", observe=-1, **layer),
        # fp16, D 128, small pages, ragged chunks beside a decode request and one whose chunk is its whole sequence
        dict(name="attn_odd", op="attn", seqs="5003,1777,2050,333", lens="709,33,1,333", observe=-1, hq=24, hk=4, d=128, page=48,
             dtype="f16"),
        # decode steps that also accumulate every key's attention weight
        dict(name="weigh_mtp", op="attn", seqs=_text([24580] * 8), lens=_text([4] * 8), observe=0, **layer),
        # a prompt chunk whose last 64 tokens weigh the keys
        dict(name="weigh_chunk", op="attn", seqs="11304", lens="2048", observe=64, **layer),
        # one request cut down to 4096 keys per head
        dict(name="evict_one", op="evict", seqs="9256", keep=4096, sink=64, recent=256, **layer),
        # 8 long requests cut to half
        dict(name="evict_batch", op="evict", seqs=_text([24580] * 8), keep=12288, sink=64, recent=256, **layer),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """Sizes spread over the listed ranges (over their logarithm), odd ones among them."""
    layer = dict(rng.choice([dict(hq=24, hk=4, d=256, dtype="bf16"), dict(hq=6, hk=1, d=256, dtype="bf16"),
                             dict(hq=24, hk=4, d=128, dtype="f16"), dict(hq=16, hk=2, d=128, dtype="bf16"),
                             dict(hq=8, hk=8, d=64, dtype="f16"), dict(hq=10, hk=2, d=256, dtype="f16")]))
    layer["page"] = rng.choice([16, 32, 48, 64, 128, 784])
    op = rng.choice(["rope", "decode", "decode", "chunk", "chunk", "evict"])
    if op == "rope":
        d = layer["d"]
        return dict(op="rope", tokens=_spread(rng, 1, 15360), rot=rng.choice([d // 4, d // 2, d]),
                    interleaved=rng.random() < 0.5, offset=rng.choice([0.0, 1.0]), write=rng.random() < 0.5, **layer)
    if op == "evict":
        seqs = [_spread(rng, 700, 24580) for _ in range(_spread(rng, 1, 8))]
        keep = _spread(rng, 400, 12288)
        return dict(op="evict", seqs=_text(seqs), keep=keep, sink=rng.choice([0, 4, 64]), recent=rng.choice([0, 33, 256]), **layer)
    observe = rng.choice([-1, -1, 0, 32, 64])
    if op == "decode":
        n = _spread(rng, 1, 64)
        lens = [rng.randint(1, 4) for _ in range(n)]
        top = min(32768, 8 * 24580 * 2 // n)
        seqs = [max(q, _spread(rng, 16, top)) for q in lens]
    else:
        n = rng.choice([1, 1, 2, 3])
        lens = [_spread(rng, 5, 8192 // n) for _ in range(n)]
        seqs = [q + rng.choice([0, _spread(rng, 1, 9256)]) for q in lens]
    return dict(op="attn", seqs=_text(seqs), lens=_text(lens), observe=observe, **layer)


# ---------------------------------------------------------------------------
def _tables(gen, seqs, page, spare):
    """Block tables of requests whose pages lie in random order in one pool of `spare` further pages."""
    need = [-(-s // page) for s in seqs]
    blocks = sum(need) + spare
    perm = torch.randperm(blocks, generator=gen, device="cuda").to(torch.int32)
    table = torch.zeros(len(seqs), max(need), dtype=torch.int32, device="cuda")
    at = 0
    for r, n in enumerate(need):
        table[r, :n] = perm[at:at + n]
        at += n
    return table, perm[at:], blocks


def _normal(gen, shape, dtype):
    return torch.empty(shape, dtype=dtype, device="cuda").normal_(generator=gen)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    hq, hk, d, page = case["hq"], case["hk"], case["d"], case["page"]
    if case["op"] == "rope":
        n, rot = case["tokens"], case["rot"]
        # q, k, v are views of one fused projection, as a model layer makes them
        qkv = _normal(gen, (n, hq + 2 * hk, d), dt)
        positions = torch.randint(0, 32768, (n,), generator=gen, device="cuda")
        inv = 1e6 ** (-torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot)
        angle = torch.arange(32768, device="cuda", dtype=torch.float64)[:, None] * inv
        blocks = -(-n // page) + 3
        slots = torch.randperm(blocks * page, generator=gen, device="cuda")[:n].contiguous()
        return dict(op="rope", q=qkv[:, :hq], k=qkv[:, hq:hq + hk], v=qkv[:, hq + hk:],
                    wq=_normal(gen, (d,), torch.float32).mul_(0.1).add_(1.0 - case["offset"]).to(dt),
                    wk=_normal(gen, (d,), torch.float32).mul_(0.1).add_(1.0 - case["offset"]).to(dt),
                    cos_sin=torch.cat([angle.cos(), angle.sin()], dim=1).float(), positions=positions, slots=slots,
                    k_cache=torch.zeros(blocks, page, hk, d, dtype=dt, device="cuda"),
                    v_cache=torch.zeros(blocks, page, hk, d, dtype=dt, device="cuda"), rot=rot,
                    interleaved=case["interleaved"], offset=case["offset"], write=case["write"])
    seqs = _ints(case["seqs"])
    if case["op"] == "evict":
        keep = case["keep"]
        fresh = [-(-min(keep, s) // page) for s in seqs]
        table, rest, blocks = _tables(gen, seqs, page, sum(fresh) + 2)
        dst = torch.zeros(len(seqs), max(fresh), dtype=torch.int32, device="cuda")
        at = 0
        for r, n in enumerate(fresh):
            dst[r, :n] = rest[at:at + n]
            at += n
        # accumulated weights are heavy-tailed, and keys that nothing attended tie at zero
        w = torch.exp(2.0 * _normal(gen, (blocks, hk, page), torch.float32) - 3.0)
        w = torch.where(torch.rand(w.shape, generator=gen, device="cuda") < 0.02, torch.zeros_like(w), w)
        return dict(op="evict", k_cache=_normal(gen, (blocks, page, hk, d), dt), v_cache=_normal(gen, (blocks, page, hk, d), dt),
                    weights=w, table=table, dst=dst, seqs=np.asarray(seqs, np.int32), seqs_dev=torch.tensor(seqs, device="cuda"),
                    keep=keep, sink=case["sink"], recent=case["recent"])
    lens = _ints(case["lens"])
    table, _, blocks = _tables(gen, seqs, page, 2)
    qsl = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    k_cache, v_cache = _normal(gen, (blocks, page, hk, d), dt), _normal(gen, (blocks, page, hk, d), dt)
    weights = None
    if case["observe"] >= 0:
        weights = torch.rand(blocks, hk, page, generator=gen, device="cuda") * 1e-2
    return dict(op="attn", q=_normal(gen, (int(qsl[-1]), hq, d), dt), k_cache=k_cache, v_cache=v_cache, table=table, qsl=qsl,
                seqs=np.asarray(seqs, np.int32), qsl_dev=torch.from_numpy(qsl).cuda().long(),
                seqs_dev=torch.tensor(seqs, device="cuda"), scale=d ** -0.5, weights=weights,
                observe=case["observe"] if case["observe"] > 0 else None)


# ---------------------------------------------------------------------------
def _rotate(y, cos, sin, rot, interleaved):
    head, tail = y[..., :rot], y[..., rot:]
    if interleaved:
        a, b = head[..., 0::2], head[..., 1::2]
        head = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    else:
        a, b = head[..., :rot // 2], head[..., rot // 2:]
        head = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    return torch.cat([head, tail], dim=-1)


def _plain_rope(s):
    row = s["cos_sin"][s["positions"]][:, None]
    cos, sin = row[..., :s["rot"] // 2], row[..., s["rot"] // 2:]

    def one(x, w):
        x = x.float()
        y = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * (w.float() + s["offset"])
        return _rotate(y, cos, sin, s["rot"], s["interleaved"])

    q, k = one(s["q"], s["wq"]).to(s["q"].dtype), one(s["k"], s["wk"]).to(s["k"].dtype)
    if not s["write"]:
        return q, k
    s["k_cache"].flatten(0, 1)[s["slots"]] = k
    s["v_cache"].flatten(0, 1)[s["slots"]] = s["v"]
    return q, s["k_cache"], s["v_cache"]


def _plain_attention(s):
    q, kc, page = s["q"], s["k_cache"], s["k_cache"].shape[1]
    n, hq, d = q.shape
    b, hk = len(s["seqs"]), kc.shape[2]
    longest, most = int(s["seqs"].max()), int(np.diff(s["qsl"]).max())
    pos = torch.arange(longest, device=q.device)
    slot = s["table"][:, pos // page].long() * page + pos % page                      # [b, keys]
    lens = s["qsl_dev"][1:] - s["qsl_dev"][:-1]
    token = torch.arange(n, device=q.device)
    req = torch.searchsorted(s["qsl_dev"], token, right=True) - 1
    at = token - s["qsl_dev"][req]
    i = torch.arange(most, device=q.device)
    padded = q[(s["qsl_dev"][:-1, None] + i).clamp(max=n - 1)].float()                # [b, most, hq, d]
    padded = padded.view(b, most, hk, hq // hk, d).permute(0, 2, 3, 1, 4).reshape(b, hk, -1, d)
    k = kc.flatten(0, 1)[slot].float().permute(0, 2, 3, 1)                            # [b, hk, d, keys]
    x = (padded @ k).view(b, hk, hq // hk, most, longest).mul_(s["scale"])
    sees = (s["seqs_dev"] - lens)[:, None] + i + 1                                    # keys that row i sees
    x.masked_fill_((pos >= sees[..., None])[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True).clamp(min=-1e30)
    p = x.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    v = s["v_cache"].flatten(0, 1)[slot].float().permute(0, 2, 1, 3)                  # [b, hk, keys, d]
    o = (p.view(b, hk, -1, longest) @ v).view(b, hk, hq // hk, most, d) / total
    lse = (top + total.log())[..., 0]
    out = o.permute(0, 3, 1, 2, 4).reshape(b, most, hq, d)[req, at].to(q.dtype)
    lse = lse.permute(0, 3, 1, 2).reshape(b, most, hq)[req, at]
    if s["weights"] is None:
        return out, lse
    counted = (i < lens[:, None]) & (i >= (lens[:, None] - (s["observe"] or most)))   # [b, most]
    mass = (p / total).mul_(counted[:, None, None, :, None]).sum((2, 3))              # [b, hk, keys]
    weights = s["weights"].clone()
    flat = weights.transpose(1, 2).reshape(-1, hk)                                    # [slots, hk]
    old = (pos < (s["seqs_dev"] - lens)[:, None])[..., None]
    value = torch.where(old, flat[slot], 0.0) + mass.transpose(1, 2)
    # positions past a request's end go to a spare row
    flat = torch.cat([flat, flat[:1]])
    flat[torch.where(pos < s["seqs_dev"][:, None], slot, flat.shape[0] - 1)] = value
    weights.copy_(flat[:-1].view(-1, page, hk).transpose(1, 2))
    return out, lse, weights


def _plain_evict(s):
    w, page, hk = s["weights"], s["k_cache"].shape[1], s["k_cache"].shape[2]
    longest = int(s["seqs"].max())
    keep = min(s["keep"], longest)
    pos = torch.arange(longest, device=w.device)
    slot = s["table"][:, pos // page].long() * page + pos % page
    seqs = s["seqs_dev"][:, None]
    key = w.transpose(1, 2).reshape(-1, hk)[slot].transpose(1, 2)                     # [b, hk, keys]
    key = torch.where(((pos < s["sink"]) | (pos >= seqs - s["recent"]))[:, None], math.inf, key)
    key = torch.where((pos >= seqs)[:, None], -math.inf, key)
    kept = torch.sort(key, dim=-1, descending=True, stable=True).indices[..., :keep].sort(-1).values
    there = kept < s["seqs_dev"][:, None, None]
    heads = torch.arange(hk, device=w.device)[:, None]
    j = torch.arange(keep, device=w.device)
    from_slot = slot.gather(1, kept.flatten(1)).view_as(kept)
    to_slot = (s["dst"][:, j // page].long() * page + j % page)[:, None].expand_as(kept)
    # places past a short request's end repeat the first request's first move
    first = slot[0][kept[0, :, :1]][None]
    from_slot = torch.where(there, from_slot, first)
    to_slot = torch.where(there, to_slot, s["dst"][0, 0].long() * page)
    kf, vf = s["k_cache"].flatten(0, 1), s["v_cache"].flatten(0, 1)
    kf[to_slot, heads] = kf[from_slot, heads]
    vf[to_slot, heads] = vf[from_slot, heads]
    w[to_slot // page, heads, to_slot % page] = w[from_slot // page, heads, from_slot % page]
    return torch.where(there, kept, -1).to(torch.int32), s["k_cache"], s["v_cache"], w


def _own(s):
    from oscar_b200 import kernels

    if s["op"] == "rope":
        if not s["write"]:
            return kernels.qk_norm_rope(s["q"], s["k"], None, s["wq"], s["wk"], EPS, s["cos_sin"], s["positions"],
                                        weight_offset=s["offset"], interleaved=s["interleaved"])
        q, _ = kernels.qk_norm_rope(s["q"], s["k"], s["v"], s["wq"], s["wk"], EPS, s["cos_sin"], s["positions"],
                                    weight_offset=s["offset"], interleaved=s["interleaved"], k_cache=s["k_cache"],
                                    v_cache=s["v_cache"], slot_mapping=s["slots"])
        return q, s["k_cache"], s["v_cache"]
    if s["op"] == "evict":
        kept = kernels.evict_cache(s["k_cache"], s["v_cache"], s["weights"], s["table"], s["seqs"], s["keep"], sink=s["sink"],
                                   recent=s["recent"], dst_table=s["dst"])
        return kept, s["k_cache"], s["v_cache"], s["weights"]
    if s["weights"] is None:
        return kernels.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["qsl"], s["seqs"], s["scale"])
    # the pass before this one's weights stay as they were: every pass accumulates onto the same ones
    weights = s["weights"].clone()
    out, lse = kernels.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["qsl"], s["seqs"], s["scale"],
                                       weights=weights, observe=s["observe"])
    return out, lse, weights


def run(state):
    if own:
        return _own(state)
    return {"rope": _plain_rope, "attn": _plain_attention, "evict": _plain_evict}[state["op"]](state)


# ---------------------------------------------------------------------------
def work(case):
    hq, hk, d = case["hq"], case["hk"], case["d"]
    if case["op"] == "rope":
        n, heads = case["tokens"], hq + (2 * hk if case["write"] else hk)
        return {"bytes": 2 * n * heads * d * 2 + n * (4 * case["rot"] + 8 + (8 if case["write"] else 0)) + 4 * d,
                "flops": n * (hq + hk) * (4 * d + 3 * case["rot"])}
    seqs = _ints(case["seqs"])
    if case["op"] == "evict":
        moved = sum(min(s, case["keep"]) for s in seqs)
        return {"bytes": hk * (4 * sum(seqs) + moved * (8 * d + 4 + 4)), "flops": 0}
    lens = _ints(case["lens"])
    pairs = sum(q * (s - q) + q * (q + 1) // 2 for q, s in zip(lens, seqs))
    n = sum(lens)
    bytes_ = sum(seqs) * hk * d * 4 + n * hq * (4 * d + 4)
    flops = 4 * hq * d * pairs
    if case["observe"] >= 0:
        bytes_ += 4 * hk * (2 * sum(s - q for q, s in zip(lens, seqs)) + n)
    return {"bytes": bytes_, "flops": flops}


# ---------------------------------------------------------------------------
def _exact_rope(s):
    d, rot, half = s["q"].shape[-1], s["rot"], s["rot"] // 2
    angle = s["cos_sin"].double().index_select(0, s["positions"])
    first = torch.arange(0, rot, 2, device="cuda") if s["interleaved"] else torch.arange(half, device="cuda")
    second = first + (1 if s["interleaved"] else half)

    def one(x, w):
        x = x.double()
        y = x / torch.sqrt((x * x).sum(-1, keepdim=True) / d + EPS) * (w.double() + s["offset"])
        z = y.clone()
        c, sn = angle[:, None, :half], angle[:, None, half:]
        z[..., first] = c * y[..., first] - sn * y[..., second]
        z[..., second] = sn * y[..., first] + c * y[..., second]
        return z

    q, k = one(s["q"], s["wq"]), one(s["k"], s["wk"])
    if not s["write"]:
        return q, k
    kc, vc = s["k_cache"].double(), s["v_cache"].double()
    kc.view(-1, *kc.shape[2:]).index_copy_(0, s["slots"], k)
    vc.view(-1, *vc.shape[2:]).index_copy_(0, s["slots"], s["v"].double())
    return q, kc, vc


def _exact_attention(s):
    n, hq, d = s["q"].shape
    page, hk = s["k_cache"].shape[1:3]
    group = hq // hk
    out = torch.zeros(n, hq, d, dtype=torch.float64, device="cuda")
    lse = torch.full((n, hq), -math.inf, dtype=torch.float64, device="cuda")
    weights = None if s["weights"] is None else s["weights"].double()
    for r, seq in enumerate(s["seqs"].tolist()):
        a, b = int(s["qsl"][r]), int(s["qsl"][r + 1])
        p = torch.arange(seq, device="cuda")
        blk, off = s["table"][r].long()[p // page], p % page
        for h in range(hk):
            k, v = s["k_cache"][blk, off, h].double(), s["v_cache"][blk, off, h].double()
            mass = torch.zeros(seq, dtype=torch.float64, device="cuda")
            for t0 in range(a, b, 1024):
                t1 = min(b, t0 + 1024)
                t = torch.arange(t0, t1, device="cuda")
                x = torch.einsum("tgd,kd->tgk", s["q"][t0:t1, h * group:(h + 1) * group].double(), k) * s["scale"]
                hidden = p[None] > (seq - (b - t))[:, None]
                x = x.masked_fill(hidden[:, None], -math.inf)
                z = torch.logsumexp(x, -1)
                prob = torch.exp(x - z[..., None])
                out[t0:t1, h * group:(h + 1) * group] = torch.einsum("tgk,kd->tgd", prob, v)
                lse[t0:t1, h * group:(h + 1) * group] = z
                if weights is not None:
                    mass += prob[(b - t) <= (s["observe"] or n)].sum((0, 1))
            if weights is not None:
                weights[blk, h, off] = torch.where(p < seq - (b - a), weights[blk, h, off], 0.0) + mass
    return (out, lse) if weights is None else (out, lse, weights)


def _exact_evict(s):
    page, hk = s["k_cache"].shape[1:3]
    kc, vc, w = s["k_cache"].double(), s["v_cache"].double(), s["weights"].double()
    source = s["weights"]
    for r, seq in enumerate(s["seqs"].tolist()):
        p = torch.arange(seq, device="cuda")
        blk, off = s["table"][r].long()[p // page], p % page
        j = torch.arange(min(seq, s["keep"]), device="cuda")
        to_blk, to_off = s["dst"][r].long()[j // page], j % page
        for h in range(hk):
            value = source[blk, h, off].cpu().numpy()
            middle = np.arange(seq)[s["sink"]:max(seq - s["recent"], s["sink"])]
            order = middle[np.lexsort((middle, -value[middle]))]
            fixed = np.setdiff1d(np.arange(seq), middle)
            chosen = np.arange(seq) if seq <= s["keep"] else np.sort(np.concatenate([fixed, order[:s["keep"] - fixed.size]]))
            c = torch.from_numpy(chosen).cuda()
            for t in (kc, vc):
                t[to_blk, to_off, h] = t[blk[c], off[c], h]
            w[to_blk, h, to_off] = w[blk[c], h, off[c]]
    return None, kc, vc, w


def exact(case, seed):
    s = prepare(case, seed)
    return {"rope": _exact_rope, "attn": _exact_attention, "evict": _exact_evict}[case["op"]](s)
