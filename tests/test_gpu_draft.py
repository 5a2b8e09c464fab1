"""DraftLayer: prompt, draft steps, eviction and steps after it, against a plain
64-bit restatement that keeps every head's rows in lists.

Tolerance: the rows that reach the attention are 16-bit; a rounding that falls
the other way moves a key or value by one unit (2 u relative).  Scores then move
by at most 2 u sum |q k| scale = SHIFT below, which weighs the output like
test_gpu_paged16's score error; the rest is that test's bound."""
import math

import numpy as np
import pytest
import torch

from gpu_helpers import need_gpu

pytestmark = pytest.mark.gpu

HQ, HK, D, PAGE, ROT = 8, 2, 64, 16, 32
U = torch.finfo(torch.bfloat16).eps / 2


def norm_rope(x, w, cos_sin, positions):
    x = x.double()
    y = x / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-6) * (1 + w.double())
    row = cos_sin.double()[positions][:, None]
    c, s, h = row[..., :ROT // 2], row[..., ROT // 2:], ROT // 2
    return torch.cat([y[..., :h] * c - y[..., h:ROT] * s, y[..., h:ROT] * c + y[..., :h] * s, y[..., ROT:]], -1)


class Plain:
    """Rows, weights and original positions per request and head."""

    def __init__(self, n):
        self.k = [[torch.zeros(0, D, dtype=torch.float64, device="cuda") for _ in range(HK)] for _ in range(n)]
        self.v = [[torch.zeros(0, D, dtype=torch.float64, device="cuda") for _ in range(HK)] for _ in range(n)]
        self.w = [[torch.zeros(0, dtype=torch.float64, device="cuda") for _ in range(HK)] for _ in range(n)]

    def step(self, q, k, v, lens):
        outs, sizes, at = [], [], 0
        for r, m in enumerate(lens):
            o = torch.zeros(m, HQ, D, dtype=torch.float64, device="cuda")
            size = torch.zeros_like(o)
            for h in range(HK):
                self.k[r][h] = torch.cat([self.k[r][h], k[at:at + m, h]])
                self.v[r][h] = torch.cat([self.v[r][h], v[at:at + m, h]])
                self.w[r][h] = torch.cat([self.w[r][h], torch.zeros(m, dtype=torch.float64, device="cuda")])
                g = slice(h * (HQ // HK), (h + 1) * (HQ // HK))
                x = torch.einsum("mgd,kd->mgk", q[at:at + m, g], self.k[r][h]) * D**-0.5
                n = self.k[r][h].shape[0]
                hidden = torch.arange(n, device="cuda")[None] > torch.arange(n - m, n, device="cuda")[:, None]
                p = torch.softmax(x.masked_fill(hidden[:, None], -math.inf), -1)
                o[:, g] = torch.einsum("mgk,kd->mgd", p, self.v[r][h])
                size[:, g] = torch.einsum("mgk,kd->mgd", p, self.v[r][h].abs())
                self.w[r][h] += p.sum((0, 1))
            outs.append(o)
            sizes.append(size)
            at += m
        return torch.cat(outs), torch.cat(sizes)

    def take(self, kept):
        for r in range(len(self.k)):
            for h in range(HK):
                c = kept[r, h][kept[r, h] >= 0].long()
                self.k[r][h], self.v[r][h], self.w[r][h] = self.k[r][h][c], self.v[r][h][c], self.w[r][h][c]


def test_prompt_steps_eviction_and_steps_after_it():
    from oscar_b200 import kernels
    from oscar_b200.draft import DraftLayer, slots_of

    dev = need_gpu()
    gen = torch.Generator(device="cuda").manual_seed(7)
    n, width = 3, 16
    pool = torch.full((n * width + 2, 2, PAGE, HK, D), math.nan, device="cuda").to(torch.bfloat16)
    perm = torch.randperm(n * width, generator=gen, device="cuda")
    table = perm.to(torch.int32).view(n, width)
    wq, wk = (torch.randn(D, generator=gen, device="cuda") * 0.1 for _ in range(2))
    angle = torch.arange(400, device="cuda", dtype=torch.float64)[:, None] / 1e4 ** (
        torch.arange(0, ROT, 2, device="cuda", dtype=torch.float64) / ROT)
    cos_sin = torch.cat([angle.cos(), angle.sin()], 1).float()
    layer = DraftLayer(HQ, (pool[:, 0], pool[:, 1]), wq, wk, cos_sin, weight_offset=1.0, keep=40, sink=3, recent=8)
    plain = Plain(n)
    cached, position = [0] * n, [0] * n

    def step(lens):
        nonlocal cached, position
        total = sum(lens)
        qkv = torch.randn(total, HQ + 2 * HK, D, generator=gen, device="cuda").to(torch.bfloat16)
        q, k, v = qkv.split([HQ, HK, HK], 1)
        positions = torch.cat([torch.arange(p, p + m, device="cuda") for p, m in zip(position, lens)])
        cached = [c + m for c, m in zip(cached, lens)]
        position = [p + m for p, m in zip(position, lens)]
        qsl = np.concatenate([[0], np.cumsum(lens)])
        out, lse = layer.forward(q, k, v, positions, slots_of(table, lens, cached, PAGE), table, qsl, cached)
        assert torch.isfinite(out.float()).all() and torch.isfinite(lse).all()
        bf = lambda t: t.to(torch.bfloat16).double()  # noqa: E731
        want, size = plain.step(bf(norm_rope(q, wq, cos_sin, positions)), bf(norm_rope(k, wk, cos_sin, positions)),
                                v.double(), lens)
        # sum |q k| scale <= |q| |k| scale with norms of at most 1.5 sqrt(D)
        shift = 2 * U * 2.25 * D * D**-0.5
        assert ((out.double() - want).abs() <= U * (size + want.abs()) * 1.01 + 2 * (shift + 2e-4) * size).all()

    step([100, 61, 30])
    for _ in range(3):
        step([2, 1, 4])
    # the layer's weights are those of the plain steps, so the same keys stay
    before = cached
    new, kept = layer.evict(table, cached)
    assert new == [40, 40, 40] and kept.shape == (n, HK, 40)
    for r in range(n):
        for h in range(HK):
            c = kept[r, h].long()
            assert c[:3].tolist() == [0, 1, 2] and c[-8:].tolist() == list(range(before[r] - 8, before[r]))
            w = plain.w[r][h].clone()
            w[:3] = w[-8:] = math.inf
            out_of = torch.ones(before[r], dtype=torch.bool, device="cuda")
            out_of[c] = False
            # (weights carry errors of a few 1e-3 through 16-bit rows: the split may differ between near ties)
            assert w[out_of].max() <= w[c].min() * 1.05
    plain.take(kept)
    cached = new
    for _ in range(3):
        step([1, 3, 2])
    # into other pages
    dst = torch.full((n, 3), -1, dtype=torch.int32, device="cuda")
    used = set(table[:, :3].flatten().tolist())
    free = [b for b in perm.tolist() if b not in used]
    for r in range(n):
        dst[r] = torch.tensor(free[3 * r:3 * r + 3], dtype=torch.int32)
    new, kept = layer.evict(table, cached, dst_table=dst)
    plain.take(kept)
    table = torch.cat([dst, torch.tensor(free[9:9 + n], dtype=torch.int32, device="cuda")[:, None]], 1)
    cached = new
    step([4, 1, 1])
    assert kernels.device_error(dev) == 0


class Rows:
    """Per request and head: the rows that the cache holds, in 64 bits, and the keys' weights."""

    def __init__(self, n, hq, hk, d, observe):
        self.hq, self.hk, self.d, self.observe = hq, hk, d, observe
        none = lambda *shape: torch.zeros(*shape, dtype=torch.float64, device="cuda")  # noqa: E731
        self.k = [[none(0, d) for _ in range(hk)] for _ in range(n)]
        self.v = [[none(0, d) for _ in range(hk)] for _ in range(n)]
        self.w = [[none(0) for _ in range(hk)] for _ in range(n)]

    def step(self, q, k, v, lens):
        g = self.hq // self.hk
        out, size = torch.zeros_like(q), torch.zeros_like(q)
        lse = torch.zeros(q.shape[:2], dtype=torch.float64, device="cuda")
        at = 0
        for r, m in enumerate(lens):
            for h in range(self.hk):
                self.k[r][h] = torch.cat([self.k[r][h], k[at:at + m, h]])
                self.v[r][h] = torch.cat([self.v[r][h], v[at:at + m, h]])
                self.w[r][h] = torch.cat([self.w[r][h], torch.zeros(m, dtype=torch.float64, device="cuda")])
                n, heads = self.k[r][h].shape[0], slice(h * g, (h + 1) * g)
                x = torch.einsum("mgd,kd->mgk", q[at:at + m, heads], self.k[r][h]) * self.d**-0.5
                hidden = torch.arange(n, device="cuda")[None] > torch.arange(n - m, n, device="cuda")[:, None]
                x = x.masked_fill(hidden[:, None], -math.inf)
                z = torch.logsumexp(x, -1)
                p = torch.exp(x - z[..., None])
                out[at:at + m, heads] = torch.einsum("mgk,kd->mgd", p, self.v[r][h])
                size[at:at + m, heads] = torch.einsum("mgk,kd->mgd", p, self.v[r][h].abs())
                lse[at:at + m, heads] = z
                self.w[r][h] = self.w[r][h] + p[max(0, m - (self.observe or m)):].sum((0, 1))
            at += m
        return out, size, lse

    def take(self, kept):
        for r in range(len(self.k)):
            for h in range(self.hk):
                c = kept[r, h][kept[r, h] >= 0].long()
                self.k[r][h], self.v[r][h], self.w[r][h] = self.k[r][h][c], self.v[r][h][c], self.w[r][h][c]


@pytest.mark.parametrize("hq,hk,d,page,rot,dtype,observe", [
    (8, 2, 64, 16, 32, torch.bfloat16, None), (24, 4, 256, 32, 64, torch.bfloat16, 2), (12, 3, 128, 48, 128, torch.float16, 1),
    (16, 2, 256, 128, 128, torch.float16, None),
])
def test_layer_on_the_rows_it_caches(hq, hk, d, page, rot, dtype, observe):
    """As above, but every part against what it was given.  The rows that the layer caches and attends
    are read back (queries: the norm alone on the same inputs) and checked against the norm and rotation
    in 64 bits within one rounding; outputs, LSE and weights are then those of these very rows.

    Bound of a score: |q|, |k| < 1.5 sqrt(D) (norm weights under 1.5), so D products summed in fp32 are
    off by at most D 2^-24 2.25 D D^-1/2; the exponential, its argument and the sum of at most 400 terms
    add less than 3e-5.  A probability carries that twice (its own and the sum's)."""
    from oscar_b200 import kernels
    from oscar_b200.draft import DraftLayer, slots_of
    from test_gpu_paged16 import check_rows, kept64, rope64

    dev = need_gpu()
    u, err = torch.finfo(dtype).eps / 2, 2.25 * d**1.5 * 2.0**-24 + 3e-5
    gen = torch.Generator(device="cuda").manual_seed(21)
    n, width, keep, sink, recent = 3, -(-250 // page), 90, 5, 20
    fresh = -(-keep // page) + 1
    pool = torch.full((n * (width + fresh) + 1, 2, page, hk, d), math.nan, device="cuda").to(dtype)
    perm = torch.randperm(pool.shape[0], generator=gen, device="cuda").to(torch.int32)
    table, dst = perm[:n * width].view(n, width), perm[n * width:n * (width + fresh)].view(n, fresh)
    wq, wk = (torch.rand(d, generator=gen, device="cuda") - 0.5 for _ in range(2))
    angle = torch.arange(400, device="cuda", dtype=torch.float64)[:, None] / 1e4 ** (
        torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot)
    cos_sin = torch.cat([angle.cos(), angle.sin()], 1).float()
    kc, vc = pool[:, 0], pool[:, 1]
    layer = DraftLayer(hq, (kc, vc), wq, wk, cos_sin, weight_offset=1.0, keep=keep, sink=sink, recent=recent, observe=observe)
    rows, cached, position, steps = Rows(n, hq, hk, d, observe), [0] * n, [0] * n, 0

    def held(r):  # pages and places of a request's cached tokens
        p = torch.arange(cached[r], device="cuda")
        return table[r].long()[p // page], p % page

    def check_cache():
        for r in range(n):
            blk, off = held(r)
            for h in range(hk):
                assert torch.equal(kc[blk, off, h].double(), rows.k[r][h])
                assert torch.equal(vc[blk, off, h].double(), rows.v[r][h])
                w = layer.weights[blk, h, off].double()
                assert ((w - rows.w[r][h]).abs() <= (2 * err + steps * 2.0**-23) * rows.w[r][h]).all()

    def step(lens):
        nonlocal cached, position, steps
        qkv = torch.randn(sum(lens), hq + 2 * hk, d, generator=gen, device="cuda").to(dtype)
        q, k, v = qkv.split([hq, hk, hk], 1)
        positions = torch.cat([torch.arange(p, p + m, device="cuda") for p, m in zip(position, lens)])
        cached, position, steps = [c + m for c, m in zip(cached, lens)], [p + m for p, m in zip(position, lens)], steps + 1
        slots = slots_of(table, lens, cached, page)
        qsl = np.concatenate([[0], np.cumsum(lens)])
        out, lse = layer.forward(q, k, v, positions, slots, table, qsl, cached)
        q16, k16 = kernels.qk_norm_rope(q, k, None, wq, wk, 1e-6, cos_sin, positions, weight_offset=1.0)
        for got, x, w in ((q16, q, wq), (k16, k, wk)):
            check_rows(got, *rope64(x, w, 1.0, 1e-6, cos_sin, positions, False), dtype)
        assert torch.equal(kc[slots // page, slots % page], k16) and torch.equal(vc[slots // page, slots % page], v)
        want, size, z = rows.step(q16.double(), k16.double(), v.double(), lens)
        tiny = max(cached) * 2.0**-25 * 6.0 if dtype == torch.float16 else 0.0
        assert ((out.double() - want).abs() <= u * (size + want.abs()) * 1.01 + 2 * err * size + tiny).all()
        assert ((lse.double() - z).abs() <= 2 * err).all()
        check_cache()

    def evict(to):
        nonlocal cached, table
        before = [layer.weights[held(r)[0], :, held(r)[1]].T.cpu().numpy() for r in range(n)]
        cached, kept = layer.evict(table, cached, dst_table=to)
        for r in range(n):
            for h in range(hk):
                c = kept64(before[r][h], keep, sink, recent)
                assert kept[r, h][kept[r, h] >= 0].tolist() == c.tolist() and cached[r] == c.size
        rows.take(kept)
        table = table if to is None else to
        check_cache()

    step([100, 61, 30])
    for _ in range(3):
        step([2, 1, 4])
    evict(None)
    for _ in range(3):
        step([1, 3, 30])
    evict(dst)
    step([4, 1, 1])
    assert kernels.device_error(dev) == 0


def test_step_replayed_from_a_graph():
    """A captured step attends the lengths it was captured with, on whatever its buffers hold."""
    from oscar_b200 import kernels
    from oscar_b200.draft import DraftLayer, slots_of

    dev = need_gpu()
    gen = torch.Generator(device="cuda").manual_seed(8)
    lens, seqs, page = [3, 150, 1], [700, 400, 90], 32
    table = torch.randperm(66, generator=gen, device="cuda").to(torch.int32).view(3, 22)
    start = torch.randn(2, 66, page, 4, 256, generator=gen, device="cuda").to(torch.bfloat16)
    wq = torch.randn(256, generator=gen, device="cuda") * 0.1
    angle = torch.arange(800, device="cuda")[:, None] / 1e4 ** (torch.arange(0, 64, 2, device="cuda") / 64)
    cos_sin = torch.cat([angle.cos(), angle.sin()], 1)
    qkv = torch.zeros(154, 32, 256, dtype=torch.bfloat16, device="cuda")
    positions = torch.zeros(154, dtype=torch.int64, device="cuda")
    slots, qsl = slots_of(table, lens, seqs, page), [0, 3, 153, 154]

    def layer_on(pool):
        return DraftLayer(24, pool, wq, wq, cos_sin, weight_offset=1.0, keep=80, sink=4, recent=16)

    def step(layer):
        out = layer.forward(qkv[:, :24], qkv[:, 24:28], qkv[:, 28:], positions, slots, table, qsl, seqs)
        return *out, layer.evict(table, seqs)[1]

    captured = layer_on(start.clone())
    step(captured)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(captured)
    for _ in range(3):
        qkv.copy_(torch.randn(qkv.shape, generator=gen, device="cuda"))
        positions.copy_(torch.randint(0, 800, (154,), generator=gen, device="cuda"))
        for t, s in ((captured.k_cache, start[0]), (captured.v_cache, start[1])):
            t.copy_(s)
        captured.weights.zero_()
        graph.replay()
        eager = layer_on(start.clone())
        want = step(eager)
        for x, y in zip((*got, captured.k_cache, captured.v_cache, captured.weights),
                        (*want, eager.k_cache, eager.v_cache, eager.weights)):
            assert torch.equal(x, y)
    assert kernels.device_error(dev) == 0
    del graph


def test_two_threads_on_streams_of_their_own():
    """Calls of two host threads share no state of the library: each gets what it gets alone."""
    from concurrent.futures import ThreadPoolExecutor

    from oscar_b200 import kernels

    dev = need_gpu()
    gen = torch.Generator(device="cuda").manual_seed(31)
    jobs = []
    for lens, seqs, d in (([3, 200], [900, 1500], 256), ([150, 2, 40], [700, 2000, 64], 128)):
        pages = [-(-s // 32) for s in seqs]
        table = torch.zeros(len(seqs), max(pages), dtype=torch.int32, device="cuda")
        perm = torch.randperm(sum(pages), generator=gen, device="cuda").to(torch.int32)
        for r, n in enumerate(pages):
            table[r, :n] = perm[sum(pages[:r]):sum(pages[:r]) + n]
        q, k = (torch.randn(sum(lens), h, d, generator=gen, device="cuda").to(torch.bfloat16) for h in (24, 4))
        pool = torch.randn(2, sum(pages), 32, 4, d, generator=gen, device="cuda").to(torch.bfloat16)
        jobs.append((q, k, pool, table, np.concatenate([[0], np.cumsum(lens)]).astype(np.int32), seqs, torch.ones(d, device="cuda"),
                     torch.randn(100, 64, generator=gen, device="cuda"), torch.arange(sum(lens), device="cuda") % 100))

    def work(job, stream):
        q, k, pool, table, qsl, seqs, w, cos_sin, positions = job
        results = []
        with torch.cuda.stream(stream):
            for _ in range(8):
                kc, vc = pool.clone()
                weights = torch.zeros(kc.shape[0], 4, 32, device="cuda")
                x, y = kernels.qk_norm_rope(q, k, None, w, w, 1e-6, cos_sin, positions)
                out = kernels.paged_attention(x, kc, vc, table, qsl, seqs, 0.1, weights=weights)
                kept = kernels.evict_cache(kc, vc, weights, table, seqs, 300, sink=3, recent=40)
                results.append((x, y, *out, kept, kc, vc, weights))
        stream.synchronize()
        return results

    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    alone = [work(job, stream) for job, stream in zip(jobs, streams)]
    with ThreadPoolExecutor(2) as pool:
        together = list(pool.map(work, jobs, streams))
    for a, b in zip(alone, together):
        for x, y in zip(a, b):
            assert all(torch.equal(s, t) for s, t in zip(x, y))
    assert kernels.device_error(dev) == 0


def test_draft_layer_refusals():
    from oscar_b200.draft import DraftLayer

    need_gpu()
    pool = torch.zeros(2, 4, PAGE, HK, D, dtype=torch.bfloat16, device="cuda")
    w, t = torch.zeros(D, device="cuda"), torch.zeros(8, ROT, device="cuda")
    with pytest.raises(ValueError, match="multiple"):
        DraftLayer(7, pool, w, w, t)
    with pytest.raises(ValueError, match="sink and recent"):
        DraftLayer(HQ, pool, w, w, t, keep=10, sink=8, recent=8)
    with pytest.raises(ValueError, match="keeps no weights"):
        DraftLayer(HQ, pool, w, w, t).evict(torch.zeros(1, 4, dtype=torch.int32, device="cuda"), [5])
