"""The 16-bit paged layer on the GPU against plain 64-bit implementations: head
norm + rotation + cache write, attention over the paged cache, the keys'
accumulated weights, eviction by weight.

Tolerances (u: unit roundoff of the type, half of its eps, 2^-8 bf16, 2^-11 fp16):
  * attention output: the probabilities are rounded to the type for the P V
    product and the result once more, so |err| <= u (sum p |v| + |o|); scores
    carry fp32 errors of at most SCORE (below), worth 2 SCORE sum p |v|; fp16
    probabilities under 2^-14 of the largest lose at most 2^-25 each.
  * LSE and weights: a score is a sum of D products in fp32, error at most
    D 2^-24 sum |q k| scale < 2^-24 * 256 * 260 / 16 < 2.6e-4 for N(0, 1)
    inputs (sum |q k| < 260 at D 256); a weight is a sum of exp(score - lse)
    with a relative error of twice that.
  * head norm: fp32 throughout, one rounding: u |y| + 4e-6 |largest partner|."""
import math

import numpy as np
import pytest
import torch

from gpu_helpers import need_gpu

pytestmark = pytest.mark.gpu

U = {t: torch.finfo(t).eps / 2 for t in (torch.bfloat16, torch.float16)}
SCORE = 2.6e-4


def randn(gen, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=gen, device="cuda").to(dtype)


def make_pool(gen, seqs, page, hk, d, dtype, *, spare=3, layout="plain", poison=True):
    """Caches whose pages lie in random order; slots no request owns hold NaN / inf."""
    need = [-(-s // page) for s in seqs]
    blocks = sum(need) + spare
    perm = torch.randperm(blocks, generator=gen, device="cuda").to(torch.int32)
    width = max(max(need, default=0), 1) + 2
    table = torch.full((len(seqs), width), -7, dtype=torch.int32, device="cuda")
    at = 0
    for r, n in enumerate(need):
        table[r, :n] = perm[at:at + n]
        at += n
    if layout == "plain":
        kc, vc = randn(gen, blocks, page, hk, d, dtype=dtype), randn(gen, blocks, page, hk, d, dtype=dtype)
    elif layout == "halves":  # K and V of a block adjacent
        pool = randn(gen, blocks, 2, page, hk, d, dtype=dtype)
        kc, vc = pool[:, 0], pool[:, 1]
    else:  # heads before tokens
        kc = randn(gen, blocks, hk, page, d, dtype=dtype).transpose(1, 2)
        vc = randn(gen, blocks, hk, page, d, dtype=dtype).transpose(1, 2)
    if poison:
        owned = torch.zeros(blocks, page, dtype=torch.bool, device="cuda")
        for r, s in enumerate(seqs):
            p = torch.arange(s, device="cuda")
            owned[table[r].long()[p // page], p % page] = True
        for c, bad in ((kc, math.nan), (vc, math.inf)):
            c.masked_fill_(~owned[:, :, None, None], bad)
    return kc, vc, table


def gather(cache, table, r, seq):
    p = torch.arange(seq, device="cuda")
    page = cache.shape[1]
    return cache[table[r].long()[p // page], p % page]


def attention64(q, kc, vc, table, lens, seqs, scale, observe=None):
    """(out, sum p |v|, lse, [mass per request [hk, seq]]) in 64 bits."""
    n, hq, d = q.shape
    hk = kc.shape[2]
    g = hq // hk
    out = torch.zeros(n, hq, d, dtype=torch.float64, device="cuda")
    size = torch.zeros_like(out)
    lse = torch.full((n, hq), -math.inf, dtype=torch.float64, device="cuda")
    masses, at = [], 0
    for r, (m, seq) in enumerate(zip(lens, seqs)):
        mass = torch.zeros(hk, seq, dtype=torch.float64, device="cuda")
        if m and seq:
            k, v = gather(kc, table, r, seq).double(), gather(vc, table, r, seq).double()
            qq = q[at:at + m].double().view(m, hk, g, d)
            x = torch.einsum("mhgd,khd->mhgk", qq, k) * scale
            sees = (seq - m + 1 + torch.arange(m, device="cuda"))[:, None]
            x = x.masked_fill((torch.arange(seq, device="cuda")[None] >= sees)[:, None, None], -math.inf)
            z = torch.logsumexp(x, -1)
            p = torch.where(x == -math.inf, 0.0, torch.exp(x - torch.where(z == -math.inf, 0.0, z)[..., None]))
            out[at:at + m] = torch.einsum("mhgk,khd->mhgd", p, v).reshape(m, hq, d)
            size[at:at + m] = torch.einsum("mhgk,khd->mhgd", p, v.abs()).reshape(m, hq, d)
            lse[at:at + m] = z.reshape(m, hq)
            mass = p[max(0, m - (observe or m)):].sum((0, 2))
        masses.append(mass)
        at += m
    return out, size, lse, masses


def check_attention(q, out, lse, want, seqs):
    o, size, z, _ = want
    u = U[q.dtype]
    tiny = max(seqs, default=0) * 2.0**-25 * 6.0 if q.dtype == torch.float16 else 0.0
    bound = u * (size + o.abs()) * 1.01 + 2 * SCORE * size + tiny
    off = (out.double() - o).abs()
    assert torch.isfinite(out.float()).all()
    assert (off <= bound).all(), float((off - bound).max())
    empty = z == -math.inf
    assert torch.equal(lse == -math.inf, empty)
    assert (out[empty] == 0).all()
    assert ((lse.double() - z)[~empty].abs() <= SCORE).all()


# (new tokens, cached lengths, options)
CASES = [
    ([1], [1], dict()),
    ([1], [64], dict()),
    ([1], [8192], dict()),
    ([4] * 3, [3000, 65, 4], dict()),
    ([1, 0, 3, 2, 4], [1500, 700, 128, 2, 129], dict(page=16)),
    ([4, 4], [2049, 700], dict(hq=6, hk=1)),
    ([2, 1], [900, 333], dict(hq=24, hk=4, d=128, dtype=torch.float16, page=48)),
    ([3, 1], [1000, 63], dict(hq=8, hk=8, d=64, dtype=torch.float16, page=32)),
    ([1, 5], [700, 77], dict(hq=16, hk=2, d=128, page=5)),                 # pages no box of two tokens divides
    ([7], [7], dict(hq=32, hk=1, d=64, page=1)),                            # every token its own page
    ([5, 3], [2, 0], dict()),                                               # rows that see no key
    ([300], [300], dict(hq=24, hk=4)),                                      # a prompt
    ([130, 1, 33], [1130, 900, 33], dict(hq=12, hk=2, page=784)),           # a chunk beside decode
    ([257], [1281], dict(hq=24, hk=4, dtype=torch.float16)),
    ([200, 129], [200, 1000], dict(hq=24, hk=4, d=128, dtype=torch.float16, page=16)),
    ([511], [3100], dict(hq=10, hk=2, d=64, page=64)),
    ([128], [4096], dict(hq=8, hk=2, d=128, page=24)),
    ([40], [100], dict(hq=40, hk=1, d=256, page=128)),
    ([3], [20000], dict(hq=8, hk=1, d=256)),
    # more than 32 key tiles per SM: few rows on the tensor-memory kernel
    ([4, 1, 3], [41000, 5003, 130], dict(hq=48, hk=8)),
    ([2, 1], [50000, 41], dict(hq=24, hk=8, d=128, dtype=torch.float16, page=48)),
    ([1, 2], [39999, 9000], dict(hq=32, hk=16, d=64, dtype=torch.float16, page=16)),
    # between 33 and 128 rows per kv head
    ([20], [3000], dict()),
    ([21, 6, 13], [21, 1000, 700], dict(page=24)),
    ([9, 30], [500, 900], dict(hq=16, hk=4, d=128, dtype=torch.float16, page=16)),
    ([17], [640], dict(hq=35, hk=5, d=64)),
    ([1, 2], [333, 90], dict(hq=128, hk=1, d=64, page=32)),
]


def make_call(lens, seqs, opts, seed=0):
    o = dict(hq=24, hk=4, d=256, dtype=torch.bfloat16, page=128, layout="plain")
    o.update(opts)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kc, vc, table = make_pool(gen, seqs, o["page"], o["hk"], o["d"], o["dtype"], layout=o["layout"])
    q = randn(gen, sum(lens), o["hq"], o["d"], dtype=o["dtype"])
    qsl = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    return q, kc, vc, table, qsl, o["d"] ** -0.5


@pytest.mark.parametrize("lens,seqs,opts", CASES)
def test_paged_attention(lens, seqs, opts):
    from oscar_b200 import kernels

    dev = need_gpu()
    q, kc, vc, table, qsl, scale = make_call(lens, seqs, opts)
    out, lse = kernels.paged_attention(q, kc, vc, table, qsl.tolist(), seqs, scale)
    check_attention(q, out, lse, attention64(q, kc, vc, table, lens, seqs, scale), seqs)
    assert out.dtype == q.dtype and lse.dtype == torch.float32
    again, lse2 = kernels.paged_attention(q, kc, vc, table, qsl, np.asarray(seqs, np.int32), scale)
    assert torch.equal(out, again) and torch.equal(lse, lse2)
    assert kernels.device_error(dev) == 0


@pytest.mark.parametrize("layout", ["halves", "heads"])
@pytest.mark.parametrize("lens,seqs", [([2, 4], [300, 1025]), ([150], [700])])
def test_paged_attention_strided(layout, lens, seqs):
    from oscar_b200 import kernels

    need_gpu()
    q, kc, vc, table, qsl, scale = make_call(lens, seqs, dict(layout=layout, page=32))
    gen = torch.Generator(device="cuda").manual_seed(9)
    fused = randn(gen, q.shape[0], q.shape[1] + 8, q.shape[2], dtype=q.dtype)
    view = fused[:, 3:3 + q.shape[1]]
    view.copy_(q)
    out, lse = kernels.paged_attention(view, kc, vc, table, qsl, seqs, scale)
    check_attention(q, out, lse, attention64(q, kc, vc, table, lens, seqs, scale), seqs)


def test_paged_attention_many_requests():
    """More requests than one launch holds, decode and chunks mixed."""
    from oscar_b200 import kernels

    need_gpu()
    lens = [1 + (i % 3) + (60 if i % 97 == 5 else 0) for i in range(600)]
    seqs = [n + (i * 37) % 301 for i, n in enumerate(lens)]
    q, kc, vc, table, qsl, scale = make_call(lens, seqs, dict(hq=4, hk=2, d=64, page=16))
    out, lse = kernels.paged_attention(q, kc, vc, table, qsl, seqs, scale)
    check_attention(q, out, lse, attention64(q, kc, vc, table, lens, seqs, scale), seqs)


@pytest.mark.parametrize("d,dtype,hq,hk", [(256, torch.bfloat16, 24, 4), (128, torch.float16, 16, 4), (64, torch.bfloat16, 16, 4)])
def test_paged_attention_long_streams(d, dtype, hq, hk):
    """Chunks long enough that every SM streams many tiles of several units, again and again."""
    from oscar_b200 import kernels

    dev = need_gpu()
    lens, seqs = [1500, 700], [5000, 700]
    q, kc, vc, table, qsl, scale = make_call(lens, seqs, dict(d=d, dtype=dtype, hq=hq, hk=hk))
    out, lse = kernels.paged_attention(q, kc, vc, table, qsl, seqs, scale)
    check_attention(q, out, lse, attention64(q, kc, vc, table, lens, seqs, scale), seqs)
    for _ in range(20):
        again, lse2 = kernels.paged_attention(q, kc, vc, table, qsl, seqs, scale)
    assert torch.equal(out, again) and torch.equal(lse, lse2)
    assert kernels.device_error(dev) == 0


def test_paged_attention_large_scores():
    """Scores that grow along the keys move the running maximum again and again."""
    from oscar_b200 import kernels

    need_gpu()
    for lens, seqs in (([2], [2000]), ([200], [2000])):
        q, kc, vc, table, qsl, scale = make_call(lens, seqs, dict(hq=4, hk=2, d=128))
        for p in range(0, 2000, 64):
            blk, off = int(table[0, p // 128]), p % 128
            kc[blk, off] = kc[blk, off] * (1 + p / 250)
        out, lse = kernels.paged_attention(q, kc, vc, table, qsl, seqs, scale)
        o, size, z, _ = attention64(q, kc, vc, table, lens, seqs, scale)
        # scores reach 9 times N(0, 1) ones
        bound = U[q.dtype] * (size + o.abs()) * 1.01 + 18 * SCORE * size
        assert ((out.double() - o).abs() <= bound).all()
        assert ((lse.double() - z).abs() <= 9 * SCORE).all()


def test_paged_attention_nan_key_and_value():
    """A NaN key makes the rows that see it NaN and leaves other requests alone."""
    from oscar_b200 import kernels

    need_gpu()
    lens, seqs = [1, 1], [200, 130]
    q, kc, vc, table, qsl, scale = make_call(lens, seqs, dict())
    kc[int(table[0, 0]), 5, 0, 3] = math.nan
    out, lse = kernels.paged_attention(q, kc, vc, table, qsl, seqs, scale)
    assert torch.isnan(out[0, :6]).all() and torch.isnan(lse[0, :6]).all()
    assert torch.isfinite(out[0, 6:]).all() and torch.isfinite(out[1]).all()


def test_paged_attention_bad_block_is_flagged():
    from oscar_b200 import kernels

    dev = need_gpu()
    for lens in ([1], [100]):
        q, kc, vc, table, qsl, scale = make_call(lens, [400], dict())
        table[0, 1] = kc.shape[0] + 5
        kernels.paged_attention(q, kc, vc, table, qsl, [400], scale)
        assert kernels.device_error(dev) & 2
    assert kernels.device_error(dev) == 0


def test_paged_attention_other_stream_and_preallocated_out():
    from oscar_b200 import kernels

    need_gpu()
    lens, seqs = [4, 4], [3000, 500]
    q, kc, vc, table, qsl, scale = make_call(lens, seqs, dict())
    want, _ = kernels.paged_attention(q, kc, vc, table, qsl, seqs, scale)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = torch.full_like(q, math.nan)
        got, _ = kernels.paged_attention(q, kc, vc, table, qsl, seqs, scale, out=out)
    side.synchronize()
    assert got.data_ptr() == out.data_ptr() and torch.equal(got, want)


@pytest.mark.parametrize("lens,seqs,opts", [
    ([300], [5000], dict()),                                     # pairs of CTAs
    ([700, 90], [900, 4000], dict(hq=16, d=128)),                # two row tiles per CTA
    ([300], [3000], dict(hq=16, d=64, dtype=torch.float16, page=16)),
    ([20, 13], [3000, 21], dict()),                              # one row tile
    ([4, 1], [41000, 5003], dict(hq=48, hk=8)),                  # few rows on the tensor-memory kernel
    ([2, 1], [50000, 41], dict(hq=24, hk=8, d=128, page=48)),
    ([4, 1], [3000, 70], dict()),                                # and on mma.sync
])
def test_paged_attention_ends_when_a_wait_runs_out(lens, seqs, opts):
    """With no patience at all the first wait that is not over ends the launch: it flags that, leaves
    nothing in flight, and the next launch is as ever."""
    from oscar_b200 import kernels

    dev = need_gpu()
    q, kc, vc, table, qsl, scale = make_call(lens, seqs, opts)
    want, lse = kernels.paged_attention(q, kc, vc, table, qsl, seqs, scale)
    assert kernels.device_error(dev) == 0
    for _ in range(3):
        try:
            kernels.set_wait_limit(0)
            for _ in range(4):
                kernels.paged_attention(q, kc, vc, table, qsl, seqs, scale)
            assert kernels.device_error(dev) == 16
        finally:
            kernels.set_wait_limit()
        got, lse2 = kernels.paged_attention(q, kc, vc, table, qsl, seqs, scale)
        assert torch.equal(got, want) and torch.equal(lse, lse2)
        assert kernels.device_error(dev) == 0


def test_paged_attention_longer_than_a_wait():
    """Waits are limited per step of a pipeline, not per launch: a launch that takes several
    times the limit ends as usual.  (The limit is 8 tries of at most a millisecond; 5e13
    operations take over 30 ms.)"""
    from oscar_b200 import kernels

    dev = need_gpu()
    m, seq = 32768, 81920
    gen = torch.Generator(device="cuda").manual_seed(6)
    kc, vc, table = make_pool(gen, [seq], 128, 4, 256, torch.bfloat16)
    q = randn(gen, m, 24, 256, dtype=torch.bfloat16)
    want, lse = kernels.paged_attention(q, kc, vc, table, [0, m], [seq], 1 / 16)
    try:
        kernels.set_wait_limit(8)
        got, lse2 = kernels.paged_attention(q, kc, vc, table, [0, m], [seq], 1 / 16)
        assert kernels.device_error(dev) == 0
    finally:
        kernels.set_wait_limit()
    assert torch.equal(got, want) and torch.equal(lse, lse2)
    # the first and last tokens against 64 bits
    for t0 in (0, m - 4):
        n = seq - m + t0 + 4
        rows = attention64(q[t0:t0 + 4], kc, vc, table, [4], [n], 1 / 16)
        check_attention(q, want[t0:t0 + 4], lse[t0:t0 + 4], rows, [n])


def test_calls_run_on_the_device_of_their_tensors(monkeypatch):
    """With another device current, every call makes the tensors' device current around its work.  (The
    other device is pretended: one is enough, and nothing is ever launched on a wrong one.)"""
    from oscar_b200 import kernels

    need_gpu()
    current, entered = [1], []

    class Device:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            entered.append(self.index)
            self.before, current[0] = current[0], self.index

        def __exit__(self, *exc):
            current[0] = self.before

    q, kc, vc, table, qsl, scale = make_call([2], [300], dict())
    w = torch.zeros(kc.shape[0], 4, 128, device="cuda")
    rope = make_rope(2, dict())
    calls = [lambda: kernels.paged_attention(q, kc, vc, table, qsl, [300], scale)[0],
             lambda: kernels.qk_norm_rope(*rope[:2], None, *rope[3:5], 1e-6, *rope[5:7])[0],
             lambda: kernels.evict_cache(kc, vc, w, table, [300], 300)]
    want = [call() for call in calls]
    monkeypatch.setattr(kernels, "_current_device", lambda: current[0])
    monkeypatch.setattr(torch.cuda, "device", Device)
    for call, x in zip(calls, want):
        entered.clear()
        assert torch.equal(call(), x)
        assert entered == [0] and current == [1]
        current[0] = 0
        assert torch.equal(call(), x) and entered == [0]
        current[0] = 1


WEIGHT_CASES = [
    ([1], [1000], None, dict()),
    ([4, 1, 0, 2], [2000, 65, 70, 1], None, dict()),
    ([4, 3], [700, 90], 2, dict(hq=24, hk=4, d=128, dtype=torch.float16, page=48)),
    ([5], [3], None, dict(hq=8, hk=2, d=64, page=16)),
    ([150, 1], [700, 300], None, dict()),
    ([300], [300], 64, dict(hq=12, hk=2, d=128, page=16)),
    ([90, 64], [1200, 64], 17, dict(hq=8, hk=1, d=64, dtype=torch.float16, page=5)),
    ([40], [30], None, dict()),
    ([4, 2, 1], [40007, 300, 64], None, dict(hq=48, hk=8)),
    ([2], [45000], 1, dict(hq=24, hk=8, d=128, dtype=torch.float16, page=16)),
    ([20, 1], [700, 500], 3, dict()),
]


@pytest.mark.parametrize("lens,seqs,observe,opts", WEIGHT_CASES)
def test_key_weights(lens, seqs, observe, opts):
    from oscar_b200 import kernels

    dev = need_gpu()
    q, kc, vc, table, qsl, scale = make_call(lens, seqs, opts)
    nb, page, hk = kc.shape[:3]
    gen = torch.Generator(device="cuda").manual_seed(4)
    start = torch.rand(nb, hk, page, generator=gen, device="cuda")
    weights = start.clone()
    out, lse = kernels.paged_attention(q, kc, vc, table, qsl, seqs, scale, weights=weights, observe=observe)
    want = attention64(q, kc, vc, table, lens, seqs, scale, observe)
    check_attention(q, out, lse, want, seqs)
    plain, _ = kernels.paged_attention(q, kc, vc, table, qsl, seqs, scale)
    assert torch.equal(out, plain)
    touched = torch.zeros(nb, page, dtype=torch.bool, device="cuda")
    for r, (m, seq) in enumerate(zip(lens, seqs)):
        if m == 0:
            continue
        p = torch.arange(seq, device="cuda")
        blk, off = table[r].long()[p // page], p % page
        touched[blk, off] = True
        old = torch.where(p < seq - m, start[blk, :, off].T.double(), 0.0)
        mass = want[3][r]
        got = weights[blk, :, off].T.double()
        assert ((got - old - mass).abs() <= 2 * SCORE * mass + 2.0**-23 * (old + mass)).all()
    untouched = ~touched[:, None, :].expand_as(weights)
    assert torch.equal(weights[untouched], start[untouched])
    assert kernels.device_error(dev) == 0


@pytest.mark.parametrize("weighted", [False, True])
@pytest.mark.parametrize("lens,seqs", [([3, 2], [700, 90]), ([20], [500]), ([150, 300], [700, 300])])
def test_out_in_place_of_the_queries(lens, seqs, weighted):
    """The attended rows may replace the queries, also where the keys' weights read those again;
    a buffer that meets them elsewhere is as good."""
    from oscar_b200 import kernels

    need_gpu()
    q, kc, vc, table, qsl, scale = make_call(lens, seqs, dict())
    weights = [torch.zeros(kc.shape[0], 4, 128, device="cuda") if weighted else None for _ in range(3)]
    want, lse = kernels.paged_attention(q, kc, vc, table, qsl, seqs, scale, weights=weights[0])
    n = q.shape[0]
    over = torch.empty(n + 7, 24, 256, dtype=q.dtype, device="cuda")
    for (query, out), w in zip(((over[:n], over[:n]), (over[:n], over[7:])), weights[1:]):
        query.copy_(q)
        got, lse2 = kernels.paged_attention(query, kc, vc, table, qsl, seqs, scale, weights=w, out=out)
        assert got.data_ptr() == out.data_ptr() and torch.equal(got, want) and torch.equal(lse, lse2)
        assert w is None or torch.equal(w, weights[0])


@pytest.mark.parametrize("lens,seqs,observe,opts", [
    # together beyond what a launch stores: several launches
    ([8] * 5, [150000, 140001, 9, 170000, 64], None, dict(hq=32, hk=8, d=64, page=64)),
    # each alone beyond it: scores computed again
    ([4, 1, 4], [270000, 100, 262145], 1, dict(hq=64, hk=8, d=64, page=64)),
])
def test_key_weights_of_more_scores_than_are_stored(lens, seqs, observe, opts):
    from oscar_b200 import kernels

    dev = need_gpu()
    q, kc, vc, table, qsl, scale = make_call(lens, seqs, opts)
    nb, page, hk = kc.shape[:3]
    weights = torch.zeros(nb, hk, page, device="cuda")
    out, lse = kernels.paged_attention(q, kc, vc, table, qsl, seqs, scale, weights=weights, observe=observe)
    want = attention64(q, kc, vc, table, lens, seqs, scale, observe)
    check_attention(q, out, lse, want, seqs)
    for r, seq in enumerate(seqs):
        p = torch.arange(seq, device="cuda")
        mass = want[3][r]
        got = weights[table[r].long()[p // page], :, p % page].T.double()
        assert ((got - mass).abs() <= 2 * SCORE * mass + 2.0**-23 * mass).all()
    assert kernels.device_error(dev) == 0


def test_key_weights_of_shared_history_add_up():
    from oscar_b200 import kernels

    need_gpu()
    lens, seqs = [1, 1], [200, 200]
    q, kc, vc, table, qsl, scale = make_call(lens, seqs, dict(page=64))
    table[1, :3] = table[0, :3]  # 192 tokens of shared prefix
    weights = torch.zeros(kc.shape[0], 4, 64, device="cuda")
    kernels.paged_attention(q, kc, vc, table, qsl, seqs, scale, weights=weights)
    masses = attention64(q, kc, vc, table, lens, seqs, scale)[3]
    p = torch.arange(192, device="cuda")
    got = weights[table[0].long()[p // 64], :, p % 64].T.double()
    want = masses[0][:, :192] + masses[1][:, :192]
    assert ((got - want).abs() <= 2 * SCORE * want + 2.0**-23).all()


# ---------------------------------------------------------------------------
def rope64(x, w, offset, eps, cos_sin, positions, interleaved):
    x = x.double()
    rot = cos_sin.shape[1]
    y = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * (w.double() + offset)
    first = torch.arange(0, rot, 2) if interleaved else torch.arange(rot // 2)
    second = first + (1 if interleaved else rot // 2)
    row = cos_sin.double()[positions][:, None]
    c, s = row[..., :rot // 2], row[..., rot // 2:]
    z = y.clone()
    z[..., first] = c * y[..., first] - s * y[..., second]
    z[..., second] = s * y[..., first] + c * y[..., second]
    reach = y.abs().amax(-1, keepdim=True)
    return z, reach


def check_rows(got, want, reach, dtype):
    assert ((got.double() - want).abs() <= U[dtype] * want.abs() * 1.001 + 4e-6 * reach + 2.0**-25).all()


ROPE_CASES = [
    (1, dict()), (32, dict()), (1237, dict(hq=16, hk=2, d=128, rot=128, interleaved=True, dtype=torch.float16, offset=0.0)),
    (7, dict(hq=5, hk=1, d=64, rot=16)), (65, dict(hq=8, hk=8, d=64, rot=64, dtype=torch.float16)),
    (33, dict(hq=3, hk=3, d=128, rot=48, w_dtype=torch.float32, table_dtype=torch.bfloat16)),
    (100, dict(rot=256)), (100, dict(rot=128, interleaved=True)), (511, dict(hq=6, hk=1, rot=64, page=16)),
]


def make_rope(n, opts, seed=3):
    o = dict(hq=24, hk=4, d=256, rot=64, dtype=torch.bfloat16, interleaved=False, offset=1.0, page=128, w_dtype=None,
             table_dtype=torch.float32)
    o.update(opts)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt, d = o["dtype"], o["d"]
    qkv = randn(gen, n, o["hq"] + 2 * o["hk"], d, dtype=dt)
    q, k, v = qkv.split([o["hq"], o["hk"], o["hk"]], dim=1)
    wq, wk = (randn(gen, d).mul(0.1).add(1 - o["offset"]).to(o["w_dtype"] or dt) for _ in range(2))
    angle = torch.arange(500, device="cuda", dtype=torch.float64)[:, None] * 1e4 ** (
        -torch.arange(0, o["rot"], 2, device="cuda", dtype=torch.float64) / o["rot"])
    cos_sin = torch.cat([angle.cos(), angle.sin()], -1).to(o["table_dtype"])
    positions = torch.randint(0, 500, (n,), generator=gen, device="cuda")
    return q, k, v, wq, wk, cos_sin, positions, o, gen


@pytest.mark.parametrize("n,opts", ROPE_CASES)
@pytest.mark.parametrize("layout", ["plain", "halves", "heads"])
def test_qk_norm_rope(n, opts, layout):
    from oscar_b200 import kernels

    dev = need_gpu()
    q, k, v, wq, wk, cos_sin, positions, o, gen = make_rope(n, opts)
    page, hk, d, dt = o["page"], o["hk"], o["d"], o["dtype"]
    blocks = -(-n // page) + 2
    kc, vc, _ = make_pool(gen, [0], page, hk, d, dt, spare=blocks, layout=layout, poison=False)
    k0, v0 = kc.clone(), vc.clone()
    slots = torch.randperm(blocks * page, generator=gen, device="cuda")[:n]
    slots[::5] = -1
    kw = dict(weight_offset=o["offset"], interleaved=o["interleaved"])
    oq, ok = kernels.qk_norm_rope(q, k, v, wq, wk, 1e-6, cos_sin, positions, k_cache=kc, v_cache=vc, slot_mapping=slots, **kw)
    assert ok is None
    wantq, reachq = rope64(q, wq, o["offset"], 1e-6, cos_sin, positions, o["interleaved"])
    wantk, reachk = rope64(k, wk, o["offset"], 1e-6, cos_sin, positions, o["interleaved"])
    check_rows(oq, wantq, reachq, dt)
    oq2, ok2 = kernels.qk_norm_rope(q, k, None, wq, wk, 1e-6, cos_sin, positions.int(), **kw)
    assert torch.equal(oq, oq2)
    check_rows(ok2, wantk, reachk, dt)
    live = slots >= 0
    k0[slots[live] // page, slots[live] % page] = ok2[live]
    v0[slots[live] // page, slots[live] % page] = v[live]
    assert torch.equal(kc, k0) and torch.equal(vc, v0)
    # in place, and keys returned beside the cache write
    qc, kk = q.clone(), k.clone()
    kernels.qk_norm_rope(qc, kk, v, wq, wk, 1e-6, cos_sin, positions, k_cache=kc, v_cache=vc, slot_mapping=slots,
                         out_q=qc, out_k=kk, **kw)
    assert torch.equal(qc, oq) and torch.equal(kk, ok2)
    assert kernels.device_error(dev) == 0


def test_qk_norm_rope_weights_and_tables_at_any_place():
    """Views that begin between the 16-byte boundaries, and one row of the table for all positions."""
    from oscar_b200 import kernels

    need_gpu()
    q, k, v, wq, wk, cos_sin, positions, o, gen = make_rope(6, dict())

    def odd(t, by):
        flat = torch.zeros(t.numel() + by, dtype=t.dtype, device="cuda")[by:]
        return flat.view(t.shape).copy_(t)

    want = kernels.qk_norm_rope(q, k, None, wq, wk, 1e-6, cos_sin, positions)
    got = kernels.qk_norm_rope(q, k, None, odd(wq, 1), odd(wk, 3), 1e-6, odd(cos_sin, 1), positions)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    wide = torch.zeros(500, 72, device="cuda")
    wide[:, 5:69] = cos_sin
    got = kernels.qk_norm_rope(q, k, None, wq, wk, 1e-6, wide[:, 5:69], positions)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    same = torch.full_like(positions, 7)
    want = kernels.qk_norm_rope(q, k, None, wq, wk, 1e-6, cos_sin, same)
    got = kernels.qk_norm_rope(q, k, None, wq, wk, 1e-6, cos_sin[7:8].expand(500, -1), positions)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_block_tables_of_any_strides():
    """An expanded row (requests with all their pages in common), one row at a stride of its own, columns."""
    from oscar_b200 import kernels

    need_gpu()
    q, kc, vc, table, qsl, scale = make_call([1, 1, 1], [300, 300, 300], dict(page=64))
    shared = table[:1].repeat(3, 1)
    want, lse = kernels.paged_attention(q, kc, vc, shared, qsl, [300] * 3, scale)
    for t in (table[:1].expand(3, -1), shared.t().contiguous().t(), shared.long(), torch.stack([shared, shared], 2)[..., 1]):
        got, lse2 = kernels.paged_attention(q, kc, vc, t, qsl, [300] * 3, scale)
        assert torch.equal(got, want) and torch.equal(lse, lse2)
    one = shared.as_strided((1, shared.shape[1]), (0, 1))
    got, _ = kernels.paged_attention(q[:1], kc, vc, one, [0, 1], [300], scale)
    again, _ = kernels.paged_attention(q[:1], kc, vc, shared, [0, 1], [300], scale)
    assert torch.equal(got, again)
    gen = torch.Generator(device="cuda").manual_seed(16)
    w = torch.rand(kc.shape[0], 4, 64, generator=gen, device="cuda")
    k2, v2, w2 = kc.clone(), vc.clone(), w.clone()
    a = kernels.evict_cache(kc, vc, w, shared[:1], [300], 100)
    b = kernels.evict_cache(k2, v2, w2, one, [300], 100)
    assert torch.equal(a, b) and torch.equal(w, w2)
    # (slots past the request hold NaN)
    assert torch.equal(kc.view(torch.int16), k2.view(torch.int16)) and torch.equal(vc.view(torch.int16), v2.view(torch.int16))


@pytest.mark.parametrize("n", [1, 5])
def test_qk_norm_rope_output_layouts(n):
    """Outputs with heads before tokens, and one token at a stride of its own."""
    from oscar_b200 import kernels

    need_gpu()
    q, k, v, wq, wk, cos_sin, positions, o, gen = make_rope(n, dict())
    want_q, want_k = kernels.qk_norm_rope(q, k, None, wq, wk, 1e-6, cos_sin, positions)
    oq = torch.zeros(24, n, 256, dtype=q.dtype, device="cuda").transpose(0, 1)
    ok = torch.zeros(4, n, 256, dtype=q.dtype, device="cuda").transpose(0, 1)
    got_q, got_k = kernels.qk_norm_rope(q, k, None, wq, wk, 1e-6, cos_sin, positions, out_q=oq, out_k=ok)
    assert got_q.data_ptr() == oq.data_ptr() and torch.equal(oq, want_q) and torch.equal(ok, want_k)
    with pytest.raises(ValueError, match="overlap"):
        kernels.qk_norm_rope(q, k, None, wq, wk, 1e-6, cos_sin, positions, out_q=oq[:, :1].expand(n, 24, 256))


def test_qk_norm_rope_extremes():
    """Zero heads stay zero, an inf or NaN stays in its head, no tokens is no work."""
    from oscar_b200 import kernels

    need_gpu()
    q, k, v, wq, wk, cos_sin, positions, o, _ = make_rope(4, dict())
    q = q.clone()
    q[0, 0] = 0
    q[1, 1, 7] = math.nan
    q[2, 2] = 1e4
    oq, _ = kernels.qk_norm_rope(q, k, None, wq, wk, 1e-6, cos_sin, positions, weight_offset=1.0)
    assert (oq[0, 0] == 0).all() and torch.isnan(oq[1, 1]).all()
    rest = torch.ones(4, 24, dtype=torch.bool, device="cuda")
    rest[1, 1] = False
    assert torch.isfinite(oq[rest]).all()
    empty, _ = kernels.qk_norm_rope(q[:0], k[:0], None, wq, wk, 1e-6, cos_sin, positions[:0])
    assert empty.shape == (0, 24, 256)


def test_qk_norm_rope_flags_bad_positions_and_slots():
    from oscar_b200 import kernels

    dev = need_gpu()
    q, k, v, wq, wk, cos_sin, positions, o, gen = make_rope(6, dict())
    kc, vc, _ = make_pool(gen, [0], 128, 4, 256, torch.bfloat16, spare=1, poison=False)
    k0 = kc.clone()
    positions[2] = 500
    positions[3] = -1
    slots = torch.tensor([-1, 128, 2, 3, -1, -1], device="cuda")
    kernels.qk_norm_rope(q, k, v, wq, wk, 1e-6, cos_sin, positions, k_cache=kc, v_cache=vc, slot_mapping=slots)
    assert kernels.device_error(dev) == 64 | 1
    assert torch.equal(kc, k0)


# ---------------------------------------------------------------------------
def kept64(w, keep, sink, recent):
    """Kept positions of one head: numpy, stable, NaN above every number."""
    n = w.size
    if n <= keep:
        return np.arange(n)
    mid = np.arange(sink, n - recent)
    rank = np.where(np.isnan(w[mid]), np.inf, w[mid].astype(np.float64))
    nan_first = ~np.isnan(w[mid])
    order = mid[np.lexsort((mid, -rank, nan_first))]
    return np.sort(np.concatenate([np.arange(sink), order[:keep - sink - recent], np.arange(n - recent, n)]))


EVICT_CASES = [
    ([300], 100, 4, 10, dict()),
    ([300, 20, 1000, 0, 101], 100, 0, 0, dict(page=16)),
    ([5000, 4097, 4096], 4096, 64, 256, dict(hk=1)),
    ([2500], 50, 25, 25, dict(hk=2, d=64, page=5, dtype=torch.float16)),     # nothing between sink and recent
    ([777], 1, 0, 0, dict(hk=8, d=64, page=1)),
    ([777], 776, 0, 1, dict(d=128, page=48, dtype=torch.float16)),
    ([60000], 33000, 10, 100, dict(hk=1, d=64, page=64)),
    ([150000, 300], 77000, 10, 100, dict(hk=1, d=64, page=64)),              # more keys than shared memory holds
]


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("values", ["spread", "ties", "zero", "signed"])
@pytest.mark.parametrize("seqs,keep,sink,recent,opts", EVICT_CASES)
def test_evict_cache(seqs, keep, sink, recent, opts, values, in_place):
    from oscar_b200 import kernels

    dev = need_gpu()
    o = dict(hk=4, d=256, dtype=torch.bfloat16, page=128)
    o.update(opts)
    page, hk = o["page"], o["hk"]
    gen = torch.Generator(device="cuda").manual_seed(11)
    fresh = [-(-min(s, keep) // page) for s in seqs]
    kc, vc, table = make_pool(gen, seqs, page, hk, o["d"], o["dtype"], spare=sum(fresh) + 1, poison=False)
    nb = kc.shape[0]
    w = torch.rand(nb, hk, page, generator=gen, device="cuda")
    if values == "ties":
        w = (w * 4).floor() / 4
    elif values == "zero":
        w = torch.zeros_like(w)
    elif values == "signed":
        w = w - 0.5
        w[torch.rand(w.shape, generator=gen, device="cuda") < 0.02] = math.nan
        w[torch.rand(w.shape, generator=gen, device="cuda") < 0.02] = -0.0
        w[torch.rand(w.shape, generator=gen, device="cuda") < 0.02] = math.inf
    dst = None
    to = table
    if not in_place:
        used = set(int(x) for r, s in enumerate(seqs) for x in table[r, :-(-s // page)].tolist())
        rest = [b for b in range(nb) if b not in used]
        dst = torch.full((len(seqs), max(fresh) + 1), -1, dtype=torch.int32, device="cuda")
        for r, n in enumerate(fresh):
            dst[r, :n] = torch.tensor([rest.pop() for _ in range(n)], dtype=torch.int32)
        to = dst
    k0, v0, w0 = kc.clone(), vc.clone(), w.clone()
    kept = kernels.evict_cache(kc, vc, w, table, seqs, keep, sink=sink, recent=recent, dst_table=dst)
    assert kept.shape == (len(seqs), hk, min(keep, max(seqs)))
    wk, wv, ww = k0.clone(), v0.clone(), w0.clone()
    for r, seq in enumerate(seqs):
        n = min(seq, keep)
        p = torch.arange(seq, device="cuda")
        blk, off = table[r].long()[p // page], p % page
        j = torch.arange(n, device="cuda")
        tb, tf = to[r].long()[j // page], j % page
        for h in range(hk):
            c = torch.from_numpy(kept64(w0[blk, h, off].cpu().numpy(), keep, sink, recent)).cuda()
            assert torch.equal(kept[r, h, :n].long(), c)
            assert (kept[r, h, n:] == -1).all()
            wk[tb, tf, h] = k0[blk[c], off[c], h]
            wv[tb, tf, h] = v0[blk[c], off[c], h]
            ww[tb, h, tf] = w0[blk[c], h, off[c]]
    assert torch.equal(kc, wk) and torch.equal(vc, wv)
    assert torch.equal(w.view(torch.int32), ww.view(torch.int32))
    assert kernels.device_error(dev) == 0


def test_evict_equal_weights_in_many_requests():
    """All keys weigh the same: the range of the weights is one value, and the CTAs that share a
    request go straight from its exchange to that of the counts."""
    from oscar_b200 import kernels

    dev = need_gpu()
    gen = torch.Generator(device="cuda").manual_seed(12)
    for base in (33, 300, 2000):
        seqs = [base + 7 * r for r in range(48)]
        keep = base // 2
        kc, vc, table = make_pool(gen, seqs, 16, 4, 64, torch.bfloat16, poison=False)
        for value in (0.0, 1.5, math.nan):
            for _ in range(3):
                w = torch.full((kc.shape[0], 4, 16), value, device="cuda")
                kept = kernels.evict_cache(kc, vc, w, table, seqs, keep, sink=2, recent=5)
                for r, seq in enumerate(seqs):
                    want = list(range(keep - 5)) + list(range(seq - 5, seq))
                    assert kept[r].tolist() == [want] * 4
    assert kernels.device_error(dev) == 0


@pytest.mark.parametrize("in_place", [True, False])
def test_evict_ends_while_another_stream_writes_the_weights(in_place):
    """A caller's mistake: more keys than shared memory holds are read again in each round, here from
    weights that change meanwhile.  What stays is then undefined, but the call ends, lists positions
    of the request in order and moves nothing else."""
    from oscar_b200 import kernels

    dev = need_gpu()
    gen = torch.Generator(device="cuda").manual_seed(13)
    seq, keep, page = 300000, 120000, 64
    fresh = -(-keep // page)
    kc, vc, table = make_pool(gen, [seq], page, 1, 64, torch.bfloat16, spare=fresh, poison=False)
    nb = kc.shape[0]
    used = torch.zeros(nb, dtype=torch.bool, device="cuda")
    used[table[0, :-(-seq // page)].long()] = True
    dst = None if in_place else (~used).nonzero().flatten().to(torch.int32)[None, :fresh].contiguous()
    w = torch.rand(nb, 1, page, generator=gen, device="cuda")
    spare_k = kc[~used].clone()
    side = torch.cuda.Stream()
    lists = []
    torch.cuda.synchronize()
    for scale in (1.0, 1e6, 1e-6, 1.0, 1e3, 1e-3):
        with torch.cuda.stream(side):
            for _ in range(20):
                w.uniform_().mul_(scale)
                w.neg_()
        for _ in range(4):
            lists.append(kernels.evict_cache(kc, vc, w, table, [seq], keep, sink=5, recent=9, dst_table=dst))
        torch.cuda.synchronize()
    for kept in lists:
        kept = kept.flatten()
        there = kept[kept >= 0]
        assert (there[1:] > there[:-1]).all() and there[-1] < seq and (kept[there.numel():] == -1).all()
    if in_place:
        assert torch.equal(kc[~used], spare_k)
    assert kernels.device_error(dev) == 0


@pytest.mark.parametrize("kind", [torch.int32, torch.int64])
def test_evict_to_the_table_it_came_from_is_in_place(kind):
    from oscar_b200 import kernels

    need_gpu()
    gen = torch.Generator(device="cuda").manual_seed(14)
    seqs = [9000, 20000]
    kc, vc, table = make_pool(gen, seqs, 32, 4, 128, torch.bfloat16, poison=False)
    w = torch.rand(kc.shape[0], 4, 32, generator=gen, device="cuda")
    k2, v2, w2 = kc.clone(), vc.clone(), w.clone()
    table = table.to(kind)
    a = kernels.evict_cache(kc, vc, w, table, seqs, 7000, sink=3, recent=7)
    b = kernels.evict_cache(k2, v2, w2, table, seqs, 7000, sink=3, recent=7, dst_table=table)
    assert torch.equal(a, b) and torch.equal(kc, k2) and torch.equal(vc, v2) and torch.equal(w, w2)


def test_evict_limits_past_32_bits_keep_everything():
    from oscar_b200 import kernels

    need_gpu()
    gen = torch.Generator(device="cuda").manual_seed(15)
    kc, vc, table = make_pool(gen, [500, 9], 32, 2, 64, torch.bfloat16, poison=False)
    w = torch.rand(kc.shape[0], 2, 32, generator=gen, device="cuda")
    k0, w0 = kc.clone(), w.clone()
    for keep, sink, recent in ((2**32 + 100, 2**32 + 1, 3), (2**31, 0, 2**31), (2**40, 64, 256), (501, 400, 101)):
        kept = kernels.evict_cache(kc, vc, w, table, [500, 9], keep, sink=sink, recent=recent)
        assert kept[0, 0].tolist() == list(range(500)) and kept[1, 1].tolist() == list(range(9)) + [-1] * 491
        assert torch.equal(kc, k0) and torch.equal(w, w0)
    with pytest.raises(ValueError, match="keep"):
        kernels.evict_cache(kc, vc, w, table, [500, 9], 2**32, sink=2**32, recent=1)


def test_lists_past_32_bits_are_refused():
    from oscar_b200 import kernels

    need_gpu()
    q, kc, vc, table, qsl, scale = make_call([2], [300], dict())
    w = torch.zeros(kc.shape[0], 4, 128, device="cuda")
    for seqs in (np.array([2**32 + 300]), torch.tensor([2**32 + 300]), np.array([300.5])):
        with pytest.raises(ValueError, match="32 bits"):
            kernels.paged_attention(q, kc, vc, table, qsl, seqs, scale)
        with pytest.raises(ValueError, match="32 bits"):
            kernels.evict_cache(kc, vc, w, table, seqs, 100)
    want, _ = kernels.paged_attention(q, kc, vc, table, qsl, [300], scale)
    got, _ = kernels.paged_attention(q, kc, vc, table, torch.from_numpy(qsl).long(), np.array([300]), scale)
    assert torch.equal(got, want)


def test_evict_strided_caches():
    from oscar_b200 import kernels

    need_gpu()
    gen = torch.Generator(device="cuda").manual_seed(1)
    kc, vc, table = make_pool(gen, [500, 300], 32, 2, 128, torch.bfloat16, layout="halves", poison=False)
    plain_k, plain_v = kc.contiguous(), vc.contiguous()
    w = torch.rand(kc.shape[0], 2, 32, generator=gen, device="cuda")
    w2 = w.clone()
    a = kernels.evict_cache(kc, vc, w, table, [500, 300], 200, sink=3, recent=7)
    b = kernels.evict_cache(plain_k, plain_v, w2, table, [500, 300], 200, sink=3, recent=7)
    assert torch.equal(a, b) and torch.equal(kc, plain_k) and torch.equal(vc, plain_v) and torch.equal(w, w2)


def test_offsets_past_32_bits():
    """The used pages lie past 2^31 elements of the caches."""
    from oscar_b200 import kernels

    dev = need_gpu()
    page, hk, d = 128, 4, 256
    nb = 2**31 // (page * hk * d) + 40
    kc, vc = (torch.empty(nb, page, hk, d, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    w = torch.zeros(nb, hk, page, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(2)
    table = (nb - 1 - torch.arange(16, device="cuda", dtype=torch.int32))[None].contiguous()
    small_table = torch.arange(15, -1, -1, device="cuda", dtype=torch.int32)[None].contiguous()
    for lens, seq in (([3], 1999), ([200], 1999)):
        kc[-16:] = randn(gen, 16, page, hk, d, dtype=torch.bfloat16)
        vc[-16:] = randn(gen, 16, page, hk, d, dtype=torch.bfloat16)
        q = randn(gen, lens[0], 24, d, dtype=torch.bfloat16)
        sk, sv, sw = kc[-16:].clone(), vc[-16:].clone(), torch.zeros(16, hk, page, device="cuda")
        w.zero_()
        out, lse = kernels.paged_attention(q, kc, vc, table, [0, lens[0]], [seq], d**-0.5, weights=w)
        want, lse2 = kernels.paged_attention(q, sk, sv, small_table, [0, lens[0]], [seq], d**-0.5, weights=sw)
        assert torch.equal(out, want) and torch.equal(lse, lse2) and torch.equal(w[-16:], sw)
        a = kernels.evict_cache(kc, vc, w, table, [seq], 700, sink=4, recent=64)
        b = kernels.evict_cache(sk, sv, sw, small_table, [seq], 700, sink=4, recent=64)
        assert torch.equal(a, b) and torch.equal(kc[-16:], sk) and torch.equal(vc[-16:], sv)
    q, k, v, wq, wk, cos_sin, positions, o, gen = make_rope(9, dict())
    slots = nb * page - 1 - torch.arange(9, device="cuda")
    _, ok = kernels.qk_norm_rope(q, k, None, wq, wk, 1e-6, cos_sin, positions)
    kernels.qk_norm_rope(q, k, v, wq, wk, 1e-6, cos_sin, positions, k_cache=kc, v_cache=vc, slot_mapping=slots)
    assert torch.equal(kc.view(-1, hk, d)[slots], ok) and torch.equal(vc.view(-1, hk, d)[slots], v)
    assert kernels.device_error(dev) == 0
