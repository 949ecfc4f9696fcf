"""Paged key/value cache, the attention over it and the verification of drafted tokens, against the plain 64-bit forms of
oracle/paged_oracle.py.

Tolerances.  Codes, scales, copies, counts and tokens are equal.  Attention: P is rounded to bf16 for its product with V (half a
step, 2^-8 of each term) and the result to bf16 (2^-8 of it); scores are fp32 sums of D <= 128 exact products, off by at
most D 2^-24 sum |q k| c, some 128 * 6e-8 * 12 = 9e-5 for the standard normal rows here (sum |q k| / sqrt(D) has mean 0.64 sqrt(D) = 7.2),
which enters a probability's numerator and its denominator: 4e-4 with the exponential's own error.  So
|o - o64| <= 2^-8 |o64| + (2^-8 + 4e-4) sum p |v|, and |lse - lse64| <= 2e-4 (+ 2^-23 |lse64|)."""
import math
import random

import pytest
import torch

from fgrpo import ops
from oracle import paged_oracle as PO

pytestmark = pytest.mark.gpu
FP8 = torch.float8_e4m3fn


def _table(lens, block, width, pages, rng):
    order = list(range(pages))
    rng.shuffle(order)
    table = torch.full((len(lens), width), -1, dtype=torch.int32)
    for b, n in enumerate(lens):
        for i in range((n + block - 1) // block):
            table[b, i] = order.pop()
    return table


def _batch(qs, ks, Hq, Hkv, D, block, fp8, seed, tail=3, spare=2, nan=True, reach=0):
    """A batch on the CPU: packed queries with ``tail`` rows behind the last sequence, and a cache whose unused places are NaN.
    ``reach``: tokens that the table has room for at least.  What a call is divided by goes by that and by ``max_len``."""
    g, rng = torch.Generator().manual_seed(seed), random.Random(seed)
    need = [(n + block - 1) // block for n in ks]
    pages, width = sum(need) + spare, max(max(need + [0]) + 1, reach // block)
    table = _table(ks, block, width, pages, rng)
    cu = torch.tensor([0] + torch.tensor(qs).cumsum(0).tolist(), dtype=torch.int32)
    lens = torch.tensor(ks, dtype=torch.int32)
    T = int(cu[-1]) + tail
    q = torch.randn(T, Hq, D, generator=g).bfloat16()
    shape = (pages, block, Hkv, D)
    caches = []
    for _ in range(2):
        x = torch.randn(shape, generator=g).bfloat16()
        if nan:
            used = torch.zeros(shape[:2], dtype=torch.bool)
            for b, n in enumerate(ks):
                for j in range(n):
                    used[PO.place(table, b, j, block)] = True
            x[~used] = math.nan
        if fp8:
            code, s = PO.quantise(x)
            if nan:
                s = torch.where(used[..., None], s, torch.full((), math.nan))
            caches.append((code, s))
        else:
            caches.append((x, None))
    return dict(q=q, k=caches[0], v=caches[1], table=table, lens=lens, cu=cu, block=block, T=T, rows=int(cu[-1]))


def _cache(s, dev):
    (k, ks), (v, vs) = s["k"], s["v"]
    to = lambda t: None if t is None else t.to(dev)      # noqa: E731
    return ops.PagedCache(to(k), to(v), to(ks), to(vs))


def _check(s, out, lse, causal=True, scale=None, hq=None):
    want, wl, size = PO.attention(s["q"], PO.held(*s["k"]), PO.held(*s["v"]), s["table"], s["lens"], s["cu"], s["block"], scale, causal)
    n = s["rows"]
    got = out.cpu().double()[:n]
    assert torch.isfinite(got).all()
    over = (got - want[:n]).abs() - (2.0 ** -8 * want[:n].abs() + (2.0 ** -8 + 4e-4) * size[:n])
    assert float(over.max() if over.numel() else 0.0) <= 0, f"off by {float(over.max())} more than allowed"
    if lse is not None:
        a, b = lse.cpu().double()[:, :n], wl[:, :n]
        none = torch.isinf(b)
        assert torch.equal(none, torch.isinf(a)) and (a[none] < 0).all()
        assert ((a - b).abs()[~none] <= 2e-4 + 2.0 ** -23 * b.abs()[~none]).all()


SHAPES = [
    # new tokens, keys with them: single tokens, around tiles and pages, rows that see nothing, empty sequences
    ([1], [1]),
    ([1, 1, 1, 1, 1], [1, 15, 16, 17, 1000]),
    ([1, 0, 1, 3], [0, 5, 64, 2]),
    ([2, 5, 1, 8], [63, 64, 65, 300]),
    ([40, 1, 0, 130], [40, 700, 0, 129]),
    ([257], [257]),
    ([20, 33], [500, 1111]),
]


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("Hq,Hkv,D", [(12, 2, 128), (14, 2, 64), (5, 5, 128), (10, 2, 64), (33, 1, 128)])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_attention_over_the_cache(dev, shape, Hq, Hkv, D, fp8):
    qs, ks = SHAPES[shape]
    block = (16, 64, 32, 256)[shape % 4]
    for causal in (True, False):
        for hint, reach in ((max(qs), 0), (0, 0), (64, 1 << 20)):
            s = _batch(qs, ks, Hq, Hkv, D, block, fp8, seed=shape, reach=reach)
            out = torch.full((s["T"], Hq, D), 7.0, dtype=torch.bfloat16, device=dev)
            got, lse = ops.paged_attention(s["q"].to(dev), _cache(s, dev), s["table"].to(dev), s["lens"].to(dev), s["cu"].to(dev), causal=causal,
                                           max_len=hint, return_lse=True, out=out)
            assert got.data_ptr() == out.data_ptr()
            _check(s, got, lse, causal)
            assert (got[s["rows"]:] == 7.0).all(), "rows behind the last sequence were written"


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("Hq,Hkv,D,qs,ks", [
    # as many tiles as work-groups and a few: whole ones in rounds, the rest in parts
    (12, 2, 128, [700, 690, 711, 705, 650, 730, 700, 680], [1000, 1100, 711, 1205, 650, 900, 1000, 980]),
    # one long sequence among short ones: shares
    (14, 2, 64, [1, 900, 3, 1, 40], [700, 1500, 64, 1, 2000]),
    # a prompt from its start, rows from one key to all
    (8, 1, 128, [1500], [1500])])
def test_attention_of_many_tiles(dev, Hq, Hkv, D, qs, ks, fp8):
    s = _batch(qs, ks, Hq, Hkv, D, 64, fp8, seed=3)
    out, lse = ops.paged_attention(s["q"].to(dev), _cache(s, dev), s["table"].to(dev), s["lens"].to(dev), s["cu"].to(dev), max_len=max(qs), return_lse=True)
    _check(s, out, lse)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("D", [128, 64])
def test_write_then_read(dev, D, fp8):
    Hkv, block = 3, 32
    qs, ks = [1, 40, 0, 5, 9], [1, 40, 70, 300, 4]            # the last has more new rows than tokens: the first five go nowhere
    s = _batch(qs, ks, Hkv, Hkv, D, block, fp8, seed=5, nan=False)
    g = torch.Generator().manual_seed(6)
    new = [torch.randn(s["T"], Hkv, D, generator=g).bfloat16() for _ in range(2)]
    new[0][0, 0] = 0
    new[0][1, 1, 3], new[0][1, 1, 4], new[1][2, 0, 0] = math.inf, math.nan, -math.inf
    new[1][3, 2] = torch.randn(D, generator=g).bfloat16() * 1e-36
    new[1][4, 2] = torch.randn(D, generator=g).bfloat16() * 1e36
    cache = _cache(s, dev)
    ops.paged_cache_write(cache, new[0].to(dev), new[1].to(dev), s["table"].to(dev), s["lens"].to(dev), s["cu"].to(dev))
    for (c, sc), x, got, gs in ((s["k"], new[0], cache.k, cache.k_scale), (s["v"], new[1], cache.v, cache.v_scale)):
        PO.write(c, sc, x, s["table"], s["lens"], s["cu"])
        assert torch.equal(got.cpu().view(torch.uint8) & 0x7F if fp8 else got.cpu().view(torch.int16),
                           c.view(torch.uint8) & 0x7F if fp8 else c.view(torch.int16))
        if fp8:
            a, b = got.cpu().float(), c.float()
            assert torch.equal(a.nan_to_num(), b.nan_to_num()) and torch.equal(gs.cpu(), sc)
    cu_k = torch.tensor([0] + torch.tensor(ks).cumsum(0).tolist(), dtype=torch.int32)
    total = int(cu_k[-1]) + 4
    out = tuple(torch.full((total, Hkv, D), 3.0, dtype=torch.bfloat16, device=dev) for _ in range(2))
    got = ops.paged_cache_read(cache, s["table"].to(dev), s["lens"].to(dev), cu_k.to(dev), total, out=out)
    for (c, sc), x in ((s["k"], got[0]), (s["v"], got[1])):
        vals = c.float() if sc is None else c.float() * sc[..., None]
        want = torch.cat([PO.gather(vals, s["table"], b, n, block) for b, n in enumerate(ks)]).bfloat16()
        assert torch.equal(x.cpu()[:total - 4].nan_to_num(), want.nan_to_num()) and torch.equal(x.cpu()[:total - 4].isnan(), want.isnan())
        assert (x[total - 4:] == 3.0).all()


@pytest.mark.parametrize("fp32", [False, True])
@pytest.mark.parametrize("with_draft", [False, True])
@pytest.mark.parametrize("V", [1, 7, 1000, 4099, 32000])
def test_verify(dev, V, with_draft, fp32):
    g = torch.Generator().manual_seed(V)
    ns = [1, 5, 0, 2, 9, 1, 70]
    cu = torch.tensor([0] + torch.tensor(ns).cumsum(0).tolist(), dtype=torch.int32)
    T, tail, B = int(cu[-1]), 2, len(ns)
    last = torch.zeros(T + tail, dtype=torch.bool)
    last[cu[1:][torch.tensor(ns) > 0].long() - 1] = True
    last[T:] = True
    logits = 2 * torch.randn(T + tail, V, generator=g)
    dt = torch.float32 if fp32 else torch.bfloat16
    target = logits.softmax(-1).to(dt)
    draft = (logits[~last] + torch.randn(T - 6, V, generator=g)).softmax(-1).to(dt) if with_draft else None
    ids = torch.randint(0, V, (T + tail,), generator=g)
    for b in range(B):                                # drafts that often stand
        for i in range(int(cu[b]) + 1, int(cu[b + 1])):
            if torch.rand((), generator=g) < 0.8:
                ids[i] = int(target[i - 1].float().argmax())
                if not with_draft:
                    target[i - 1, ids[i]] = 1.0
    u = torch.rand(T + tail, generator=g)
    u[0], u[T - 1] = 0.0, 1 - 2.0 ** -24
    accepted, tokens = ops.verify_drafts(target.to(dev), None if draft is None else draft.to(dev), ids.to(dev), u.to(dev), cu.to(dev))
    want_a, want_t = PO.verify(target, draft, ids, u, cu)
    assert torch.equal(accepted.cpu(), want_a) and torch.equal(tokens.cpu()[:T], want_t[:T])
