"""The paged cache as it is used: layouts and strides, bad values in device memory, shared and far blocks, many sequences, streams and
captured graphs, the attention callables, and a model that generates with drafts over it.  Tolerances: test_gpu_paged.py."""
import math
import random

import pytest
import torch

from fgrpo import ops
from oracle import paged_oracle as PO
from test_gpu_paged import FP8, _batch, _cache, _check

pytestmark = pytest.mark.gpu


def _dev(s, dev):
    return s["q"].to(dev), s["table"].to(dev), s["lens"].to(dev), s["cu"].to(dev)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("qs,ks", [([3, 1, 40], [70, 33, 41]), ([200, 300], [200, 1000])])
def test_layouts(dev, qs, ks, fp8):
    """Heads in front of tokens in a block, K and V side by side in one allocation, queries inside a wider row, a wider 64-bit table."""
    Hq, Hkv, D, block = 6, 3, 128, 32
    s = _batch(qs, ks, Hq, Hkv, D, block, fp8, seed=11, reach=(1 << 20) * (max(qs) > 64))
    q, table, lens, cu = _dev(s, dev)
    want, wl = ops.paged_attention(q, _cache(s, dev), table, lens, cu, return_lse=True, max_len=max(qs))
    _check(s, want, wl)

    def both(a, b, order):               # [2, ...] in the order given, seen as [blocks, block, heads, D]
        x = torch.stack([a, b]).to(dev)
        inner = x.permute(0, *(1 + i for i in order)).contiguous()
        back = [order.index(i) for i in range(len(order))]
        return [inner[i].permute(*back) for i in range(2)]
    k, v = both(s["k"][0].view(torch.uint8) if fp8 else s["k"][0], s["v"][0].view(torch.uint8) if fp8 else s["v"][0], [2, 0, 1, 3])
    scales = both(s["k"][1], s["v"][1], [0, 2, 1]) if fp8 else []
    cache = ops.PagedCache(k.view(FP8) if fp8 else k, v.view(FP8) if fp8 else v, *scales)
    assert not cache.k.is_contiguous()
    wide = torch.randn(s["T"], Hq + 2 * Hkv, D + 8, device=dev).bfloat16()
    wide[:, :Hq, :D] = q
    table64 = torch.full((len(qs), 2 * table.shape[1]), -7, dtype=torch.int64, device=dev)
    table64[:, :table.shape[1]] = table
    got, gl = ops.paged_attention(wide[:, :Hq, :D], cache, table64[:, :table.shape[1]], lens.long(), cu.long(), return_lse=True, max_len=max(qs))
    n = s["rows"]
    assert torch.equal(got[:n], want[:n]) and torch.equal(gl[:, :n], wl[:, :n])
    new = torch.randn(s["T"], Hkv, 2, D, device=dev).bfloat16()           # K and V of a token's head beside each other
    other = _cache(s, dev)
    ops.paged_cache_write(cache, new[:, :, 0], new[:, :, 1], table64[:, :table.shape[1]], lens, cu)
    ops.paged_cache_write(other, new[:, :, 0].contiguous(), new[:, :, 1].contiguous(), table, lens, cu)
    cu_k = torch.tensor([0] + torch.tensor(ks).cumsum(0).tolist(), dtype=torch.int32, device=dev)
    for a, b in zip(ops.paged_cache_read(cache, table64[:, :table.shape[1]], lens, cu_k, sum(ks)), ops.paged_cache_read(other, table, lens, cu_k, sum(ks))):
        assert torch.equal(a, b)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("n,ks", [(1, (1, 300)), (4, (4, 90)), (0, (0, 200))])
def test_many_sequences(dev, n, ks, fp8):
    """More sequences than lanes, among them empty ones; n = 0: as many new tokens as the sequence's number mod 4."""
    rng = random.Random(n)
    B = 700
    lens = [rng.randint(*ks) for _ in range(B)]
    qs = [n if n else b % 4 for b in range(B)]
    s = _batch(qs, lens, 4, 1, 64, 16, fp8, seed=n, nan=False)
    q, table, ln, cu = _dev(s, dev)
    out, lse = ops.paged_attention(q, _cache(s, dev), table, ln, cu, return_lse=True, max_len=max(qs))
    _check(s, out, lse)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("n,hint", [(1, 1), (1, 500), (5, 1), (5, 0), (150, 1), (150, 5), (150, 2 ** 30)])
def test_one_long_sequence_in_many_parts_and_wrong_hints(dev, n, hint, fp8):
    s = _batch([n], [30001], 12, 2, 128, 64, fp8, seed=n, nan=False, reach=(1 << 20) * (hint > 8))
    q, table, ln, cu = _dev(s, dev)
    out, lse = ops.paged_attention(q, _cache(s, dev), table, ln, cu, return_lse=True, max_len=hint)
    again, _ = ops.paged_attention(q, _cache(s, dev), table, ln, cu, return_lse=True, max_len=hint)
    assert torch.equal(out[:n], again[:n]), "not the same bits twice"
    _check(s, out, lse)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("Hq,Hkv,D,block,qs,ks", [
    (128, 128, 64, 16, [1, 2], [40, 300]),                 # every head its own keys
    (71, 1, 64, 32, [1, 1, 1], [5, 64, 700]),              # more heads of a group than a block has rows
    (8, 2, 64, 65536, [3, 1], [70, 1500]),                 # a block longer than any sequence
    (8, 2, 128, 1024, [2, 90], [1025, 2047])])
def test_head_counts_and_block_sizes(dev, Hq, Hkv, D, block, qs, ks, fp8):
    s = _batch(qs, ks, Hq, Hkv, D, block, fp8, seed=31, spare=0)
    q, table, ln, cu = _dev(s, dev)
    for hint in (max(qs), 0, 500):
        out, lse = ops.paged_attention(q, _cache(s, dev), table, ln, cu, return_lse=True, max_len=hint)
        _check(s, out, lse)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("n", [1, 5, 90])
def test_a_very_long_sequence(dev, n, fp8):
    """1.3 million keys, against 64 bits on the device."""
    L, block, Hq, D = 1300007, 64, 2, 64
    g = torch.Generator(dev).manual_seed(n)
    pages = (L + block - 1) // block
    x = [torch.randn(pages, block, 1, D, generator=g, device=dev).bfloat16() for _ in range(2)]
    if fp8:
        a = [t.float().abs().amax(-1) / 448 for t in x]
        codes = [(t.float() / s[..., None]).to(FP8) for t, s in zip(x, a)]
        cache, held = ops.PagedCache(*codes, *a), [c.float().double() * s.double()[..., None] for c, s in zip(codes, a)]
    else:
        cache, held = ops.PagedCache(*x), [t.double() for t in x]
    order = torch.randperm(pages, generator=g, device=dev)
    k, v = (t[order].reshape(-1, D)[:L] for t in held)
    q = torch.randn(n, Hq, D, generator=g, device=dev).bfloat16()
    i32 = lambda *y: torch.tensor(y, dtype=torch.int32, device=dev)      # noqa: E731
    out, lse = ops.paged_attention(q, cache, order[None], i32(L), i32(0, n), return_lse=True, max_len=n)
    hidden = torch.arange(L - n, L, device=dev)[None, :] > torch.arange(L - n, L, device=dev)[:, None]
    for h in range(Hq):
        score = (q[:, h].double() @ k.T) * D ** -0.5
        score[:, L - n:].masked_fill_(hidden, -math.inf)
        want = torch.logsumexp(score, 1)
        score.sub_(want[:, None]).exp_()
        o, size = score @ v, score @ v.abs()
        assert ((out[:, h].double() - o).abs() <= 2.0 ** -8 * o.abs() + (2.0 ** -8 + 4e-4) * size).all()
        assert ((lse[h].double() - want).abs() <= 2e-4 + 2.0 ** -23 * want.abs()).all()


@pytest.mark.parametrize("fp8", [False, True])
def test_shared_blocks(dev, fp8):
    """Answers of one prompt read its blocks, each with blocks of its own behind it."""
    Hq, Hkv, D, block, prompt = 6, 2, 128, 16, 64
    own = [5, 17, 1]
    s = _batch([1, 3, 1], [prompt + n for n in own], Hq, Hkv, D, block, fp8, seed=4, nan=False)
    s["table"][1:, :prompt // block] = s["table"][0, :prompt // block]
    q, table, ln, cu = _dev(s, dev)
    for hint, reach in ((3, 0), (100, 1 << 20)):
        wide = torch.full((3, max(table.shape[1], reach // block)), -1, dtype=torch.int32, device=dev)
        wide[:, :table.shape[1]] = table
        out, lse = ops.paged_attention(q, _cache(s, dev), wide, ln, cu, return_lse=True, max_len=hint)
        _check(s, out, lse)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("Hq,n", [(8, 1), (8, 4), (8, 70)])
def test_blocks_behind_32_bits(dev, Hq, n, fp8):
    """A cache whose last blocks begin behind 2^32 elements."""
    Hkv, D, block, pages = 8, 128, 64, 66000
    assert (pages - 10) * block * Hkv * D > 2 ** 32
    s = _batch([n, n], [130, 300], Hq, Hkv, D, block, fp8, seed=9, spare=0, nan=False, reach=(1 << 20) * (n > 32))
    need = s["k"][0].shape[0]
    at = [pages - 1 - i if i % 2 else i for i in range(need)]                  # far and near in turn
    big = [torch.empty(pages, block, Hkv, D, dtype=FP8 if fp8 else torch.bfloat16, device=dev) for _ in range(2)]
    scales = [torch.empty(pages, block, Hkv, device=dev) for _ in range(2)] if fp8 else [None, None]
    for x, sc, (c, cs) in zip(big, scales, (s["k"], s["v"])):
        for i, page in enumerate(at):
            x[page].view(torch.uint8).copy_(c[i].view(torch.uint8))
            if fp8:
                sc[page].copy_(cs[i])
    far = s["table"].clone()
    far[far >= 0] = torch.tensor(at, dtype=torch.int32)[far[far >= 0].long()]
    cache = ops.PagedCache(*big, *scales)
    q, _, ln, cu = _dev(s, dev)
    out, lse = ops.paged_attention(q, cache, far.to(dev), ln, cu, return_lse=True, max_len=n)
    _check(s, out, lse)
    new = torch.randn(s["T"], Hkv, D).bfloat16()
    ops.paged_cache_write(cache, new.to(dev), new.to(dev), far.to(dev), ln, cu)
    PO.write(*s["k"], new, s["table"], s["lens"], s["cu"])
    cu_k = torch.tensor([0, 130, 430], dtype=torch.int32, device=dev)
    got, _ = ops.paged_cache_read(cache, far.to(dev), ln, cu_k, 430)
    vals = s["k"][0].float() if not fp8 else s["k"][0].float() * s["k"][1][..., None]
    want = torch.cat([PO.gather(vals, s["table"], b, m, block) for b, m in enumerate((130, 300))]).bfloat16()
    assert torch.equal(got.cpu(), want)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("n", [1, 4, 100])
def test_masked_keys_may_hold_anything_and_seen_ones_count(dev, n, fp8):
    """A NaN in a key makes NaN of the rows that see it and of no others."""
    Hq, Hkv, D, block, L = 4, 2, 128, 16, 100
    s = _batch([n], [L], Hq, Hkv, D, block, fp8, seed=2, nan=False, reach=(1 << 20) * (n > 32))
    j = L - 1 - n // 2                           # seen by the last n // 2 + 1 rows
    page, at = PO.place(s["table"], 0, j, block)
    clean, _, _ = PO.attention(s["q"], PO.held(*s["k"]), PO.held(*s["v"]), s["table"], s["lens"], s["cu"], block)
    if fp8:
        s["k"][0].view(torch.uint8)[page, at, 1, 5] = 0x7F
    else:
        s["k"][0][page, at, 1, 5] = math.nan
    q, table, ln, cu = _dev(s, dev)
    out, lse = ops.paged_attention(q, _cache(s, dev), table, ln, cu, return_lse=True, max_len=n)
    out, first = out.cpu().float()[:n], n - 1 - n // 2       # rows from `first` on see it
    assert out[first:, 2:].isnan().all() and lse.cpu()[2:, first:n].isnan().all()
    rest = out.clone()
    rest[first:, 2:] = clean[:n].float()[first:, 2:]
    assert torch.isfinite(rest).all()
    assert ((rest - clean[:n]).abs() <= 0.05).all()          # that it is the same answer, whose tolerance the other tests hold


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("hint", [1, 8, 200])
def test_values_out_of_range_stay_inside(dev, hint, fp8):
    """Lengths, cu_seqlens and blocks from device memory that fit nothing are held inside their arrays; the sequences that are right are right."""
    Hq, Hkv, D, block = 4, 2, 64, 16
    s = _batch([2, 4, 3, 6], [30, 40, 50, 60], Hq, Hkv, D, block, fp8, seed=8, nan=False, reach=(1 << 20) * (hint > 8))
    q, table, ln, cu = _dev(s, dev)
    want = ops.paged_attention(q, _cache(s, dev), table, ln, cu, max_len=hint)
    reach = table.shape[1] * block

    def run(table, ln, cu):
        cache = _cache(s, dev)
        out = ops.paged_attention(q, cache, table, ln, cu, max_len=hint)
        ops.paged_cache_write(cache, q[:, :Hkv].contiguous(), q[:, :Hkv].contiguous(), table, ln, cu)
        k, v = ops.paged_cache_read(cache, table, ln, cu, s["T"])
        torch.cuda.synchronize()
        return out
    bad = table.clone()
    bad[1, :5] = torch.tensor([2 ** 31 - 1, -2 ** 31, 10 ** 6, -1, 5], dtype=torch.int32)
    got = run(bad, ln, cu)
    assert torch.equal(got[:2], want[:2]) and torch.equal(got[6:15], want[6:15])
    long = ln.clone()
    long[1], long[2] = 2 ** 31 - 1, -5
    got = run(table, long, cu)
    assert torch.equal(got[:2], want[:2]) and (got[6:9] == 0).all() and torch.equal(got[9:15], want[9:15])
    assert reach < 2 ** 31 - 1
    for wild in ([0, 2, 6, 9, 2 ** 31 - 1], [0, 2, -9, 2 ** 30, 15], [7, 2, 1, 0, -4], [-2 ** 31, -1, 0, 3, 2]):
        run(table, ln, torch.tensor(wild, dtype=torch.int32, device=dev))


def test_nothing_to_do(dev):
    cache = ops.PagedCache.empty(4, 16, 2, 128, device=dev)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)      # noqa: E731
    none = torch.zeros(2, 0, dtype=torch.int32, device=dev)
    q = torch.randn(3, 4, 128, device=dev).bfloat16()
    out, lse = ops.paged_attention(q, cache, none, i32(0, 7), i32(0, 1, 3), return_lse=True)      # a table of no blocks: no keys
    assert (out == 0).all() and torch.isinf(lse).all() and (lse < 0).all()
    ops.paged_cache_write(cache, q[:, :2], q[:, :2], none, i32(0, 7), i32(0, 1, 3))
    assert ops.paged_attention(q[:0], cache, none, i32(0, 0), i32(0, 0, 0)).shape == (0, 4, 128)
    left = torch.full_like(q, 3.0)
    assert (ops.paged_attention(q, cache, none[:0], i32(), i32(0), out=left) == 3.0).all()
    k, v = ops.paged_cache_read(cache, none, i32(0, 0), i32(0, 0, 0), 0)
    assert k.shape == v.shape == (0, 2, 128)
    accepted, tokens = ops.verify_drafts(torch.ones(2, 5, device=dev), None, torch.zeros(2, dtype=torch.long, device=dev), torch.zeros(2, device=dev), i32(0))
    assert accepted.numel() == 0 and tokens.numel() == 2


@pytest.mark.parametrize("fp32", [False, True])
def test_verify_rows_of_any_place_and_values(dev, fp32):
    """Rows that begin anywhere, ends of u, rows that hold no probability, tokens outside the vocabulary, equal distributions."""
    g = torch.Generator().manual_seed(3)
    V, dt = 5003, torch.float32 if fp32 else torch.bfloat16
    ns = [3, 2, 2, 4, 1, 3, 2]
    cu = torch.tensor([0] + torch.tensor(ns).cumsum(0).tolist(), dtype=torch.int32)
    T, B = sum(ns), len(ns)
    target = (2 * torch.randn(T, V, generator=g)).softmax(-1).to(dt)
    draft = (2 * torch.randn(T - B, V, generator=g)).softmax(-1).to(dt)
    ids = torch.randint(0, V, (T,), generator=g)
    u = torch.rand(T, generator=g)
    target[0] = math.nan                          # nothing left in it
    target[3] = draft[2]                          # equal: every draft stands
    ids[6], ids[8] = V, -1                        # not in the vocabulary
    target[12, 7], target[12, 9] = math.inf, -1.0
    u[5], u[9], u[11] = 0.0, 1 - 2.0 ** -24, 0.0
    target[14] = 0
    target[14, 4098] = 0.5                        # one token, behind the first chunk's border
    for off in (0, 1, 3):
        wide = torch.zeros(T, V + 8, dtype=dt)
        wide_d = torch.zeros(T - B, V + 5, dtype=dt)
        wide[:, off:off + V], wide_d[:, off:off + V] = target, draft
        for d in (draft, None):
            x = wide.to(dev)[:, off:off + V]
            y = None if d is None else wide_d.to(dev)[:, off:off + V]
            got_a, got_t = ops.verify_drafts(x, y, ids.to(dev), u.to(dev), cu.to(dev))
            want_a, want_t = PO.verify(target, d, ids, u, cu)
            assert torch.equal(got_a.cpu(), want_a) and torch.equal(got_t.cpu(), want_t)


def test_verify_with_offsets_out_of_range(dev):
    """cu_seqlens that fit nothing are held inside the rows; rows that are right are right."""
    g = torch.Generator().manual_seed(5)
    T, V = 9, 300
    target = torch.randn(T, V, generator=g).softmax(-1)
    ids, u = torch.randint(0, V, (T,), generator=g), torch.rand(T, generator=g)
    draft = torch.randn(5, V, generator=g).softmax(-1)
    for wild in ([0, 3, 2 ** 31 - 1], [0, 3, -4, 9], [9, 5, 0], [-2 ** 31, 3, 2 ** 31 - 1, 0]):
        cu = torch.tensor(wild, dtype=torch.int32)
        for d in (None, draft):
            accepted, tokens = ops.verify_drafts(target.to(dev), None if d is None else d.to(dev), ids.to(dev), u.to(dev), cu.to(dev))
            accepted = accepted.cpu()
            assert ((accepted >= 0) & (accepted < T)).all()
            if wild[:2] == [0, 3]:
                want_a, want_t = PO.verify(target[:3], d, ids[:3], u[:3], torch.tensor([0, 3]))
                assert accepted[0] == want_a[0]
                if wild[2] > 0:
                    assert torch.equal(tokens.cpu()[:3], want_t)


def test_verify_without_rows(dev):
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)      # noqa: E731
    accepted, tokens = ops.verify_drafts(torch.ones(0, 5, device=dev), None, torch.zeros(0, dtype=torch.long, device=dev), torch.zeros(0, device=dev), i32(0, 0, 0))
    assert accepted.tolist() == [0, 0] and tokens.numel() == 0
    # drafts without a row of their distribution count as drawn with probability 0: they stand where the target has anything
    target = torch.tensor([[0.5, 0.5, 0.0], [0.0, 0.0, 1.0]], device=dev)
    for last, want in ((0, [1]), (2, [0])):
        ids, u = torch.tensor([1, last], device=dev), torch.tensor([0.3, 0.3], device=dev)
        accepted, tokens = ops.verify_drafts(target, torch.zeros(0, 3, device=dev), ids, u, i32(0, 2))
        assert accepted.tolist() == want and tokens.tolist() == ([0, 2] if want == [1] else [0, -1])


def test_callable_with_a_block_table(dev):
    import varlen_attention as VA
    for qs, ks in (([1, 1, 1], [5, 70, 33]), ([60, 200], [60, 333])):
        s = _batch(qs, ks, 6, 2, 128, 64, False, seed=1, tail=0)
        q, table, ln, cu = _dev(s, dev)
        cache = _cache(s, dev)
        cu_k = torch.tensor([0] + torch.tensor(ks).cumsum(0).tolist(), dtype=torch.int32, device=dev)
        got = VA.flash_attn_varlen_func(q, cache.k, cache.v, cu, cu_k, max(qs), max(ks), causal=True, block_table=table)
        _check(s, got, None)
        assert torch.equal(got, ops.paged_attention(q, cache, table, ln, cu, max_len=max(qs)))
        full = VA.flash_attn_varlen_func(q, cache.k, cache.v, cu, cu_k, softmax_scale=0.2, block_table=table)
        _check(s, full, None, causal=False, scale=0.2)


def _softmax(model, hidden):
    return model.lm_head(hidden).float().softmax(-1)


@pytest.mark.parametrize("fp8", [False, True])
def test_a_model_reads_prompts_in_pieces_and_verifies_drafts(dev, fp8, monkeypatch):
    """A small random Qwen2 model over paged caches: pieces of prompts, then a chunk of drafts a sequence, then single tokens behind
    what was accepted.  Each layer's cache holds the keys that were handed over, its attention is the 64-bit one's over what the cache holds,
    and the tokens are the 64-bit verification's."""
    from transformers import Qwen2Config, Qwen2ForCausalLM
    import varlen_attention as VA
    torch.manual_seed(0)
    V, layers, block, Hkv, D = 256, 2, 16, 2, 128
    model = Qwen2ForCausalLM(Qwen2Config(vocab_size=V, hidden_size=512, intermediate_size=512, num_hidden_layers=layers, num_attention_heads=4,
                                         num_key_value_heads=Hkv, max_position_embeddings=1024)).to(dev).to(torch.bfloat16).eval()
    VA.install_explicit_varlen_wrapper(model)
    seen = []
    inner = VA._paged_forward

    def record(module, query, key, value, *a):
        out = inner(module, query, key, value, *a)
        seen.append((module.layer_idx, query, key, value, out[0]))
        return out
    monkeypatch.setattr(VA, "_paged_forward", record)
    g = torch.Generator().manual_seed(1)
    B, width = 3, 8
    caches = [ops.PagedCache.empty(B * width, block, Hkv, D, FP8 if fp8 else torch.bfloat16, dev) for _ in range(layers)]
    table = torch.randperm(B * width, generator=g).int().view(B, width)
    held = [[torch.zeros(B, width * block, Hkv, D, dtype=torch.bfloat16) for _ in range(2)] for _ in range(layers)]      # what was handed over
    length = [0] * B

    def step(tokens):                   # a list of new tokens a sequence -> final hidden rows, packed
        ns = [len(t) for t in tokens]
        now = [a + n for a, n in zip(length, ns)]
        cu = torch.tensor([0] + torch.tensor(ns).cumsum(0).tolist(), dtype=torch.int32)
        lens = torch.tensor(now, dtype=torch.int32)
        pos = torch.cat([torch.arange(a, b) for a, b in zip(length, now)])
        batch = VA.PagedBatch(caches, table.to(dev), lens.to(dev), cu.to(dev), max(ns))
        ids = torch.cat([torch.tensor(t, dtype=torch.long) for t in tokens])
        seen.clear()
        with torch.no_grad():
            hidden = model.model(input_ids=ids[None].to(dev), position_ids=pos[None].to(dev), use_cache=False, paged_batch=batch).last_hidden_state[0]
        assert [x[0] for x in seen] == list(range(layers))
        for i, query, key, value, out in seen:
            c = caches[i]
            cpu = [c.k.cpu(), c.v.cpu()]
            sc = [c.k_scale.cpu(), c.v_scale.cpu()] if fp8 else [None, None]
            for w, new in enumerate((key, value)):
                for b in range(B):
                    held[i][w][b, length[b]:now[b]] = new[0].transpose(0, 1)[int(cu[b]):int(cu[b + 1])].cpu()
                    for j in range(now[b]):
                        page, at = PO.place(table, b, j, block)
                        if fp8:
                            code, s = PO.quantise(held[i][w][b, j])
                            assert torch.equal(code.float(), cpu[w][page, at].float()) and torch.equal(s, sc[w][page, at])
                        else:
                            assert torch.equal(held[i][w][b, j], cpu[w][page, at])
            s = dict(q=query[0].transpose(0, 1).cpu(), k=(cpu[0].float().nan_to_num().bfloat16() if not fp8 else cpu[0], sc[0]), v=(cpu[1], sc[1]),
                     table=table, lens=lens, cu=cu, block=block, rows=int(cu[-1]))
            _check_scaled(s, out[0])
        length[:] = now
        return hidden, cu
    prompts = [torch.randint(0, V, (n,), generator=g).tolist() for n in (37, 5, 64)]
    step([p[:20] for p in prompts])                                # pieces: one prompt ends in the first
    hidden, cu = step([p[20:] for p in prompts])
    # drafts: the model's own best guesses for some, random tokens for others
    last = [int(torch.randint(0, V, (), generator=g)) for _ in range(B)]
    chunk = [[last[b]] + torch.randint(0, V, (b + 2,), generator=g).tolist() for b in range(B)]
    hidden, cu = step(chunk)
    with torch.no_grad():
        target = _softmax(model, hidden)
    ids = torch.tensor(sum(chunk, []))
    u = torch.rand(len(ids), generator=g) * 0.01
    for draft in (None, torch.rand(len(ids) - B, V, generator=g).softmax(-1)):
        accepted, tokens = ops.verify_drafts(target, None if draft is None else draft.to(dev), ids.to(dev), u.to(dev), cu.to(dev))
        want_a, want_t = PO.verify(target.cpu(), draft, ids, u, cu)
        assert torch.equal(accepted.cpu(), want_a) and torch.equal(tokens.cpu(), want_t)
    assert 0 < int(want_a.sum()), "no draft stood"
    for b in range(B):                                             # rejected drafts are written over
        length[b] += int(want_a[b]) + 1 - len(chunk[b])
    step([[int(want_t[int(cu[b]) + int(want_a[b])])] for b in range(B)])


def _check_scaled(s, out):
    """_check for rows that are not standard normal: the scores' error goes by their own sizes."""
    scale = s["q"].shape[-1] ** -0.5
    want, _, size = PO.attention(s["q"], PO.held(*s["k"]), PO.held(*s["v"]), s["table"], s["lens"], s["cu"], s["block"], scale)
    k = PO.held(*s["k"])
    most = float(s["q"].float().norm(dim=-1).max()) * max(float(PO.gather(k, s["table"], b, int(n), s["block"]).norm(dim=-1).max()) for b, n in enumerate(s["lens"]))
    err = 2 * 128 * 2.0 ** -24 * most * scale + 2e-4                # of numerator and denominator; the exponential's own
    over = (out.cpu().double() - want).abs() - (2.0 ** -8 * want.abs() + (2.0 ** -8 + err) * size)
    assert float(over.max()) <= 0


@pytest.mark.parametrize("fp8", [False, True])
def test_captured_step_follows_new_lengths(dev, fp8):
    """Write, attention and verification in one graph, replayed for other lengths, blocks and rows, with eager work between."""
    Hq, Hkv, D, block, B, V = 8, 2, 128, 16, 5, 1000
    g = torch.Generator().manual_seed(0)
    pages, width, T = 64, 12, 20
    cache = ops.PagedCache.empty(pages, block, Hkv, D, FP8 if fp8 else torch.bfloat16, dev)
    for t in (cache.k, cache.v):
        t.view(torch.uint8).zero_()
    for t in ((cache.k_scale, cache.v_scale) if fp8 else ()):
        t.fill_(1.0)
    mk = lambda *sh: torch.randn(*sh, generator=g)       # noqa: E731

    def draw(i):
        ns = [[4, 4, 4, 4, 4], [1, 7, 0, 2, 3], [0, 0, 20, 0, 0], [1, 1, 1, 1, 1]][i % 4]
        lens = [n + int(torch.randint(0, width * block - 20, (), generator=g)) for n in ns]
        table = torch.randperm(pages, generator=g)[:B * width].int().view(B, width)
        cu = torch.tensor([0] + torch.tensor(ns).cumsum(0).tolist(), dtype=torch.int32)
        return dict(q=mk(T, Hq, D).bfloat16(), k=mk(T, Hkv, D).bfloat16(), v=mk(T, Hkv, D).bfloat16(), table=table, lens=torch.tensor(lens, dtype=torch.int32), cu=cu,
                    target=mk(T, V).softmax(-1), ids=torch.randint(0, V, (T,), generator=g), u=torch.rand(T, generator=g))
    at = {k: v.to(dev) for k, v in draw(0).items()}
    out = torch.zeros(T, Hq, D, dtype=torch.bfloat16, device=dev)

    def run(out):
        ops.paged_cache_write(cache, at["k"], at["v"], at["table"], at["lens"], at["cu"])
        o, lse = ops.paged_attention(at["q"], cache, at["table"], at["lens"], at["cu"], return_lse=True, max_len=4, out=out)
        return (o, lse) + ops.verify_drafts(at["target"], None, at["ids"], at["u"], at["cu"])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(out)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run(out)
    for i in range(1, 6):
        for k, v in draw(i).items():
            at[k].copy_(v)
        n = int(at["cu"][-1])
        before = [t.clone() for t in (cache.k, cache.v)]
        graph.replay()
        torch.cuda.synchronize()
        have = [t.clone() for t in got]
        for t, b in zip((cache.k, cache.v), before):
            t.copy_(b)
        want = run(torch.zeros_like(out))
        torch.cuda.synchronize()
        assert torch.equal(have[0][:n], want[0][:n]) and torch.equal(have[1][:, :n], want[1][:, :n]), f"replay {i}"
        assert torch.equal(have[2], want[2]) and torch.equal(have[3][:n], want[3][:n]), f"replay {i}"


def test_two_streams_at_once(dev):
    cases = [_batch([1] * 6, [500, 3, 70, 900, 33, 64], 8, 2, 128, 16, False, seed=21), _batch([300], [1200], 8, 2, 128, 16, True, seed=22, reach=1 << 20)]
    ins = [(*_dev(s, dev), _cache(s, dev)) for s in cases]
    want = [ops.paged_attention(q, c, t, ln, cu, max_len=64) for q, t, ln, cu, c in ins]
    streams = [torch.cuda.Stream() for _ in ins]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, (q, t, ln, cu, c) in enumerate(ins):
            with torch.cuda.stream(streams[i]):
                got[i].append(ops.paged_attention(q, c, t, ln, cu, max_len=64))
    torch.cuda.synchronize()
    for s, w, gs in zip(cases, want, got):
        _check(s, w, None)
        for x in gs:
            assert torch.equal(x[:s["rows"]], w[:s["rows"]])
