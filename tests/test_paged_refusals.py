"""What the paged cache, the attention over it and the verification of drafts refuse, without a GPU: through the C ABI with
addresses that are looked at before they are used, and through the torch layer with CPU tensors."""
import ctypes as C
import os

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
AT, ODD = 4096, 4098                       # refused before they are read


@pytest.fixture(scope="module")
def lib():
    from fgrpo import _lib
    from fgrpo.build import LIB_PATH, build
    if not os.path.exists(LIB_PATH):
        build(verbose=False)
    return _lib.load()


def _cache(**over):
    from fgrpo import _lib
    c = _lib.PagedCacheStruct(k=AT, v=AT, k_scale=None, v_scale=None, num_blocks=4, block_size=16, heads=2, head_dim=128, dtype=_lib.BF16)
    for name in ("k_stride", "v_stride"):
        setattr(c, name, (C.c_longlong * 3)(16 * 2 * 128, 2 * 128, 128))
    for name, value in over.items():
        setattr(c, name, (C.c_longlong * 3)(*value) if isinstance(value, tuple) else value)
    return c


BAD_CACHES = [
    (dict(k=None), -1), (dict(v=None), -1), (dict(num_blocks=0), -1), (dict(heads=0), -1), (dict(block_size=8), -2), (dict(block_size=48), -2),
    (dict(block_size=1 << 17), -2), (dict(head_dim=96), -2), (dict(dtype=1), -1), (dict(dtype=7), -1), (dict(dtype=2), -1), (dict(k=ODD), -5),
    (dict(v_stride=(4096, 256, 100)), -5), (dict(k_stride=(-4096, 256, 128)), -5),
]


@pytest.mark.parametrize("over,rc", BAD_CACHES)
def test_caches_are_checked_by_every_call(lib, over, rc):
    c = C.byref(_cache(**over))
    assert lib.fgrpo_paged_cache_write(c, AT, AT, 256, 128, 256, 128, AT, 8, 8, AT, AT, 2, 5, None) == rc
    assert lib.fgrpo_last_error().startswith(b"paged_cache_write: ")
    assert lib.fgrpo_paged_cache_read(c, AT, 8, 8, AT, AT, 2, 5, AT, AT, None) == rc
    assert lib.fgrpo_last_error().startswith(b"paged_cache_read: ")
    assert _attend(lib, c) == rc
    assert lib.fgrpo_last_error().startswith(b"paged_attn_fwd: ")


def _attend(lib, c, q=AT, q_t=1536, q_h=128, table=AT, table_st=8, width=8, lens=AT, cu=AT, n_seq=2, T=5, Hq=12, max_len=0, scale=0.1, out=AT, ws=AT,
            ws_bytes=1 << 40):
    return lib.fgrpo_paged_attn_fwd(q, q_t, q_h, c, table, table_st, width, lens, cu, n_seq, T, Hq, max_len, scale, 1, out, None, ws, ws_bytes, None)


@pytest.mark.parametrize("over,rc", [
    (dict(q=None), -1), (dict(out=None), -1), (dict(lens=None), -1), (dict(cu=None), -1), (dict(table=None), -1), (dict(n_seq=0), -1), (dict(T=0), -1),
    (dict(width=-1), -1), (dict(table_st=4), -1), (dict(width=1 << 27, table_st=1 << 27), -2), (dict(Hq=7), -1), (dict(Hq=0), -1), (dict(scale=0.0), -1),
    (dict(scale=float("nan")), -1), (dict(q=ODD), -5), (dict(out=ODD), -5), (dict(q_t=100), -5), (dict(q_h=-128), -5),
    (dict(ws=None), -3), (dict(ws_bytes=64), -3), (dict(ws=ODD), -5)])
def test_attention_arguments(lib, over, rc):
    assert _attend(lib, C.byref(_cache()), **over) == rc
    assert lib.fgrpo_last_error().startswith(b"paged_attn_fwd: ")


@pytest.mark.parametrize("at,value,rc", [(0, None, -1), (1, 10, -1), (3, 10, -1), (4, -1, -1), (5, 7, -1), (6, None, -1), (7, None, -1), (8, None, -1),
                                         (9, 0, -1), (10, 0, -1), (11, 0, -1), (11, 1 << 30, -1), (12, None, -1), (13, None, -1), (14, None, -3), (14, ODD, -5), (15, 8, -3)])
def test_verify_arguments(lib, at, value, rc):
    args = [AT, 1000, AT, 1000, 3, 1, AT, AT, AT, 2, 5, 1000, AT, AT, AT, 1 << 40, None]
    args[at] = value
    assert lib.fgrpo_verify_drafts(*args) == rc and lib.fgrpo_last_error().startswith(b"verify_drafts: ")


def test_torch_layer_refuses_before_it_takes_an_address():
    from fgrpo import ops
    kv = torch.zeros(4, 16, 2, 128, dtype=torch.bfloat16)
    table, lens, cu = torch.zeros(1, 4, dtype=torch.int32), torch.ones(1, dtype=torch.int32), torch.tensor([0, 1], dtype=torch.int32)
    new, q = torch.zeros(1, 2, 128, dtype=torch.bfloat16), torch.zeros(1, 4, 128, dtype=torch.bfloat16)
    for call in (lambda: ops.paged_cache_write(ops.PagedCache(kv, kv), new, new, table, lens, cu),
                 lambda: ops.paged_cache_read(ops.PagedCache(kv, kv), table, lens, cu, 1),
                 lambda: ops.paged_attention(q, ops.PagedCache(kv, kv), table, lens, cu),
                 lambda: ops.verify_drafts(torch.zeros(2, 8), None, torch.zeros(2, dtype=torch.long), torch.zeros(2), cu)):
        with pytest.raises(RuntimeError, match="GPU"):
            call()
    with pytest.raises(RuntimeError, match="head_dim"):
        ops.paged_attention(q, ops.PagedCache(kv[0], kv[0]), table, lens, cu)
    with pytest.raises(RuntimeError, match="bf16 or float8"):
        ops.paged_attention(q, ops.PagedCache(kv.half(), kv.half()), table, lens, cu)
    with pytest.raises(RuntimeError, match="contiguous"):
        ops.paged_attention(q, ops.PagedCache(kv.transpose(2, 3), kv.transpose(2, 3)), table, lens, cu)
    with pytest.raises(RuntimeError, match="gradient"):
        ops.paged_attention(q.clone().requires_grad_(True), ops.PagedCache(kv, kv), table, lens, cu)
    with pytest.raises(RuntimeError, match="gradient"):
        ops.paged_cache_write(ops.PagedCache(kv, kv), new.clone().requires_grad_(True), new, table, lens, cu)
    with pytest.raises(RuntimeError, match="float8_e4m3fn"):
        ops.PagedCache.empty(4, 16, 2, 128, torch.float16, "cpu")
    with pytest.raises(RuntimeError, match="unsupported dtype"):
        ops.verify_drafts(torch.zeros(2, 8, dtype=torch.float64), None, torch.zeros(2, dtype=torch.long), torch.zeros(2), cu)


def test_callables_refuse(monkeypatch):
    import varlen_attention as VA
    from types import SimpleNamespace
    from fgrpo import ops
    kv = torch.zeros(4, 16, 2, 128, dtype=torch.bfloat16)
    q, cu, table = torch.zeros(3, 4, 128, dtype=torch.bfloat16), torch.tensor([0, 1, 3], dtype=torch.int32), torch.zeros(2, 4, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="GPU"):
        VA.flash_attn_varlen_func(q, kv, kv, cu, cu, block_table=table)
    with pytest.raises(RuntimeError, match="entry for each"):
        VA.flash_attn_varlen_func(q, kv, kv, cu, cu[:2], block_table=table)
    with pytest.raises(RuntimeError, match="gradient"):
        VA.flash_attn_varlen_func(q, kv.clone().requires_grad_(True), kv, cu, cu, block_table=table)
    for name, value in (("dropout_p", 0.1), ("window_size", (5, 0)), ("softcap", 1.0), ("return_attn_probs", True)):
        with pytest.raises(RuntimeError, match="fgrpo varlen attention"):
            VA.flash_attn_varlen_func(q, kv, kv, cu, cu, block_table=table, **{name: value})
    with pytest.raises(RuntimeError, match="cache for each layer"):
        VA.PagedBatch([], table, cu[1:], cu)
    batch = VA.PagedBatch([ops.PagedCache(kv, kv)], table, cu[1:], cu)
    assert batch.reach() == 64
    x, y = torch.zeros(1, 4, 3, 128, dtype=torch.bfloat16), torch.zeros(1, 2, 3, 128, dtype=torch.bfloat16)
    layer = SimpleNamespace(layer_idx=0, is_causal=True)
    with pytest.raises(RuntimeError, match="GPU"):
        VA.varlen_attention_forward(layer, x, y, y, paged_batch=batch)
    with pytest.raises(RuntimeError, match="no cache for layer 1"):
        VA.varlen_attention_forward(SimpleNamespace(layer_idx=1), x, y, y, paged_batch=batch)
    with pytest.raises(RuntimeError, match="no cache for layer None"):
        VA.varlen_attention_forward(SimpleNamespace(), x, y, y, paged_batch=batch)
    with pytest.raises(RuntimeError, match="one packed row"):
        VA.varlen_attention_forward(layer, x.expand(2, -1, -1, -1), y.expand(2, -1, -1, -1), y.expand(2, -1, -1, -1), paged_batch=batch)
    with pytest.raises(RuntimeError, match="sliding"):
        VA.varlen_attention_forward(layer, x, y, y, sliding_window=63, paged_batch=batch)
    with pytest.raises(RuntimeError, match="paged caches"):
        VA.varlen_attention_forward(layer, x, y[:, :, :2], y[:, :, :2], paged_batch=batch)


def test_tables_that_reach_the_end_of_32_bits(lib):
    c = C.byref(_cache(block_size=65536))
    assert _attend(lib, c, width=32768, table_st=32768) == -2 and b"2^31" in lib.fgrpo_last_error()
    assert _attend(lib, c, width=32767, table_st=32767, ws_bytes=8) == -3          # this far it goes


def test_outputs_and_caches_that_want_gradients():
    from fgrpo import ops
    kv = torch.zeros(4, 16, 2, 128, dtype=torch.bfloat16)
    table, lens, cu = torch.zeros(1, 4, dtype=torch.int32), torch.ones(1, dtype=torch.int32), torch.tensor([0, 1], dtype=torch.int32)
    q = torch.zeros(1, 4, 128, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="gradient"):
        ops.paged_attention(q, ops.PagedCache(kv, kv.clone().requires_grad_(True)), table, lens, cu)
    with pytest.raises(RuntimeError, match="gradient"):
        ops.paged_cache_write(ops.PagedCache(kv.clone().requires_grad_(True), kv), q[:, :2], q[:, :2], table, lens, cu)


def test_verify_needs_a_vocabulary():
    from fgrpo import ops
    with pytest.raises(RuntimeError, match="vocabulary"):
        ops.verify_drafts(torch.zeros(2, 0), None, torch.zeros(2, dtype=torch.long), torch.zeros(2), torch.tensor([0, 2], dtype=torch.int32))
