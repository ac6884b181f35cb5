"""Host side of the serving operators: argument blocks, the C entry points'
refusals (which launch nothing), and the wrappers' answers to CPU tensors."""

from __future__ import annotations

import ctypes

import pytest
import torch

from cortex import _lib as L
from cortex.kernels.kv_evict import evict_by_weight
from cortex.kernels.lora import lora_linear
from cortex.kernels.paged_attention import paged_attention


@pytest.mark.parametrize("packed,struct", [
    (L.PAGED_ATTENTION_ARGS, L.PagedAttentionArgs),
    (L.EVICT_ARGS, L.EvictArgs),
    (L.LORA_ARGS, L.LoraArgs),
])
def test_packed_blocks_have_the_struct_layout(packed, struct):
    assert packed.size == ctypes.sizeof(struct)
    values = list(range(1, len(struct._fields_) + 1))
    block = struct.from_buffer_copy(packed.pack(*values))
    assert [getattr(block, name) or 0 for name, _ in struct._fields_] == values


def _paged(**kw):
    base = dict(dtype=L.CK_BF16, B=2, H=8, Hkv=4, Dh=64, q=16, q_ld_b=512, q_ld_h=64, pool=16,
                num_pages=4, page_ld=16 * 512, row_ld=512, page_size=16, page_table_width=4,
                page_table=16, page_table_ld=4, lengths=16, o=16, o_ld_b=512, o_ld_h=64, scale=0.1)
    base.update(kw)
    return bytes(L.PagedAttentionArgs(**base))


def test_paged_attention_refusals():
    lib = L.load()

    def rc(ws=0, n=0, **kw):
        return lib.ck_paged_attention(_paged(**kw), ws, n, 0)

    assert lib.ck_paged_attention(None, 0, 0, 0) == L.CK_ERR_INVALID_ARG
    assert rc(dtype=L.CK_I8) == L.CK_ERR_UNSUPPORTED
    assert rc(Dh=257) == L.CK_ERR_UNSUPPORTED
    assert rc(H=4100) == L.CK_ERR_UNSUPPORTED
    for bad in (dict(B=-1), dict(H=0), dict(Hkv=0), dict(H=6), dict(Dh=0), dict(page_size=0),
                dict(page_table_width=-1), dict(num_pages=-1), dict(scale=float("nan")),
                dict(page_table_width=2 ** 28), dict(w_out=16), dict(w_out=16, w_in=16, w_width=63)):
        assert rc(**bad) == L.CK_ERR_INVALID_ARG, bad
    assert rc(B=0) == L.CK_OK
    big = dict(page_table_width=512)
    need = lib.ck_paged_attention_workspace_bytes(_paged(**big))
    assert need > 0
    assert rc(**big) == L.CK_ERR_WORKSPACE
    assert rc(ws=16, n=need - 1, **big) == L.CK_ERR_WORKSPACE
    assert rc(ws=8, n=need, **big) == L.CK_ERR_WORKSPACE
    for missing in ("q", "o", "lengths", "pool", "page_table"):
        assert rc(ws=16, n=need, **big, **{missing: None}) == L.CK_ERR_INVALID_ARG
    assert lib.ck_paged_attention_workspace_bytes(None) == 0


def _evict(**kw):
    base = dict(elem_bytes=2, B=2, pool=16, num_pages=8, page_ld=16 * 64, row_ld=64, page_size=16,
                width=64, page_table=16, page_table_ld=100, page_table_width=100, budget=500, recent=3,
                fill=1, lengths=16, lengths_out=32, w_in=16, w_out=32, pos_in=16, pos_out=32,
                w_in_ld=1600, w_out_ld=500, pos_in_ld=1600, pos_out_ld=500, in_width=1600, out_width=500)
    base.update(kw)
    return bytes(L.EvictArgs(**base))


def test_evict_refusals():
    lib = L.load()
    need = lib.ck_evict_workspace_bytes(_evict())
    assert need > 0

    def rc(ws=16, n=need, **kw):
        return lib.ck_evict_by_weight(_evict(**kw), ws, n, 0)

    assert lib.ck_evict_by_weight(None, 0, 0, 0) == L.CK_ERR_INVALID_ARG
    assert rc(elem_bytes=1) == L.CK_ERR_UNSUPPORTED
    for bad in (dict(B=-1), dict(budget=0), dict(recent=501), dict(recent=-1), dict(width=0),
                dict(page_size=0), dict(in_width=1599), dict(out_width=499), dict(num_pages=-1),
                dict(page_table_width=2 ** 28), dict(w_out=16), dict(pos_out=16)):
        assert rc(**bad) == L.CK_ERR_INVALID_ARG, bad
    for missing in ("lengths", "lengths_out", "w_in", "w_out", "pos_in", "pos_out", "pool",
                    "page_table"):
        assert rc(**{missing: None}) == L.CK_ERR_INVALID_ARG
    assert rc(ws=0) == L.CK_ERR_WORKSPACE
    assert rc(n=need - 1) == L.CK_ERR_WORKSPACE
    assert rc(B=0) == L.CK_OK
    # a budget that no sequence can pass, or by a few rows only, needs no workspace
    assert lib.ck_evict_workspace_bytes(_evict(budget=1600, out_width=1600)) == 0
    assert lib.ck_evict_workspace_bytes(_evict(budget=1580, out_width=1600)) == 0
    assert lib.ck_evict_workspace_bytes(None) == 0


def _lora(**kw):
    base = dict(dtype=L.CK_BF16, n_adapters=3, rank=8, M=300, K=64, N=32, x=16, ldx=64, w=16,
                ldw=64, a=16, b=16, ids=16, y=16, ldy=32)
    base.update(kw)
    return bytes(L.LoraArgs(**base))


def test_lora_refusals():
    lib = L.load()

    def rc(ws=16, n=1 << 40, **kw):
        return lib.ck_lora_linear(_lora(**kw), ws, n, 0)

    assert lib.ck_lora_linear(None, 0, 0, 0) == L.CK_ERR_INVALID_ARG
    assert rc(dtype=L.CK_I8) == L.CK_ERR_UNSUPPORTED
    for big in (dict(rank=257), dict(M=2 ** 28 + 1), dict(N=2 ** 31 - 100), dict(K=2 ** 31 - 100)):
        assert rc(**big) == L.CK_ERR_UNSUPPORTED, big
    for bad in (dict(M=-1), dict(N=-1), dict(K=0), dict(rank=0), dict(n_adapters=-1)):
        assert rc(**bad) == L.CK_ERR_INVALID_ARG, bad
    for missing in ("x", "w", "a", "b", "ids", "y"):
        for M in (3, 300):
            assert rc(M=M, **{missing: None}) == L.CK_ERR_INVALID_ARG
    assert rc(M=0) == L.CK_OK and rc(N=0) == L.CK_OK
    for M in (40, 300):
        for dtype in (L.CK_BF16, L.CK_F32):
            need = lib.ck_lora_workspace_bytes(_lora(M=M, dtype=dtype))
            assert need > 0
            assert rc(M=M, dtype=dtype, n=need - 1) == L.CK_ERR_WORKSPACE
            assert rc(M=M, dtype=dtype, ws=0) == L.CK_ERR_WORKSPACE
    # a few rows in one launch: no workspace
    assert lib.ck_lora_workspace_bytes(_lora(M=1)) == 0
    assert lib.ck_lora_workspace_bytes(None) == 0


def test_cpu_tensors_are_refused():
    i32 = torch.int32
    pool, table, n = torch.zeros(4, 16, 512), torch.zeros(2, 3, dtype=i32), torch.zeros(2, dtype=i32)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        paged_attention(torch.zeros(2, 4, 64), pool, table, n)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        evict_by_weight(pool, table, n, torch.zeros(2, 48), torch.zeros(2, 48, dtype=i32), budget=3)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        lora_linear(torch.zeros(2, 8), torch.zeros(4, 8), torch.zeros(1, 2, 8), torch.zeros(1, 4, 2),
                    torch.zeros(2, dtype=i32))


def test_outputs_that_share_memory_are_refused():
    buf = torch.zeros(4, 16)
    x, y = buf[:2], buf[2:]
    L.check_output("op", "out", y, x, None)
    L.check_output("op", "out", torch.zeros(3, 1, 5)[:, :, ::2], x)  # strides, a dimension of one
    L.check_output("op", "out", torch.zeros(6, 2).t(), x)
    L.check_output("op", "out", torch.zeros(0, 4), x)
    for out in (torch.zeros(4).expand(2, 4), torch.zeros(8).as_strided((3, 4), (2, 1))):
        with pytest.raises(ValueError, match="share memory"):
            L.check_output("op", "out", out, x)
    for out in (x, buf[1:3], buf[:, 8:]):
        with pytest.raises(ValueError, match="overlaps an input"):
            L.check_output("op", "out", out, x)


def test_a_refused_call_leaves_no_workspace_size():
    """The size query answers 0 for a block that the call refuses: the next call of
    the same key asks again."""
    sizes, seen = [0, 512], []

    def query(block):
        return sizes[len(seen)]

    def call(block, ws, n, stream):
        seen.append(n)
        return L.CK_OK if n == 512 else L.CK_ERR_INVALID_ARG

    key, cpu = ("a key of this test",), torch.device("cpu")
    with pytest.raises(ValueError):
        L.launch("op", call, query, key, b"", cpu, 0)
    L.launch("op", call, query, key, b"", cpu, 0)
    L.launch("op", call, lambda block: 1 / 0, key, b"", cpu, 0)  # remembered: not asked again
    assert seen == [0, 512, 512]


def test_cache_methods_refuse_capture(monkeypatch):
    from cortex.cache import StreamingKVCache

    cache = object.__new__(StreamingKVCache)  # the refusal comes before any of its state
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="captured"):
        cache.page_table([])
    with pytest.raises(RuntimeError, match="captured"):
        cache.append_rows([], torch.zeros(0, 1, 8))
    with pytest.raises(RuntimeError, match="captured"):
        cache.evict_rows([], torch.zeros(0, 8), torch.zeros(0, 8, dtype=torch.int32), budget=1)


def test_evict_tables_without_columns():
    """No slots: the inputs may be NULL, outputs that are filled may not."""
    lib = L.load()

    def rc(**kw):
        none = dict(page_table_width=0, page_table=None, w_in=None, pos_in=None, in_width=0)
        return lib.ck_evict_by_weight(_evict(**{**none, **kw}), 0, 0, 0)

    assert rc(B=0) == L.CK_OK
    for missing in ("w_out", "pos_out", "lengths", "lengths_out"):
        assert rc(**{missing: None}) == L.CK_ERR_INVALID_ARG
