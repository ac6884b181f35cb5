"""The serving operators on sizes that reach each of their kernels' paths: lists of
many tiles a warp, warps that take several units in turn, every head layout of the
streaming kernels, clusters of 16 that select, K split over 8 CTAs.

References are in float64 on the device; the tolerances are those that
test_gpu_paged_attention.py and test_gpu_lora.py derive.
"""

from __future__ import annotations

import pytest
import torch

from cortex import _lib as L
from cortex.kernels.kv_evict import evict_by_weight
from cortex.kernels.lora import lora_linear
from cortex.kernels.paged_attention import paged_attention

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
BF, F = torch.bfloat16, torch.float32


# ── paged_attention ──────────────────────────────────────────────────────────


def attention_state(lens, H, Hkv, Dh, page, dtype, seed=0):
    """(q, pool, table, lengths, rows of every sequence): scattered pages, NaN in
    every row that is not live, wild entries behind the last page."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    need = [-(-n // page) for n in lens]
    pages = sum(need) + 2
    order = torch.randperm(pages, generator=g, device=DEV)
    table = torch.full((len(lens), max(max(need), 1)), 2 ** 31 - 1, dtype=torch.int32, device=DEV)
    pool = torch.full((pages * page, 2 * Hkv * Dh), float("nan"), dtype=dtype, device=DEV)
    at, rows = 0, []
    for b, n in enumerate(lens):
        own = order[at:at + need[b]]
        table[b, :need[b]] = own.int()
        r = torch.randn(n, 2 * Hkv * Dh, generator=g, device=DEV).to(dtype)
        j = torch.arange(n, device=DEV)
        pool[own[j // page] * page + j % page] = r
        rows.append(r)
        at += need[b]
    q = (1.5 * torch.randn(len(lens), H, Dh, generator=g, device=DEV)).to(dtype)
    return (q, pool.view(pages, page, -1), table,
            torch.tensor(lens, dtype=torch.int32, device=DEV), rows)


def check_attention(lens, H, Hkv, Dh, page, dtype, seed=0):
    q, pool, table, lengths, rows = attention_state(lens, H, Hkv, Dh, page, dtype, seed)
    cap = table.shape[1] * page
    base = torch.rand(len(lens), cap + 5, device=DEV)
    out = paged_attention(q, pool, table, lengths)
    out_w, acc = paged_attention(q, pool, table, lengths, weights=base)
    bf = dtype == BF
    for b, n in enumerate(lens):
        assert torch.equal(acc[b, n:], base[b, n:])
        if n == 0:
            assert not bool(out[b].any()) and not bool(out_w[b].any())
            continue
        k, v = rows[b].double().reshape(n, 2, Hkv, Dh).unbind(1)
        qb = q[b].double().reshape(Hkv, H // Hkv, Dh)
        s = torch.einsum("kgd,nkd->kgn", qb, k) * Dh ** -0.5
        M = (torch.einsum("kgd,nkd->kgn", qb.abs(), k.abs()) * Dh ** -0.5).amax(2, keepdim=True)
        p = torch.softmax(s, 2)
        rel = 4 * (Dh + 8) * U * M + (8 + 2 * n) * U
        o = torch.einsum("kgn,nkd->kgd", p, v)
        A = torch.einsum("kgn,nkd->kgd", p, v.abs())
        tol = (rel + (2.0 ** -8 if bf else 0)) * A + (2.0 ** -8 if bf else U) * o.abs() + 1e-30
        for got in (out[b], out_w[b]):
            err = (got.double().reshape(Hkv, H // Hkv, Dh) - o).abs()
            assert bool((err <= tol).all()), (b, n, float((err / tol).max()))
        w = base[b, :n].double() + p.sum((0, 1))
        wtol = (p * (rel + 2 * H * U) + 2.0 ** -126).sum((0, 1)) + U * w
        err = (acc[b, :n].double() - w).abs()
        assert bool((err <= wtol).all()), (b, n, float((err / wtol).max()))
    assert L.device_status()[0] == 0


def ragged(B, longest, seed):
    """Lengths over the whole range, every fourth sequence empty, ends on and off tiles."""
    g = torch.Generator().manual_seed(seed)
    lens = torch.randint(1, longest + 1, (B,), generator=g)
    lens[3::4] = 0
    lens[1], lens[2] = longest, 32 * (longest // 64)
    return lens.tolist()


# several times more tiles than the 1184 (1776 for rows of 64 bytes) warps take runs of
@pytest.mark.parametrize("B,longest,H,Hkv,Dh,page,dtype", [
    (40, 4096, 12, 12, 64, 64, BF),
    (40, 4096, 12, 12, 64, 24, F),
    (23, 5000, 16, 4, 128, 64, BF),
    (17, 3000, 8, 2, 128, 16, F),
    (64, 3000, 8, 8, 32, 128, BF),
    (31, 4000, 32, 16, 32, 48, F),
    (9, 9000, 4, 2, 96, 64, BF),
    (9, 4000, 3, 3, 40, 64, F),
])
def test_runs_of_many_tiles(B, longest, H, Hkv, Dh, page, dtype):
    check_attention(ragged(B, longest, seed=B), H, Hkv, Dh, page, dtype)


@pytest.mark.parametrize("Hkv,Dh,dtype", [(1800, 32, BF), (1200, 64, BF), (1200, 32, F),
                                          (2500, 64, BF)])
def test_more_units_than_warps(Hkv, Dh, dtype):
    check_attention([70, 0, 3, 33, 0, 0], Hkv, Hkv, Dh, 16, dtype)


@pytest.mark.parametrize("dtype,H,Hkv", [(BF, 3, 3), (BF, 9, 1), (BF, 24, 2), (BF, 16, 1), (BF, 40, 2),
                                         (F, 3, 3), (F, 4, 1), (F, 10, 2)])
@pytest.mark.parametrize("Dh", [32, 64, 128])
@pytest.mark.parametrize("lens", [[200, 1, 0, 33], [255, 16], [2100, 700, 0, 5]])
def test_head_layouts(dtype, H, Hkv, Dh, lens):
    """One launch (short tables) and a list, every width of the heads' operand."""
    check_attention(lens, H, Hkv, Dh, 16, dtype, seed=H)


# ── evict_by_weight ──────────────────────────────────────────────────────────


def kept_order(w, pos, budget, recent):
    """Slots of a sequence by rank, best first: newest, weight, slot."""
    safe = pos.long() > int(pos.max()) - recent
    order = torch.argsort(w, descending=True, stable=True)
    return order[torch.argsort(~safe[order], stable=True)][:budget]


@pytest.mark.parametrize("lens,page,width,budget,recent", [
    ([131072], 128, 8, 20000, 1024),          # 16 CTAs, keys in shared memory
    ([70001, 66000, 5], 64, 16, 65000, 7),    # three such clusters, few moves a list
    ([900001], 256, 2, 333333, 1000),         # more keys than 16 CTAs hold
    ([100000, 40000], 100, 4, 99990, 0),      # a handful of moves after 16 CTAs
])
@pytest.mark.parametrize("ties", [False, True])
def test_selection_by_sixteen_ctas(lens, page, width, budget, recent, ties):
    g = torch.Generator(device=DEV).manual_seed(len(lens))
    need = [-(-n // page) for n in lens]
    order = torch.randperm(sum(need) + 1, generator=g, device=DEV)
    table = torch.full((len(lens), max(need)), 2 ** 31 - 1, dtype=torch.int32, device=DEV)
    at = 0
    for b, k in enumerate(need):
        table[b, :k] = order[at:at + k].int()
        at += k
    slots = max(need) * page
    pool = torch.randn(len(order), page, width, generator=g, device=DEV)
    w = torch.rand(len(lens), slots, generator=g, device=DEV)
    if ties:
        w = (w * 5).floor()
    pos = torch.stack([torch.randperm(slots, generator=g, device=DEV) for _ in lens]).int()
    lengths = torch.tensor(lens, dtype=torch.int32, device=DEV)
    want = pool.view(-1, width).clone()
    want_w, want_p = w.clone(), pos.clone()
    for b, n in enumerate(lens):
        if n <= budget:
            continue
        kept = torch.zeros(n, dtype=torch.bool, device=DEV)
        kept[kept_order(w[b, :n], pos[b, :n], budget, recent)] = True
        holes = (~kept[:budget]).nonzero().flatten()
        movers = budget + kept[budget:].nonzero().flatten()
        place = lambda j: table[b, j // page].long() * page + j % page  # noqa: E731
        want[place(holes)] = want[place(movers)]
        want_w[b, holes], want_p[b, holes] = w[b, movers], pos[b, movers]
    short = torch.minimum(lengths, torch.full_like(lengths, budget))
    live = torch.arange(budget, device=DEV) < short[:, None]
    cols = min(budget, slots)
    pool2 = pool.clone()
    n1, w1, p1 = evict_by_weight(pool, table, lengths, w, pos, budget=budget, recent=recent)
    assert torch.equal(pool.view(-1, width), want) and torch.equal(n1, short)
    assert torch.equal(w1, torch.where(live[:, :cols], want_w[:, :cols], 0))
    assert torch.equal(p1, torch.where(live[:, :cols], want_p[:, :cols], -1))
    evict_by_weight(pool2, table, lengths, w, pos, budget=budget, recent=recent,
                    out=(lengths, w, pos))
    assert torch.equal(pool2, pool) and torch.equal(lengths, short)
    assert torch.equal(w, want_w) and torch.equal(pos, want_p)
    assert L.device_status()[0] == 0


# ── lora_linear ──────────────────────────────────────────────────────────────


@pytest.mark.parametrize("M,K,N,rank,n,run", [
    (200, 2048, 520, 16, 5, 7),      # h by 8 CTAs of a tile, every width of its columns
    (200, 2048, 520, 24, 5, 64),
    (200, 2056, 520, 64, 5, 40),
    (130, 1024, 264, 100, 9, 1),
    (64, 4096, 512, 32, 9, 3),       # rows: 8 CTAs, 64 rows of x an operand
    (128, 2048, 1000, 16, 4, 5),     # two operands of rows
])
def test_k_over_eight_ctas(M, K, N, rank, n, run):
    g = torch.Generator(device=DEV).manual_seed(M)
    x = torch.randn(M, K, generator=g, device=DEV).to(BF)
    w = (torch.randn(N, K, generator=g, device=DEV) * K ** -0.5).to(BF)
    a = (torch.randn(n, rank, K, generator=g, device=DEV) * K ** -0.5).to(BF)
    b = (torch.randn(n, N, rank, generator=g, device=DEV) * rank ** -0.5).to(BF)
    ids = ((torch.arange(M, device=DEV) // run) % (n + 1) - 1).int()
    got = lora_linear(x, w, a, b, ids)
    own = ids.long().clamp(min=0)
    has = (ids >= 0)[:, None].double()
    y = x.double() @ w.double().t()
    P = x.double().abs() @ w.double().abs().t()
    h = torch.einsum("mk,mrk->mr", x.double(), a.double()[own])
    y += has * torch.einsum("mr,mnr->mn", h, b.double()[own])
    hb = has * torch.einsum("mr,mnr->mn", h.abs(), b.double().abs()[own])
    P += has * torch.einsum("mr,mnr->mn", torch.einsum("mk,mrk->mr", x.double().abs(),
                                                      a.double().abs()[own]), b.double().abs()[own])
    tol = (K + rank + 4) * U * P + 2.0 ** -8 * y.abs() + 2.0 ** -8 * hb
    err = (got.double() - y).abs()
    assert bool((err <= tol).all()), float((err / tol).max())
    assert L.device_status()[0] == 0
