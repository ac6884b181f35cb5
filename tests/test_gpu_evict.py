"""evict_by_weight on the GPU against its definition, exactly: everything it
writes is a copy of something it reads."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from cortex import _lib as L
from cortex.kernels.kv_evict import evict_by_weight

pytestmark = pytest.mark.gpu
DEV = "cuda"


def make(lens, page, width, dtype, seed=0, weights="spread", extra=0, pages_wide=None):
    rng = np.random.default_rng(seed)
    B = len(lens)
    need = [-(-n // page) for n in lens]
    pages = sum(need) + 2
    perm = rng.permutation(pages)
    tw = max(max(need), 1) if pages_wide is None else pages_wide
    table = np.full((B, tw), 2 ** 31 - 1, np.int32)
    at = 0
    for b in range(B):
        table[b, :need[b]] = perm[at:at + need[b]]
        at += need[b]
    slots = tw * page + extra
    pool = torch.from_numpy(rng.standard_normal((pages, page, width)).astype(np.float32))
    w = {"spread": lambda: np.exp(2 * rng.standard_normal((B, slots))),
         "few": lambda: rng.integers(0, 4, (B, slots)).astype(float),
         "equal": lambda: np.full((B, slots), 0.25),
         "wild": lambda: rng.choice([np.nan, -np.nan, np.inf, -np.inf, 0.0, -0.0, 1e-45, -1e-45,
                                     3e38, -3e38, 1.0], (B, slots))}[weights]().astype(np.float32)
    pos = np.stack([rng.permutation(slots) for _ in range(B)]).astype(np.int32)
    return (pool.to(dtype).to(DEV), torch.from_numpy(table).to(DEV),
            torch.tensor(lens, dtype=torch.int32, device=DEV), torch.from_numpy(w).to(DEV),
            torch.from_numpy(pos).to(DEV))


def rank_key(w):
    """Weights as numbers to sort by: NaN below everything, -0 equal to 0."""
    return np.where(np.isnan(w), -np.inf, w.astype(np.float64)), ~np.isnan(w)


def want(pool, table, lengths, w, pos, budget, recent):
    pool, table = pool.clone().cpu(), table.cpu().numpy()
    w, pos, lens = w.cpu().numpy().copy(), pos.cpu().numpy().copy(), lengths.tolist()
    page = pool.shape[1]
    out = []
    for b, n in enumerate(lens):
        if n > budget:
            safe = pos[b, :n].astype(np.int64) > int(pos[b, :n].max()) - recent
            value, real = rank_key(w[b, :n])
            order = np.lexsort((np.arange(n), -value, ~real, ~safe))
            kept = np.zeros(n, bool)
            kept[order[:budget]] = True
            holes, movers = np.flatnonzero(~kept[:budget]), budget + np.flatnonzero(kept[budget:])
            assert len(holes) == len(movers)
            for h, m in zip(holes, movers):
                pool[table[b, h // page], h % page] = pool[table[b, m // page], m % page]
                w[b, h], pos[b, h] = w[b, m], pos[b, m]
        out.append(min(n, budget))
    return pool, out, w, pos


def same(a, b):
    """Equal bit for bit (NaNs and signs of zero included)."""
    a, b = a.contiguous().cpu(), b.contiguous().cpu()
    kind = {4: torch.int32, 2: torch.int16}[a.element_size()]
    return a.shape == b.shape and torch.equal(a.view(kind), b.view(kind))


def run_case(state, budget, recent):
    pool, table, lengths, w, pos = state
    pool_x, lens_x, w_x, pos_x = want(*state, budget, recent)
    pool_in = pool.clone()
    n1, w1, p1 = evict_by_weight(pool, table, lengths, w, pos, budget=budget, recent=recent)
    assert same(pool, pool_x)
    assert n1.tolist() == lens_x
    assert w1.shape == p1.shape == (len(lens_x), budget)
    for b, n in enumerate(lens_x):
        assert same(w1[b, :n], torch.from_numpy(w_x[b, :n]))
        assert p1[b, :n].tolist() == pos_x[b, :n].tolist()
        assert bool((w1[b, n:] == 0).all()) and bool((p1[b, n:] == -1).all())
    # in place: the same, and nothing behind the new lengths changes
    lens2, w2, pos2 = lengths.clone(), w.clone(), pos.clone()
    got = evict_by_weight(pool_in, table, lens2, w2, pos2, budget=budget, recent=recent,
                          out=(lens2, w2, pos2))
    assert got[0] is lens2 and same(pool_in, pool_x) and lens2.tolist() == lens_x
    assert same(w2, torch.from_numpy(w_x)) and same(pos2, torch.from_numpy(pos_x))
    assert L.device_status()[0] == 0


CASES = [
    # lens, page, width, dtype, budget, recent, weights
    ([513] * 5, 64, 128, torch.bfloat16, 512, 64, "spread"),
    ([0, 1, 9, 10, 11, 30, 100], 7, 24, torch.float32, 10, 3, "spread"),
    ([2, 3], 1, 8, torch.float32, 1, 0, "spread"),
    ([2, 3], 1, 8, torch.float32, 1, 1, "few"),
    ([300, 299, 64], 16, 16, torch.bfloat16, 64, 64, "few"),
    ([1000, 37], 24, 5, torch.bfloat16, 333, 10, "equal"),
    ([1000, 700], 24, 6, torch.bfloat16, 333, 10, "wild"),
    ([1000, 4096, 70], 64, 3, torch.float32, 1, 0, "wild"),
    ([4096, 4095, 33], 64, 40, torch.float32, 4000, 0, "spread"),
    ([4097, 5000, 200, 0], 64, 8, torch.bfloat16, 300, 17, "spread"),
    ([9000, 8999], 24, 264, torch.bfloat16, 8000, 4000, "few"),
    ([33000], 128, 8, torch.float32, 5, 2, "equal"),
    ([20000, 6], 100, 8, torch.float32, 19999, 0, "wild"),
    ([300, 290, 151], 16, 2056, torch.bfloat16, 150, 9, "spread"),
    ([290, 151, 10], 16, 2050, torch.bfloat16, 150, 9, "few"),
    ([140, 100], 16, 4000, torch.bfloat16, 70, 9, "spread"),
]


@pytest.mark.parametrize("lens,page,width,dtype,budget,recent,weights", CASES)
def test_against_definition(lens, page, width, dtype, budget, recent, weights):
    run_case(make(lens, page, width, dtype, weights=weights, extra=3), budget, recent)


def test_more_slots_than_shared_memory_holds():
    run_case(make([450001] + [100] * 9, 512, 2, torch.float32, weights="few"), 77777, 50)


def test_many_moves_of_long_rows():
    run_case(make([32768, 20], 128, 1024, torch.float32), 16384, 100)


def test_more_sequences_than_a_list_holds():
    rng = np.random.default_rng(5)
    run_case(make(rng.integers(0, 300, 1100).tolist(), 60, 8, torch.bfloat16), 150, 7)


def test_budget_beyond_the_table():
    run_case(make([30, 5], 16, 8, torch.float32), 500, 7)


def test_strided_pool_and_tables():
    pool, table, lengths, w, pos = make([90, 50], 16, 8, torch.bfloat16, seed=3)
    wide = torch.zeros(pool.shape[0], 18, 20, dtype=pool.dtype, device=DEV)
    view = wide[:, 1:17, 5:13]
    view.copy_(pool)
    x = want(pool, table, lengths, w, pos, 40, 4)
    t2 = torch.full((2, 2 * table.shape[1]), -9, dtype=torch.int32, device=DEV)
    t2[:, ::2] = table
    n, w1, p1 = evict_by_weight(view, t2[:, ::2], torch.stack([lengths, lengths], 1)[:, 0],
                                torch.cat([w, w], 1)[:, :w.shape[1]], pos, budget=40, recent=4)
    assert same(view, x[0]) and n.tolist() == x[1]
    assert same(w1, torch.from_numpy(x[2][:, :40])) and same(p1, torch.from_numpy(x[3][:, :40]))
    assert bool((wide[:, 0] == 0).all()) and bool((wide[:, :, :5] == 0).all())
    assert bool((wide[:, 17] == 0).all()) and bool((wide[:, :, 13:] == 0).all())


def test_positions_at_the_ends_of_their_range():
    pool, table, lengths, w, pos = make([40], 16, 8, torch.float32)
    pos[0, :40] = torch.arange(-2 ** 31, -2 ** 31 + 40, device=DEV, dtype=torch.int64).int()
    run_case((pool.clone(), table, lengths, w, pos), 20, 20)
    pos[0, 7] = 2 ** 31 - 1
    run_case((pool, table, lengths, w, pos), 20, 20)


def test_bad_lengths_and_pages_are_recorded():
    pool, table, lengths, w, pos = make([60, 60, 60], 16, 8, torch.float32)
    cap = table.shape[1] * 16
    x = want(pool, table, lengths, w, pos, 20, 2)
    for bad in (-1, cap + 1, 2 ** 31 - 1, -2 ** 31):
        p, n = pool.clone(), lengths.clone()
        n[1] = bad
        n1, w1, p1 = evict_by_weight(p, table, n, w, pos, budget=20, recent=2)
        with pytest.raises(IndexError):
            L.check_device_status("evict_by_weight")
        assert n1.tolist() == [20, bad, 20]
        assert bool((w1[1] == 0).all()) and bool((p1[1] == -1).all())
        own = table[1, :4].long()
        assert same(p[own], pool[own])
        for b in (0, 2):
            assert same(p[table[b, :4].long()], x[0][table[b, :4].long().cpu()])
    for page in (-1, pool.shape[0], 2 ** 31 - 1):
        p, t = pool.clone(), table.clone()
        t[1, 0] = page
        n1, w1, p1 = evict_by_weight(p, t, lengths, w, pos, budget=20, recent=2)
        with pytest.raises(IndexError):
            L.check_device_status("evict_by_weight")
        assert n1.tolist() == [20, 20, 20] and same(p1, torch.from_numpy(x[3][:, :20]))
        assert same(p[table[1, 0].long()], pool[table[1, 0].long()])


def test_capture_replay_and_streams():
    states = [make([700, 20, 300], 16, 24, torch.bfloat16, seed=i, pages_wide=300)
              for i in range(3)]
    pages = max(s[0].shape[0] for s in states)
    pool = torch.zeros(pages, 16, 24, dtype=torch.bfloat16, device=DEV)
    table, lengths, w, pos = (torch.zeros_like(t) for t in states[0][1:])
    evict_by_weight(pool, table, lengths, w, pos, budget=100, recent=10)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        with torch.cuda.graph(graph, stream=s):
            out = evict_by_weight(pool, table, lengths, w, pos, budget=100, recent=10)
    for st in states:
        pool[:st[0].shape[0]] = st[0]
        for dst, src in zip((table, lengths, w, pos), st[1:]):
            dst.copy_(src)
        x = want(*st, 100, 10)
        graph.replay()
        torch.cuda.synchronize()
        assert same(pool[:st[0].shape[0]], x[0]) and out[0].tolist() == x[1]
        for b, n in enumerate(x[1]):
            assert out[2][b, :n].tolist() == x[3][b, :n].tolist()
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    for st, q in zip(states, streams):
        with torch.cuda.stream(q):
            evict_by_weight(*st, budget=100, recent=10)
    torch.cuda.synchronize()
    for i, st in enumerate(states):
        fresh = make([700, 20, 300], 16, 24, torch.bfloat16, seed=i, pages_wide=300)
        assert same(st[0], want(*fresh, 100, 10)[0])
    assert L.device_status()[0] == 0


def test_refusals():
    pool, table, lengths, w, pos = make([30, 30], 16, 8, torch.float32)
    ok = dict(budget=10, recent=2)
    for bad in (dict(budget=0), dict(budget=5, recent=6), dict(budget=5, recent=-1)):
        with pytest.raises(ValueError):
            evict_by_weight(pool, table, lengths, w, pos, **bad)
    with pytest.raises(TypeError):
        evict_by_weight(pool, table, lengths, w.double(), pos, **ok)
    with pytest.raises(TypeError):
        evict_by_weight(pool, table, lengths, w, pos.long(), **ok)
    with pytest.raises(TypeError):
        evict_by_weight(pool, table, lengths.long(), w, pos, **ok)
    with pytest.raises(ValueError):
        evict_by_weight(pool, table, lengths, w[:, :31], pos, **ok)
    with pytest.raises(ValueError):
        evict_by_weight(pool, table[:1], lengths, w, pos, **ok)
    with pytest.raises(ValueError):
        evict_by_weight(pool, table, lengths, w, pos, out=(lengths, w[:, :9], pos), **ok)
    with pytest.raises(NotImplementedError):
        evict_by_weight(pool.half(), table, lengths, w, pos, **ok)
    with pytest.raises(RuntimeError):
        evict_by_weight(pool.cpu(), table, lengths, w, pos, **ok)
    empty = evict_by_weight(pool, table[:0], lengths[:0], w[:0], pos[:0], **ok)
    assert empty[0].shape == (0,) and empty[1].shape == (0, 10)


def test_outputs_apart_from_inputs():
    pool, table, lengths, w, pos = make([30, 30], 16, 8, torch.float32)
    ok = dict(budget=10, recent=2)
    fresh = lambda: (lengths.clone(), w.clone(), pos.clone())  # noqa: E731
    for i, bad in ((0, torch.zeros(1, dtype=torch.int32, device=DEV).expand(2)),
                   (1, w[:, 1:12]), (1, pos.view(torch.float32)), (2, w.view(torch.int32)),
                   (1, torch.zeros(1, 10, device=DEV).expand(2, 10))):
        out = list(fresh())
        out[i] = bad
        with pytest.raises(ValueError):
            evict_by_weight(pool, table, lengths, w, pos, out=tuple(out), **ok)
    n1, w1, p1 = fresh()
    with pytest.raises(ValueError):
        evict_by_weight(pool, table, lengths, w, pos, out=(n1, p1.view(torch.float32), p1), **ok)
    with pytest.raises(ValueError):
        evict_by_weight(pool[:1].expand(4, 16, 8), table, lengths, w, pos, **ok)
    state = make([30, 30], 16, 8, torch.float32)
    assert same(pool, state[0])


@pytest.mark.parametrize("dtype,width", [(torch.bfloat16, 1024), (torch.float32, 24),
                                         (torch.bfloat16, 33)])
def test_rows_past_four_gigabytes(dtype, width):
    """Pages whose elements lie more than 2^31 elements from the pool's start."""
    pool, table, lengths, w, pos = make([900, 333, 1], 16, width, dtype)
    x = want(pool, table, lengths, w, pos, 100, 10)
    first = 2 ** 31 // (16 * width) + 5
    big = torch.empty(first + len(pool), 16, width, dtype=dtype, device=DEV)
    big[first:] = pool
    wide = torch.where(table < len(pool), table + first, table)
    n, w1, p1 = evict_by_weight(big, wide, lengths, w, pos, budget=100, recent=10)
    assert same(big[first:], x[0]) and n.tolist() == x[1]
    for b, k in enumerate(x[1]):
        assert same(w1[b, :k], torch.from_numpy(x[2][b, :k]))
        assert p1[b, :k].tolist() == x[3][b, :k].tolist()


def test_the_largest_budget():
    """Tables of INT32_MAX columns: the columns behind the rows are filled to the end."""
    pool, table, lengths, w, pos = make([7], 16, 8, torch.float32)
    n, w1, p1 = evict_by_weight(pool, table, lengths, w, pos, budget=2 ** 31 - 1)
    assert n.tolist() == [7] and same(w1[0, :7], w[0, :7]) and same(p1[0, :7], pos[0, :7])
    assert not bool(w1[0, 7:].any()) and int(p1[0, 7:].max()) == int(p1[0, 7:].min()) == -1


def test_tables_without_columns():
    """Sequences without a page: nothing to evict, and lengths other than 0 are bad."""
    pool, table, lengths, w, pos = make([30, 5], 16, 8, torch.float32)
    none = (pool, table[:, :0], torch.zeros_like(lengths), w[:, :0], pos[:, :0])
    before = pool.clone()
    n, w1, p1 = evict_by_weight(*none, budget=3, recent=1)
    assert n.tolist() == [0, 0] and w1.tolist() == [[0] * 3] * 2 and p1.tolist() == [[-1] * 3] * 2
    got = evict_by_weight(*none, budget=3, out=(none[2], none[3], none[4]))
    assert got[0].tolist() == [0, 0] and got[1].shape == (2, 0)
    fresh = evict_by_weight(*none, budget=3, out=(torch.ones_like(lengths), w.clone(), pos.clone()))
    assert fresh[0].tolist() == [0, 0] and same(fresh[1], w) and same(fresh[2], pos)
    assert L.device_status()[0] == 0
    n, _, _ = evict_by_weight(pool, table[:, :0], lengths, w[:, :0], pos[:, :0], budget=3)
    with pytest.raises(IndexError):
        L.check_device_status("evict_by_weight")
    assert n.tolist() == lengths.tolist() and same(pool, before)
