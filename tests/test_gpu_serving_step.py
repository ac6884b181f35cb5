"""The serving operators together, as a token-by-token server uses them: adapted
projections make every session's query and K|V row, the rows go into the paged
cache, attention reads them and adds up what each position received, eviction
keeps every session inside its budget."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from cortex import _lib as L
from cortex.cache import StreamingKVCache
from cortex.kernels.kv_evict import evict_by_weight
from cortex.kernels.lora import lora_linear
from cortex.kernels.paged_attention import paged_attention

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24


def projections(g, D, H, Hkv, Dh, n, rank, dtype):
    def rnd(*shape, scale):
        return (torch.randn(*shape, generator=g) * scale).to(dtype).to(DEV)

    wide = H * Dh + 2 * Hkv * Dh
    return (rnd(wide, D, scale=1.5 * D ** -0.5), rnd(n, rank, D, scale=D ** -0.5),
            rnd(n, wide, rank, scale=rank ** -0.5), torch.rand(n, generator=g).to(DEV))


def exact_projection(x, w, a, b, ids, s):
    x, w, a, b, s = (t.double().cpu() for t in (x, w, a, b, s))
    y, P, hb = x @ w.t(), x.abs() @ w.abs().t(), torch.zeros(len(x), len(w)).double()
    for m, i in enumerate(ids.tolist()):
        if i >= 0:
            h = s[i] * (a[i] @ x[m])
            y[m] += b[i] @ h
            P[m] += s[i] * (b[i].abs() @ (a[i].abs() @ x[m].abs()))
            hb[m] = b[i].abs() @ h.abs()
    return y, P, hb


@pytest.mark.parametrize("dtype,H,Hkv", [(torch.bfloat16, 8, 8), (torch.bfloat16, 8, 2),
                                         (torch.float32, 4, 4)])
def test_a_server_of_many_steps(dtype, H, Hkv):
    g = torch.Generator().manual_seed(3)
    D, Dh, page, budget, recent, steps, rank, n = 256, 64, 8, 24, 6, 40, 16, 5
    half = 2.0 ** -8 if dtype == torch.bfloat16 else U
    cache = StreamingKVCache(40, page, 2 * Hkv * Dh, dtype, DEV)
    first = [0, 3, 30, 8, 24]  # rows that the sessions start with
    B = len(first)
    metas = [cache.write_rows(f"s{b}", 0, k) for b, k in enumerate(first)]
    store = []  # the sessions' rows, as the cache should hold them, in slot order
    for m in metas:
        rows = torch.randn(m.n_events, 2 * Hkv * Dh, generator=g).to(dtype).to(DEV)
        for k, p in enumerate(m.pages):
            cache.pool[p, :len(rows[k * page:(k + 1) * page])] = rows[k * page:(k + 1) * page]
        store.append(rows.cpu())
    w, a, b, s = projections(g, D, H, Hkv, Dh, n, rank, dtype)
    ids = torch.tensor([0, 4, -1, 2, 4], dtype=torch.int32, device=DEV)
    slots = 8 * page
    weights = torch.zeros(B, slots, device=DEV)
    positions = torch.arange(slots, dtype=torch.int32, device=DEV).repeat(B, 1)
    nxt = list(first)  # each session's next position
    for step in range(steps):
        x = torch.randn(B, D, generator=g).to(dtype).to(DEV)
        qkv = lora_linear(x, w, a, b, ids, scaling=s)
        y, P, hb = exact_projection(x, w, a, b, ids, s)
        tol = (D + rank + 4) * U * P + half * y.abs() + (2.0 ** -8 * hb if half > U else 0)
        assert bool(((qkv.double().cpu() - y).abs() <= tol).all())
        q = qkv[:, :H * Dh].reshape(B, H, Dh)
        cache.append_rows(metas, qkv[:, None, H * Dh:])
        for i, m in enumerate(metas):
            store[i] = torch.cat([store[i], qkv[i:i + 1, H * Dh:].cpu()])
            positions[i, m.n_events - 1] = nxt[i]
            weights[i, m.n_events - 1] = 0
            nxt[i] += 1
        table, lengths = cache.page_table(metas)
        assert lengths.tolist() == [len(r) for r in store]
        before = weights.clone()
        out, _ = paged_attention(q, cache.pool, table, lengths, weights=weights,
                                 weights_out=weights)
        for i in range(B):
            k, v = store[i].double().reshape(-1, 2, Hkv, Dh).unbind(1)
            nr = len(k)
            add = torch.zeros(nr).double()
            for h in range(H):
                kk, vv = k[:, h // (H // Hkv)], v[:, h // (H // Hkv)]
                qh = q[i, h].double().cpu()
                p = torch.softmax(kk @ qh / 8, 0)
                M = float((kk.abs() @ qh.abs()).max()) / 8
                rel = 4 * (Dh + 8) * U * M + (8 + 2 * nr) * U
                o = p @ vv
                bound = (rel + (2.0 ** -8 if half > U else 0)) * (p @ vv.abs()) + half * o.abs()
                assert bool(((out[i, h].double().cpu() - o).abs() <= bound).all())
                add += p
            got = (weights[i, :nr] - before[i, :nr]).double().cpu()
            # (the difference of two fp32 sums: their roundings besides rel)
            slack = add * (rel + 2 * H * U) + 2 * U * weights[i, :nr].double().cpu() + 2.0 ** -126
            assert bool(((got - add).abs() <= slack).all())
            assert torch.equal(weights[i, nr:], before[i, nr:])
        # which rows go, from the weights as they are
        wh, ph = weights.cpu().numpy(), positions.cpu().numpy()
        cache.evict_rows(metas, weights, positions, budget=budget, recent=recent)
        for i, m in enumerate(metas):
            nr = len(store[i])
            if nr > budget:
                safe = ph[i, :nr] > ph[i, :nr].max() - recent
                order = np.lexsort((np.arange(nr), -wh[i, :nr], ~safe))
                kept = np.zeros(nr, bool)
                kept[order[:budget]] = True
                holes = np.flatnonzero(~kept[:budget])
                movers = budget + np.flatnonzero(kept[budget:])
                perm = np.arange(budget)
                perm[holes] = movers
                store[i] = store[i][torch.from_numpy(perm)]
                assert positions[i, :budget].tolist() == ph[i, perm].tolist()
                assert weights[i, :budget].tolist() == wh[i, perm].tolist()
            assert m.n_events == len(store[i]) and len(m.pages) == max(1, -(-m.n_events // page))
            held = cache.pool[m.pages].reshape(-1, 2 * Hkv * Dh)[:m.n_events].cpu()
            assert torch.equal(held, store[i])
    assert cache.pages_used == sum(len(m.pages) for m in metas)
    assert L.device_status()[0] == 0


def test_a_captured_step():
    """Projection, attention and eviction of a step in one graph, replayed."""
    g = torch.Generator().manual_seed(4)
    D, H, Dh, page, budget, B, n = 256, 4, 64, 16, 64, 6, 3
    pages = 5
    pool = torch.randn(B * pages, page, 2 * H * Dh, generator=g).bfloat16().to(DEV)
    table = torch.randperm(B * pages, generator=g).reshape(B, pages).int().to(DEV)
    lengths = torch.full((B,), budget + 1, dtype=torch.int32, device=DEV)
    weights = torch.rand(B, pages * page, generator=g).to(DEV)
    positions = torch.stack([torch.randperm(pages * page, generator=g) for _ in range(B)]).int().to(DEV)
    w, a, b, s = projections(g, D, H, H, Dh, n, 8, torch.bfloat16)
    x = torch.randn(B, D, generator=g).bfloat16().to(DEV)
    ids = torch.tensor([0, 1, 2, -1, 0, 1], dtype=torch.int32, device=DEV)

    def step(pool, lengths, weights, positions):
        q = lora_linear(x, w, a, b, ids, scaling=s)[:, :H * Dh].reshape(B, H, Dh)
        out, weights = paged_attention(q, pool, table, lengths, weights=weights)
        return out, evict_by_weight(pool, table, lengths, weights, positions, budget=budget,
                                    recent=4)

    step(pool.clone(), lengths, weights, positions)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    held = pool.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            out, kept = step(held, lengths, weights, positions)
    for seed in range(3):
        g.manual_seed(seed)
        x.copy_(torch.randn(B, D, generator=g))
        weights.copy_(torch.rand(B, pages * page, generator=g))
        held.copy_(pool)
        graph.replay()
        torch.cuda.synchronize()
        fresh = pool.clone()
        want_out, want = step(fresh, lengths, weights, positions)
        assert torch.equal(out, want_out) and torch.equal(held, fresh)
        for p, q in zip(kept, want):
            assert torch.equal(p, q)
    assert L.device_status()[0] == 0


def test_cache_entries_grow_and_shrink():
    cache = StreamingKVCache(8, 4, 16, torch.float32, DEV)
    a, b = cache.write_rows("a", 0, 3), cache.write_rows("b", 0, 4)
    other = cache.write_rows("c", 0, 9)
    assert cache.pages_used == 5
    rows = torch.arange(2 * 7 * 16, dtype=torch.float32, device=DEV).reshape(2, 7, 16)
    cache.append_rows([a, b], rows)  # 3 + 7 rows: 3 pages; 4 + 7: 3 pages
    assert (a.n_events, b.n_events) == (10, 11) and (len(a.pages), len(b.pages)) == (3, 3)
    assert not cache.is_live(other) and cache.pages_used == 6  # "c" made room
    for m, r in ((a, rows[0]), (b, rows[1])):
        assert torch.equal(cache.pool[m.pages].reshape(-1, 16)[m.n_events - 7:m.n_events], r)
    with pytest.raises(RuntimeError):  # 3 more pages each, 2 can be had: nothing changes
        cache.append_rows([a, b], torch.zeros(2, 12, 16, device=DEV))
    assert (a.n_events, b.n_events) == (10, 11) and cache.pages_used == 6
    with pytest.raises(ValueError):
        cache.append_rows([a, a], torch.zeros(2, 1, 16, device=DEV))
    with pytest.raises(ValueError):
        cache.append_rows([other], torch.zeros(1, 1, 16, device=DEV))
    with pytest.raises(ValueError):
        cache.append_rows([a], torch.zeros(1, 1, 8, device=DEV))
    with pytest.raises(ValueError):
        cache.append_rows([a], torch.zeros(1, 1, 16, device=DEV, dtype=torch.bfloat16))
    table, lengths = cache.page_table([b, a, b])
    assert table.tolist() == [b.pages, a.pages, b.pages] and lengths.tolist() == [11, 10, 11]
    w = torch.arange(12, dtype=torch.float32, device=DEV).repeat(2, 1)
    pos = torch.arange(12, dtype=torch.int32, device=DEV).repeat(2, 1)
    with pytest.raises(ValueError):
        cache.evict_rows([a, a], w, pos, budget=4)
    cache.evict_rows([a, b], w, pos, budget=4)
    assert (a.n_events, b.n_events) == (4, 4) and (len(a.pages), len(b.pages)) == (1, 1)
    assert cache.pages_used == 2 and sorted(cache._free + a.pages + b.pages) == list(range(8))
    assert pos[0, :4].tolist() == [6, 7, 8, 9] and pos[1, :4].tolist() == [7, 8, 9, 10]
    cache.evict_session("a")
    with pytest.raises(ValueError):
        cache.page_table([a])
    cache.append_rows([], torch.zeros(0, 3, 16, device=DEV))
    cache.evict_rows([], w[:0], pos[:0], budget=4)


def test_an_edited_entry_is_not_a_windows_rows():
    """forward_streaming recomputes a window whose entry grew or shrank since."""
    from cortex.workloads import WORKLOADS, build_model, make_events

    wl = WORKLOADS["cfg1"]
    model = build_model(wl, DEV)
    ev = make_events(np.array([320]), seed=5)
    win = [{"session_id": "s", "bin_start": 0, "neuron_ids": ev["neuron_ids"],
            "time_bins": ev["time_bins"], "values": ev["values"]}]
    cache = StreamingKVCache(64, 64, 2 * wl.config.latent_dim, torch.bfloat16, DEV)
    with torch.no_grad():
        fresh = model.forward_streaming(win, cache)["behavior"]
        meta = cache.lookup("s", 0)
        cache.append_rows([meta], torch.randn(1, 1, cache.hidden_dim, device=DEV).bfloat16())
        w = torch.rand(1, len(meta.pages) * 64, device=DEV)
        pos = torch.arange(len(meta.pages) * 64, dtype=torch.int32, device=DEV)[None].clone()
        cache.evict_rows([meta], w, pos, budget=320)
        assert meta.n_events == 320  # as many rows as the window has events
        again = model.forward_streaming(win, cache)["behavior"]
        hit = model.forward_streaming(win, cache)["behavior"]
    assert torch.equal(fresh, again) and torch.equal(fresh, hit)


def test_rows_to_append_at_any_address():
    """Rows that begin off a 16-byte boundary arrive like others, over page ends too."""
    cache = StreamingKVCache(8, 4, 8, torch.float32, DEV)
    a, b = cache.write_rows("a", 0, 3), cache.write_rows("b", 0, 4)
    flat = torch.arange(2 * 6 * 8 + 1, dtype=torch.float32, device=DEV)
    rows = flat[1:].reshape(2, 6, 8)
    assert rows.data_ptr() % 16 != 0
    cache.append_rows([a, b], rows)
    for m, first, r in ((a, 3, rows[0]), (b, 4, rows[1])):
        assert (m.n_events, len(m.pages)) == (first + 6, 3)
        assert torch.equal(cache.pool[m.pages].reshape(-1, 8)[first:first + 6], r)
    assert L.device_status()[0] == 0


def test_rows_to_append_that_lie_in_the_pool():
    """Rows read from pages that the same call writes: they arrive as they were."""
    cache = StreamingKVCache(5, 4, 4096, torch.float32, DEV)
    a, b = cache.write_rows("a", 0, 4), cache.write_rows("b", 0, 12)
    cache.rows.copy_(torch.arange(20, device=DEV)[:, None].expand(20, 4096))
    assert (a.pages, b.pages) == ([4], [3, 2, 1])
    cache.append_rows([a], cache.rows[2:14][None])  # "b" makes room: its pages 1, 2 and 3
    assert a.pages == [4, 1, 2, 3] and not cache.is_live(b)
    got = cache.pool[a.pages].reshape(-1, 4096)
    assert got[:, 0].tolist() == [16, 17, 18, 19] + list(range(2, 14))
    assert torch.equal(got, got[:, :1].expand(16, 4096))
    assert L.device_status()[0] == 0


def test_a_rewritten_key_is_another_entry():
    """Rows written under the key of an entry that grew or shrank replace it: its
    PageMeta does not stand for the new rows, however many pages they take."""
    for n in (2, 4, 5):
        for rewrite in ("write_rows", "write"):
            cache = StreamingKVCache(8, 4, 16, torch.float32, DEV)
            a = cache.write_rows("a", 0, 3)
            cache.append_rows([a], torch.ones(1, 1, 16, device=DEV))
            if rewrite == "write_rows":
                new = cache.write_rows("a", 0, n)
            else:
                cache.write("a", 0, torch.zeros(n, 16, device=DEV))
                new = cache.lookup("a", 0)
            assert new is not a and not cache.is_live(a) and cache.is_live(new)
            assert not new.edited and new.n_events == (min(n, 4) if rewrite == "write" else n)
            with pytest.raises(ValueError):
                cache.page_table([a])
            assert cache.page_table([new])[1].tolist() == [new.n_events]
            assert sorted(cache._free + new.pages) == list(range(8))


def test_grown_rows_stay():
    """Rows that were appended exist nowhere else: nothing that makes room takes them."""
    cache = StreamingKVCache(6, 4, 16, torch.float32, DEV)
    a, b = cache.write_rows("a", 0, 4), cache.write_rows("b", 0, 4)
    rows = torch.arange(32, dtype=torch.float32, device=DEV).reshape(1, 2, 16)
    cache.append_rows([a], rows)
    kept = a.pages[1]
    assert cache.write_rows("c", 0, 16) is not None  # "b" makes room, "a" does not
    assert cache.is_live(a) and not cache.is_live(b) and cache.pages_used == 6
    assert cache.write_rows("d", 0, 17) is None and cache.pages_used == 6
    d = cache.write_rows("d", 0, 12)
    assert not cache.lookup("c", 0) and cache.is_live(a) and a.n_events == 6
    with pytest.raises(RuntimeError):  # 5 pages needed, 3 can be had: nothing changes
        cache.append_rows([a], torch.zeros(1, 20, 16, device=DEV))
    assert a.n_events == 6 and len(a.pages) == 2 and cache.is_live(d)
    cache.append_rows([a], torch.zeros(1, 18, 16, device=DEV))
    assert len(a.pages) == 6 and not cache.is_live(d)
    assert torch.equal(cache.pool[kept, :2], rows[0])
    assert cache.write_rows("d", 0, 1) is None  # "a" holds every page
    with pytest.raises(RuntimeError):
        cache.write("d", 0, torch.zeros(1, 16, device=DEV))
    cache.write("a", 0, torch.zeros(1, 16, device=DEV))  # its own key: replaced
    assert not cache.is_live(a) and cache.pages_used == 1
    e = cache.write_rows("e", 0, 9)
    pos = torch.arange(12, dtype=torch.int32, device=DEV)[None].clone()
    cache.evict_rows([e], torch.rand(1, 12, device=DEV), pos, budget=8)
    assert cache.write_rows("f", 0, 17) is None and cache.is_live(e)
    assert cache.evict_session("e") == 1 and cache.write_rows("f", 0, 17) is not None


def test_forward_streaming_leaves_edited_entries():
    from cortex.workloads import WORKLOADS, build_model, make_events

    wl = WORKLOADS["cfg1"]
    model = build_model(wl, DEV)
    wins = []
    for i in range(3):
        ev = make_events(np.array([200 + i]), seed=7 + i)
        wins.append({"session_id": f"s{i}", "bin_start": 0, "neuron_ids": ev["neuron_ids"],
                     "time_bins": ev["time_bins"], "values": ev["values"]})
    cache = StreamingKVCache(10, 64, 2 * wl.config.latent_dim, torch.bfloat16, DEV)
    with torch.no_grad():
        fresh = model.forward_streaming(wins, StreamingKVCache(64, 64, cache.hidden_dim,
                                                               torch.bfloat16, DEV))["behavior"]
        model.forward_streaming(wins[:1], cache)
        meta = cache.lookup("s0", 0)
        cache.append_rows([meta], torch.randn(1, 9, cache.hidden_dim, device=DEV).bfloat16())
        held = cache.pool[meta.pages].clone()
        for _ in range(2):  # 10 pages: "s0" and one of the others
            assert torch.equal(model.forward_streaming(wins, cache)["behavior"], fresh)
            assert cache.is_live(meta) and meta.n_events == 209
            assert torch.equal(cache.pool[meta.pages], held)
    assert L.device_status()[0] == 0


def test_cache_methods_are_not_captured():
    """They refuse, nothing changes, and the capture around them goes on."""
    cache = StreamingKVCache(8, 4, 16, torch.float32, DEV)
    a = cache.write_rows("a", 0, 3)
    rows, one = torch.ones(1, 2, 16, device=DEV), torch.ones(1, device=DEV)
    w, pos = torch.rand(1, 4, device=DEV), torch.zeros(1, 4, dtype=torch.int32, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            for call in (lambda: cache.page_table([a]), lambda: cache.append_rows([a], rows),
                         lambda: cache.evict_rows([a], w, pos, budget=1)):
                with pytest.raises(RuntimeError, match="captured"):
                    call()
            one.add_(1)
    graph.replay()
    torch.cuda.synchronize()
    assert one.tolist() == [2] and a.n_events == 3 and not a.edited and cache.pages_used == 1
    cache.append_rows([a], rows)
    assert cache.page_table([a])[1].tolist() == [5]
