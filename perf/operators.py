"""The serving operators that work on a batch of sessions, as calls to measure.

Three operators of one serving step: attention of one new token per session
over its paged K|V rows, eviction from those rows by accumulated attention
weight, and a projection that many sessions share beside each session's own
low-rank adapter. ``listed`` and ``draw`` give cases, ``prepare`` a case's
inputs, ``run`` one call, ``work`` what a call cannot do without and ``exact``
the same outputs from the definitions in 64 bits.

With ``own`` false, ``run`` computes the plain form in elementary torch
operations; with ``own`` true it calls the framework's kernels.
"""

from __future__ import annotations

import math
import os
import sys

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
BYTES = {"bf16": 2, "f32": 4}


def _cortex():
    """The framework's package (only imported where its kernels are called)."""
    path = os.path.abspath("cortex-engine_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    from cortex.kernels.kv_evict import evict_by_weight
    from cortex.kernels.lora import lora_linear
    from cortex.kernels.paged_attention import paged_attention

    return paged_attention, evict_by_weight, lora_linear


# ── cases ────────────────────────────────────────────────────────────────────


def _attn(name, B, heads, kv_heads, dh, page, lo, hi, dtype, weights):
    return {"name": name, "op": "paged_attention", "B": B, "heads": heads, "kv_heads": kv_heads,
            "dh": dh, "page": page, "len_min": lo, "len_max": hi, "dtype": dtype,
            "weights": weights}


def _evict(name, B, row, page, lo, hi, budget, recent, dtype):
    return {"name": name, "op": "evict", "B": B, "row": row, "page": page, "len_min": lo,
            "len_max": hi, "budget": budget, "recent": recent, "dtype": dtype}


def _lora(name, M, K, N, rank, adapters, run_len, dtype, bias):
    return {"name": name, "op": "lora", "M": M, "K": K, "N": N, "rank": rank,
            "adapters": adapters, "run_len": run_len, "dtype": dtype, "bias": bias}


def listed():
    return [
        # one session's newest token over a few hundred events (Cortex-S heads): latency
        _attn("attn_one_session", 1, 8, 8, 64, 64, 300, 300, "bf16", False),
        # a serving batch of ragged sessions (32 to 4096 events, Cortex-M heads), with the
        # accumulated weights that a later eviction reads
        _attn("attn_ragged_weights", 32, 12, 12, 64, 64, 32, 4096, "bf16", True),
        # long histories, four query heads to a K|V head
        _attn("attn_long_grouped", 16, 32, 8, 128, 64, 3000, 32768, "bf16", False),
        # the float32 model (Cortex-XS heads), small odd pages
        _attn("attn_f32", 24, 4, 4, 64, 24, 1, 2049, "f32", True),
        # steady state: every session is one row over its budget (Cortex-S rows)
        _evict("evict_step", 32, 1024, 64, 513, 513, 512, 64, "bf16"),
        # histories of very different lengths cut down to one budget
        _evict("evict_ragged", 24, 1536, 64, 700, 16384, 1000, 128, "bf16"),
        # one very long history, float32 rows
        _evict("evict_long", 1, 512, 128, 131072, 131072, 20000, 1024, "f32"),
        # one row through an adapted projection (Cortex-S qkv): latency
        _lora("lora_one_row", 1, 512, 1536, 16, 32, 1, "bf16", False),
        # one row each of many sessions, every row its own adapter, a wide projection
        _lora("lora_rows", 48, 4096, 4096, 16, 64, 1, "bf16", True),
        # a batch of 32 windows of 256 latents (Cortex-S qkv), an adapter per window
        _lora("lora_windows", 8192, 512, 1536, 16, 8, 256, "bf16", False),
        # Cortex-M latents of ragged requests, higher rank
        _lora("lora_ragged", 12001, 768, 2304, 32, 24, 333, "bf16", True),
        # the float32 model (Cortex-XS qkv), odd rows
        _lora("lora_f32", 301, 256, 768, 8, 5, 37, "f32", False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["paged_attention", "evict", "lora"])
    dtype = "f32" if rng.random() < 0.25 else "bf16"
    if op == "paged_attention":
        heads, kv = rng.choice([(4, 4), (8, 8), (12, 12), (8, 2), (16, 2), (32, 8), (8, 1), (6, 3)])
        dh = rng.choice([64, 64, 128, 32])
        page = rng.choice([16, 24, 64, 64, 128])
        hi = _log_int(rng, 1, 32768)
        lo = rng.choice([0, 1, max(1, hi // 100), hi])
        B = _log_int(rng, 1, 96)
        # no more rows than the longest listed batch holds
        cap = 16 * 12000 * 8 * 128 * 2
        B = max(1, min(B, int(cap / (max(hi, 1) * kv * dh * BYTES[dtype]))))
        return {"op": op, "B": B, "heads": heads, "kv_heads": kv, "dh": dh, "page": page,
                "len_min": min(lo, hi), "len_max": hi, "dtype": dtype,
                "weights": rng.random() < 0.5}
    if op == "evict":
        row = rng.choice([256, 512, 1024, 1536, 2048, 104])
        hi = _log_int(rng, 2, 131072)
        B = max(1, min(_log_int(rng, 1, 64), int(24 * 5000 * 1536 * 2 / (hi * row * BYTES[dtype]))))
        budget = max(1, int(hi * rng.uniform(0.05, 1.0)))
        return {"op": op, "B": B, "row": row, "page": rng.choice([16, 24, 64, 64, 128]),
                "len_min": max(1, int(hi * rng.choice([0.05, 0.5, 1.0]))), "len_max": hi,
                "budget": budget, "recent": int(budget * rng.choice([0.0, 0.1, 0.5])),
                "dtype": dtype}
    K = rng.choice([256, 512, 768, 1024, 2048, 4096, 520, 1000])
    N = rng.choice([256, 512, 768, 1536, 2304, 2048, 4096, 1000, 77])
    M = _log_int(rng, 1, 12000)
    if dtype == "f32":
        M = min(M, 1500)
    M = max(1, min(M, int(12001 * 768 * 2304 / (K * N))))
    return {"op": op, "M": M, "K": K, "N": N, "rank": rng.choice([4, 8, 16, 16, 32, 64, 12]),
            "adapters": _log_int(rng, 1, 64), "run_len": rng.choice([1, 1, 7, 64, 256, 333]),
            "dtype": dtype, "bias": rng.random() < 0.5}


def _lengths(case):
    """The case's lengths: spread evenly over the logarithm, the same for every seed."""
    B, lo, hi = case["B"], case["len_min"], case["len_max"]
    if B == 1:
        return [hi]
    base = max(lo, 1)
    out = [int(round(base * (max(hi, 1) / base) ** (i / (B - 1)))) for i in range(B)]
    out[0], out[-1] = lo, hi
    return out


def _adapter_ids(case):
    """Adapter of each row: runs of run_len rows, round robin, every ninth run without one."""
    runs = -(-case["M"] // case["run_len"])
    ids = [(-1 if i % 9 == 4 else i % case["adapters"]) for i in range(runs)]
    return [i for i in ids for _ in range(case["run_len"])][:case["M"]]


# ── inputs ───────────────────────────────────────────────────────────────────


def _paged(g, lengths, page, width, dtype):
    """A pool of rows, every session's pages scattered over it, spare pages and all."""
    B = len(lengths)
    need = [-(-n // page) for n in lengths]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros(B, max(max(need), 1), dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    pool = torch.empty(pages, page, width, dtype=dtype, device="cuda")
    pool.normal_(generator=g)
    return pool, table


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    state = {"case": case}
    if case["op"] == "lora":
        M, K, N, r, n = (case[k] for k in ("M", "K", "N", "rank", "adapters"))
        state["x"] = torch.randn(M, K, generator=g, device="cuda").to(dt)
        state["w"] = (torch.randn(N, K, generator=g, device="cuda") * K ** -0.5).to(dt)
        state["a"] = (torch.randn(n, r, K, generator=g, device="cuda") * K ** -0.5).to(dt)
        state["b"] = (torch.randn(n, N, r, generator=g, device="cuda") * 0.3 * r ** -0.5).to(dt)
        state["scaling"] = torch.rand(n, generator=g, device="cuda") + 0.5
        state["bias"] = (torch.randn(N, generator=g, device="cuda").to(dt) if case["bias"]
                         else None)
        state["ids"] = torch.tensor(_adapter_ids(case), dtype=torch.int32, device="cuda")
        return state
    lengths = _lengths(case)
    np.random.RandomState(seed % (1 << 31)).shuffle(lengths)
    B = len(lengths)
    state["lengths"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    if case["op"] == "paged_attention":
        H, Hkv, Dh = case["heads"], case["kv_heads"], case["dh"]
        state["pool"], state["table"] = _paged(g, lengths, case["page"], 2 * Hkv * Dh, dt)
        state["q"] = (1.5 * torch.randn(B, H, Dh, generator=g, device="cuda")).to(dt)
        slots = state["table"].shape[1] * case["page"]
        state["weights"] = (torch.rand(B, slots, generator=g, device="cuda") if case["weights"]
                            else None)
        return state
    # accumulated weights as attention leaves them: a few rows carry most of it
    state["pool"], state["table"] = _paged(g, lengths, case["page"], case["row"], dt)
    slots = state["table"].shape[1] * case["page"]
    state["weights"] = torch.exp(2.0 * torch.randn(B, slots, generator=g, device="cuda") - 4.0)
    # slots of a session that has been through evictions: positions out of order
    gaps = torch.rand(B, slots, generator=g, device="cuda")
    live = torch.arange(slots, device="cuda") < state["lengths"][:, None]
    state["positions"] = torch.where(live, gaps, 2.0).argsort(1).argsort(1).to(torch.int32)
    return state


# ── the calls ────────────────────────────────────────────────────────────────


def _plain_attention(s):
    c = s["case"]
    B, H, Hkv, Dh = c["B"], c["heads"], c["kv_heads"], c["dh"]
    slots = s["table"].shape[1] * c["page"]
    rows = s["pool"][s["table"].long()].reshape(B, slots, 2, Hkv, Dh).float()
    k, v = rows[:, :, 0].transpose(1, 2), rows[:, :, 1].transpose(1, 2)  # (B, Hkv, slots, Dh)
    q = s["q"].float().reshape(B, Hkv, H // Hkv, Dh)
    dead = (torch.arange(slots, device=q.device) >= s["lengths"][:, None])[:, None, None, :]
    score = (q @ k.transpose(2, 3) * Dh ** -0.5).masked_fill(dead, -math.inf)
    top = score.amax(3, keepdim=True)
    e = torch.exp(score - torch.where(top > -math.inf, top, 0.0))
    total = e.sum(3, keepdim=True)
    p = e / torch.where(total > 0, total, 1.0)
    out = (p @ v).reshape(B, H, Dh).to(s["q"].dtype)
    if s["weights"] is None:
        return out
    return out, s["weights"] + p.sum((1, 2))


def _plain_evict(s):
    c = s["case"]
    budget, recent, page = c["budget"], c["recent"], c["page"]
    n, w, pos = s["lengths"].long(), s["weights"], s["positions"]
    B, slots = w.shape
    slot = torch.arange(slots, device=w.device).expand(B, slots)
    live = slot < n[:, None]
    newest = torch.where(live, pos, -1).amax(1, keepdim=True)
    key = torch.where(live, torch.where(pos > newest - recent, math.inf, w), -1.0)
    order = torch.sort(key, dim=1, descending=True, stable=True).indices
    kept = torch.zeros_like(live).scatter_(1, order[:, :budget], True) & live
    cut = n[:, None] > budget
    hole = cut & live & ~kept & (slot < budget)
    mover = cut & kept & (slot >= budget)
    hb, hs = hole.nonzero(as_tuple=True)
    mb, ms = mover.nonzero(as_tuple=True)
    table = s["table"].long()
    s["pool"][table[hb, hs // page], hs % page] = s["pool"][table[mb, ms // page], ms % page]
    new_n = torch.clamp(n, max=budget)
    new_w = torch.zeros(B, budget, device=w.device)
    new_p = torch.full((B, budget), -1, dtype=torch.int32, device=w.device)
    m = min(slots, budget)
    keep_to = slot[:, :m] < new_n[:, None]
    new_w[:, :m] = torch.where(keep_to, w[:, :m], 0.0)
    new_p[:, :m] = torch.where(keep_to, pos[:, :m], -1)
    new_w[hb, hs] = w[mb, ms]
    new_p[hb, hs] = pos[mb, ms]
    return s["pool"], new_n.to(torch.int32), new_w, new_p


def _plain_lora(s):
    c = s["case"]
    n, r, K, N = c["adapters"], c["rank"], c["K"], c["N"]
    x = s["x"].float()
    h = (x @ s["a"].float().reshape(n * r, K).t()).reshape(-1, n, r)
    own_rows = s["ids"][:, None] == torch.arange(n, device=x.device)
    h = torch.where(own_rows[:, :, None], h * s["scaling"][:, None], 0.0)
    y = x @ s["w"].float().t()
    y = y + h.reshape(-1, n * r) @ s["b"].float().transpose(1, 2).reshape(n * r, N)
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return y.to(s["x"].dtype)


def run(state):
    c = state["case"]
    if not own:
        return {"paged_attention": _plain_attention, "evict": _plain_evict,
                "lora": _plain_lora}[c["op"]](state)
    paged_attention, evict_by_weight, lora_linear = _cortex()
    if c["op"] == "paged_attention":
        return paged_attention(state["q"], state["pool"], state["table"], state["lengths"],
                               weights=state["weights"])
    if c["op"] == "evict":
        lengths, weights, positions = evict_by_weight(
            state["pool"], state["table"], state["lengths"], state["weights"],
            state["positions"], budget=c["budget"], recent=c["recent"])
        return state["pool"], lengths, weights, positions
    return lora_linear(state["x"], state["w"], state["a"], state["b"], state["ids"],
                       scaling=state["scaling"], bias=state["bias"])


# ── what a call cannot do without ────────────────────────────────────────────


def work(case):
    el = BYTES[case["dtype"]]
    if case["op"] == "lora":
        M, K, N, r = case["M"], case["K"], case["N"], case["rank"]
        ids = _adapter_ids(case)
        used, rows = len(set(ids) - {-1}), sum(i >= 0 for i in ids)
        return {"bytes": el * (M * K + N * K + M * N + used * r * (K + N)
                               + (N if case["bias"] else 0)) + 4 * M + 4 * used,
                "flops": 2 * M * N * K + 2 * rows * r * (K + N)}
    lengths = _lengths(case)
    total = sum(lengths)
    if case["op"] == "paged_attention":
        H, Hkv, Dh = case["heads"], case["kv_heads"], case["dh"]
        slots = max(-(-max(lengths) // case["page"]), 1) * case["page"]
        by = el * (total * 2 * Hkv * Dh + 2 * case["B"] * H * Dh)
        by += 4 * (case["B"] + sum(-(-n // case["page"]) for n in lengths))
        by += 8 * case["B"] * slots if case["weights"] else 0
        return {"bytes": by, "flops": 4 * total * H * Dh}
    # eviction: read every live weight and position, move the kept rows that lie behind the
    # budget (their expected number), write the new tables
    budget = case["budget"]
    moves = sum((n - budget) / n * budget for n in lengths if n > budget)
    return {"bytes": int(8 * total + 8 * case["B"] * budget + 2 * moves * case["row"] * el
                         + 8 * case["B"]),
            "flops": 2 * total}


# ── the definitions in 64 bits ───────────────────────────────────────────────


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "lora":
        # row by row group: y = W x + scaling_i B_i (A_i x) + bias
        x, ids = s["x"].double(), _adapter_ids(case)
        y = torch.einsum("mk,nk->mn", x, s["w"].double())
        if s["bias"] is not None:
            y += s["bias"].double()
        groups = {}
        for m, i in enumerate(ids):
            groups.setdefault(i, []).append(m)
        for i, rows in groups.items():
            if i < 0:
                continue
            at = torch.tensor(rows, device="cuda")
            h = torch.einsum("mk,rk->mr", x[at], s["a"][i].double())
            y[at] += float(s["scaling"][i]) * torch.einsum("mr,nr->mn", h, s["b"][i].double())
        return y
    lengths = s["lengths"].tolist()
    page = case["page"]
    if case["op"] == "paged_attention":
        H, Hkv, Dh = case["heads"], case["kv_heads"], case["dh"]
        out = torch.zeros(case["B"], H, Dh, dtype=torch.float64, device="cuda")
        acc = None if s["weights"] is None else s["weights"].double()
        for b, n in enumerate(lengths):
            if n == 0:
                continue
            rows = torch.cat([s["pool"][p] for p in s["table"][b, :-(-n // page)].tolist()])[:n]
            rows = rows.reshape(n, 2, Hkv, Dh)
            for h in range(H):
                kv = h // (H // Hkv)
                t = rows[:, 0, kv].double() @ s["q"][b, h].double() / math.sqrt(Dh)
                p = torch.softmax(t, 0)
                out[b, h] = p @ rows[:, 1, kv].double()
                if acc is not None:
                    acc[b, :n] += p
        return out if acc is None else (out, acc)
    # eviction on the host, one session at a time
    budget, recent = case["budget"], case["recent"]
    w_all, p_all = s["weights"].cpu().numpy(), s["positions"].cpu().numpy()
    table = s["table"].cpu().numpy()
    new_w = np.zeros((case["B"], budget), np.float32)
    new_p = np.full((case["B"], budget), -1, np.int32)
    src, dst = [], []
    for b, n in enumerate(lengths):
        w, p = w_all[b, :n].copy(), p_all[b, :n].copy()
        if n > budget:
            safe = p > p.max() - recent
            rank = np.lexsort((np.arange(n), -w.astype(np.float64), ~safe))
            kept = np.zeros(n, bool)
            kept[rank[:budget]] = True
            for h, m in zip(np.flatnonzero(~kept[:budget]), budget + np.flatnonzero(kept[budget:])):
                src.append((table[b, m // page], m % page))
                dst.append((table[b, h // page], h % page))
                w[h], p[h] = w[m], p[m]
        new_w[b, :min(n, budget)] = w[:budget]
        new_p[b, :min(n, budget)] = p[:budget]
    pool = s["pool"]
    if src:
        src, dst = torch.tensor(np.array(src)).cuda(), torch.tensor(np.array(dst)).cuda()
        pool[dst[:, 0].long(), dst[:, 1].long()] = pool[src[:, 0].long(), src[:, 1].long()]
    return (pool, torch.tensor([min(n, budget) for n in lengths], dtype=torch.int32, device="cuda"),
            torch.from_numpy(new_w).cuda(), torch.from_numpy(new_p).cuda())
