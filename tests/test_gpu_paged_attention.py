"""paged_attention on the GPU against its definition in 64 bits.

Tolerances, with u = 2^-24 (half a step of fp32) and A_d = sum_j p_j |v_jd|:
* a score is a sum of Dh products in fp32 and three more roundings (scale, the
  log2 factor, the subtraction of the maximum), so |ds| <= (Dh + 8) u M for
  M = scale max_j sum_d |q_d k_jd| (and the subtraction's operands are at most
  2 M); p changes by at most 2 |ds| relative (numerator and sum), plus 8 u for
  the exponentials;
* sums over n positions in fp32, in any order: n u relative to A_d (and n u for l);
* a probability below fp32's smallest normal number, 2^-126, has no relative
  precision there: an absolute error of at most 2^-126 a head (the first run of
  the test with scores far apart had probabilities of 1e-46, where fp32 holds
  0 or 1.4e-45, and no tolerance for it);
* bf16: p is rounded to bf16 for the matrix instruction, 2^-8 A_d, and the
  output once, 2^-8 |o|; fp32 rounds the output by u |o|.
"""

from __future__ import annotations

import pytest
import torch

from cortex import _lib as L
from cortex.kernels.paged_attention import paged_attention

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24


def make(lens, H, Hkv, Dh, page, dtype, seed=0, slack=0, nan=True):
    """(q, pool, table, lengths): pages in random order; everything that is not
    a live row (page tails, unused pages) is NaN, unused table entries are wild."""
    g = torch.Generator().manual_seed(seed)
    B = len(lens)
    need = [-(-n // page) for n in lens]
    pages = sum(need) + 2
    perm = torch.randperm(pages, generator=g)
    width = max(max(need, default=0), 1) + slack
    table = torch.full((B, width), 2 ** 31 - 1, dtype=torch.int32)
    pool = torch.full((pages, page, 2 * Hkv * Dh), float("nan") if nan else 0.0)
    at = 0
    for b, n in enumerate(lens):
        table[b, :need[b]] = perm[at:at + need[b]].int()
        for j in range(n):
            pool[perm[at + j // page], j % page] = torch.randn(2 * Hkv * Dh, generator=g)
        at += need[b]
    q = 1.5 * torch.randn(B, H, Dh, generator=g)
    return (q.to(dtype).to(DEV), pool.to(dtype).to(DEV), table.to(DEV),
            torch.tensor(lens, dtype=torch.int32, device=DEV))


def want(q, pool, table, lengths, scale=None):
    """(o, its tolerance, summed probabilities, their tolerance) in float64."""
    q, pool, table, lens = q.double().cpu(), pool.cpu(), table.cpu(), lengths.tolist()
    B, H, Dh = q.shape
    page, Hkv = pool.shape[1], pool.shape[2] // (2 * Dh)
    half = 2.0 ** -8 if pool.dtype == torch.bfloat16 else 0.0
    half_out = 2.0 ** -8 if pool.dtype == torch.bfloat16 else U
    scale = Dh ** -0.5 if scale is None else scale
    o, tol = torch.zeros(B, H, Dh).double(), torch.zeros(B, H, Dh).double()
    cap = table.shape[1] * page
    w, wtol = torch.zeros(B, cap).double(), torch.zeros(B, cap).double()
    for b, n in enumerate(lens):
        if n == 0:
            continue
        rows = torch.stack([pool[table[b, j // page].item(), j % page] for j in range(n)]).double()
        k, v = rows.reshape(n, 2, Hkv, Dh).unbind(1)
        for h in range(H):
            kk, vv = k[:, h // (H // Hkv)], v[:, h // (H // Hkv)]
            p = torch.softmax(kk @ q[b, h] * scale, 0)
            M = abs(scale) * float((kk.abs() @ q[b, h].abs()).max())
            rel = 2 * 2 * (Dh + 8) * U * M + 8 * U + 2 * n * U
            A = p @ vv.abs()
            o[b, h] = p @ vv
            tol[b, h] = (rel + half) * A + half_out * o[b, h].abs() + 1e-30
            w[b, :n] += p
            wtol[b, :n] += p * rel + 2 * H * U * p + 2.0 ** -126
    return o, tol, w, wtol


def check(got, o, tol):
    err = (got.double().cpu() - o).abs()
    assert bool((err <= tol).all()), float((err - tol).max())


CASES = [
    # lens, H, Hkv, Dh, page, dtype
    ([1], 8, 8, 64, 64, torch.bfloat16),
    ([0, 1, 15, 16, 17, 63, 64, 65], 8, 8, 64, 64, torch.bfloat16),
    ([300], 8, 8, 64, 64, torch.bfloat16),
    ([511, 512, 513, 1500, 0], 12, 12, 64, 64, torch.bfloat16),
    ([700, 3, 129], 8, 2, 128, 48, torch.bfloat16),
    ([90, 33], 6, 3, 128, 7, torch.bfloat16),
    ([257, 31], 8, 1, 32, 16, torch.bfloat16),
    ([400, 20], 16, 1, 64, 64, torch.bfloat16),
    ([100, 65], 17, 1, 64, 24, torch.bfloat16),
    ([130, 2], 4, 2, 96, 16, torch.bfloat16),
    ([70, 9], 3, 3, 20, 5, torch.bfloat16),
    ([70, 9], 2, 1, 256, 16, torch.bfloat16),
    ([77], 2, 2, 33, 1, torch.bfloat16),
    ([1000, 3, 0, 513], 8, 8, 64, 64, torch.bfloat16),
    ([1000], 4, 2, 32, 128, torch.bfloat16),
    ([500, 9], 4, 4, 64, 16, torch.float32),
    ([0, 1, 7, 8, 9, 24, 25, 1025], 4, 4, 64, 24, torch.float32),
    ([200, 600], 8, 2, 128, 64, torch.float32),
    ([50, 3], 5, 1, 32, 16, torch.float32),
    ([50, 33], 2, 2, 96, 16, torch.float32),
    ([50, 33], 2, 1, 256, 16, torch.float32),
    ([41, 5], 3, 3, 37, 8, torch.float32),
    ([41], 4, 1, 200, 8, torch.float32),
]


@pytest.mark.parametrize("lens,H,Hkv,Dh,page,dtype", CASES)
def test_against_definition(lens, H, Hkv, Dh, page, dtype):
    q, pool, table, lengths = make(lens, H, Hkv, Dh, page, dtype)
    o, tol, w, wtol = want(q, pool, table, lengths)
    check(paged_attention(q, pool, table, lengths), o, tol)
    base = torch.rand(len(lens), table.shape[1] * page + 3, device=DEV)
    out, got = paged_attention(q, pool, table, lengths, weights=base)
    check(out, o, tol)
    cap = table.shape[1] * page
    full, ftol = base.double().cpu(), torch.zeros(base.shape).double()
    full[:, :cap] += w
    ftol[:, :cap] = wtol + U * full[:, :cap].abs()
    check(got, full, ftol)
    keep = base.clone()
    _, same = paged_attention(q, pool, table, lengths, weights=keep, weights_out=keep)
    assert same is keep and torch.equal(keep, got)
    assert L.device_status()[0] == 0


def test_same_inputs_same_bits():
    q, pool, table, lengths = make([900, 40, 0, 333], 8, 2, 64, 24, torch.bfloat16, nan=False)
    w = torch.zeros(4, table.shape[1] * 24, device=DEV)
    a = paged_attention(q, pool, table, lengths, weights=w)
    for _ in range(5):
        b = paged_attention(q, pool, table, lengths, weights=w)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_strides_and_scale():
    """A pool that is a slice of a wider one, transposed queries, strided tables."""
    Hkv, Dh = 2, 64
    q, pool, table, lengths = make([130, 64, 77], 4, Hkv, Dh, 16, torch.bfloat16)
    wide = torch.full((pool.shape[0], 20, pool.shape[2] + 32), float("nan"), device=DEV,
                      dtype=pool.dtype)
    view = wide[:, 2:18, 16:16 + pool.shape[2]]
    view.copy_(pool)
    qt = q.transpose(0, 1).contiguous().transpose(0, 1)
    table2 = torch.full((3, 2 * table.shape[1]), -7, dtype=torch.int32, device=DEV)
    table2[:, ::2] = table
    len2 = torch.stack([lengths, lengths + 10 ** 6], 1)
    o, tol, _, _ = want(q, pool, table, lengths, scale=0.3)
    out = torch.full((3, 6, 64), 5.0, dtype=q.dtype, device=DEV)
    got = paged_attention(qt, view, table2[:, ::2], len2[:, 0], scale=0.3, out=out[:, 1:5])
    check(got, o, tol)
    assert bool((out[:, 0] == 5).all()) and bool((out[:, 5] == 5).all())
    # an odd row stride leaves the 16-byte path
    odd = torch.full((pool.shape[0], 16, pool.shape[2] + 1), float("nan"), device=DEV,
                     dtype=pool.dtype)
    odd[:, :, :pool.shape[2]] = pool
    check(paged_attention(q, odd[:, :, :pool.shape[2]], table, lengths, scale=0.3), o, tol)
    assert L.device_status()[0] == 0


def test_shared_pages_and_extreme_scores():
    """Two sequences on the same pages; scores far apart, infinite values that
    are alive, and a row of -inf scores."""
    q, pool, table, lengths = make([100, 100], 4, 4, 64, 16, torch.float32, nan=False)
    table[1] = table[0]
    q = q * 40
    o, tol, w, wtol = want(q, pool, table, lengths)
    got, acc = paged_attention(q, pool, table, lengths,
                               weights=torch.zeros(2, table.shape[1] * 16, device=DEV))
    check(got, o, tol)
    check(acc, w, wtol + U * w)
    pool2 = pool.clone()
    pool2[table[0, 2], 5, 64 * 4] = float("inf")  # a live V element
    got = paged_attention(q, pool2, table, lengths)
    bad = ~torch.isfinite(got)
    assert bool(bad[:, 0, 0].all()) and int(bad.sum()) == 2
    # every score -inf: no key counts, the output is 0 (as for an empty row)
    pool3 = pool.clone()
    pool3[:, :, :64 * 4] = float("-inf")
    got = paged_attention(q.abs() + 1, pool3, table, lengths)
    assert bool((got == 0).all())
    # -inf in the first tiles only
    pool4 = pool.clone()
    pool4[table[0, :3], :, :64 * 4] = float("-inf")
    qa = q.abs() / 40 + 0.1
    live = torch.arange(48, 100)
    rows = torch.stack([pool[table[0, j // 16], j % 16] for j in live.tolist()]).double().cpu()
    k, v = rows.reshape(52, 2, 4, 64).unbind(1)
    p = torch.softmax(torch.einsum("nhd,hd->hn", k, qa[0].double().cpu()) / 8, 1)
    ref = torch.einsum("hn,nhd->hd", p, v)
    got = paged_attention(qa, pool4, table, lengths)[0].double().cpu()
    assert float((got - ref).abs().max()) < 1e-5
    assert L.device_status()[0] == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_bad_pages_and_lengths_are_recorded(dtype):
    q, pool, table, lengths = make([100, 40], 4, 4, 64, 16, dtype)
    for page in (-1, pool.shape[0], -2 ** 31):
        t = table.clone()
        t[0, 1] = page  # rows 16..31 of sequence 0 count as absent
        got = paged_attention(q, pool, t, lengths)
        with pytest.raises(IndexError):
            L.check_device_status("paged_attention")
        keep = [j for j in range(100) if not 16 <= j < 32]
        packed = pool.clone()
        rows = torch.stack([pool[table[0, j // 16], j % 16] for j in keep])
        t2 = table.clone()
        for i in range(len(keep)):
            packed[t2[0, i // 16], i % 16] = rows[i]
        o, tol, _, _ = want(q, packed, t2, torch.tensor([84, 40]))
        check(got, o, tol)
    cap = table.shape[1] * 16
    for bad in (-5, cap + 1, 2 ** 31 - 1):
        n = lengths.clone()
        n[1] = bad
        t = table.clone()
        t[1] = table[0]
        full = pool.clone()
        full[torch.isnan(full)] = 0
        got = paged_attention(q, full, t, n)
        with pytest.raises(IndexError):
            L.check_device_status("paged_attention")
        o, tol, _, _ = want(q, full, t, torch.tensor([100, 0 if bad < 0 else cap]))
        check(got, o, tol)


def test_capture_replay_and_streams():
    q, pool, table, lengths = make([600, 50, 0], 8, 4, 64, 16, torch.bfloat16, nan=False)
    w = torch.zeros(3, table.shape[1] * 16, device=DEV)
    pool[pool != pool] = 0
    paged_attention(q, pool, table, lengths, weights=w)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        with torch.cuda.graph(graph, stream=s):
            out, acc = paged_attention(q, pool, table, lengths, weights=w)
    for lens in ([600, 50, 0], [1, 600, 17]):
        lengths.copy_(torch.tensor(lens))
        q.normal_()
        table[2] = table[0]
        table[1] = table[0]
        graph.replay()
        torch.cuda.synchronize()
        o, tol, ws, wtol = want(q, pool, table, lengths)
        check(out, o, tol)
        check(acc, ws, wtol + U * ws)
    # two calls at once on two streams
    s2 = torch.cuda.Stream()
    s2.wait_stream(torch.cuda.current_stream())
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        a = [paged_attention(q, pool, table, lengths, weights=w) for _ in range(20)]
    with torch.cuda.stream(s2):
        b = [paged_attention(-q, pool, table, lengths, weights=w) for _ in range(20)]
    torch.cuda.synchronize()
    o2, tol2, _, _ = want(-q, pool, table, lengths)
    for x, y in zip(a, b):
        check(x[0], o, tol)
        check(y[0], o2, tol2)
    assert L.device_status()[0] == 0


def test_no_sequences_and_no_pages():
    q, pool, table, lengths = make([5], 4, 4, 64, 16, torch.bfloat16)
    assert paged_attention(q[:0], pool, table[:0], lengths[:0]).shape == (0, 4, 64)
    zero = torch.zeros(1, dtype=torch.int32, device=DEV)
    out, w = paged_attention(q, pool, table[:, :0], zero, weights=torch.ones(1, 4, device=DEV))
    assert bool((out == 0).all()) and bool((w == 1).all())
    out = paged_attention(q, pool[:0], table, zero)
    assert bool((out == 0).all())
    assert L.device_status()[0] == 0


def test_refusals():
    q, pool, table, lengths = make([5, 6], 4, 4, 64, 16, torch.bfloat16)
    w = torch.zeros(2, 16, device=DEV)
    with pytest.raises(TypeError):
        paged_attention(q.float(), pool, table, lengths)
    with pytest.raises(TypeError):
        paged_attention(q, pool, table.long(), lengths)
    with pytest.raises(ValueError):
        paged_attention(q[:1], pool, table, lengths)
    with pytest.raises(ValueError):
        paged_attention(q[:, :3], pool, table, lengths)
    with pytest.raises(ValueError):
        paged_attention(q[:, :, :60], pool, table, lengths)
    with pytest.raises(ValueError):
        paged_attention(q, pool[0], table, lengths)
    with pytest.raises(ValueError):
        paged_attention(q, pool, table, lengths, weights=w[:, :15])
    with pytest.raises(ValueError):
        paged_attention(q, pool, table, lengths, weights=w.double())
    with pytest.raises(ValueError):
        paged_attention(q, pool, table, lengths, weights_out=w)
    with pytest.raises(ValueError):
        paged_attention(q, pool, table, lengths, out=q[:, :2])
    with pytest.raises(RuntimeError):
        paged_attention(q.cpu(), pool, table, lengths)
    with pytest.raises(NotImplementedError):
        paged_attention(q.half(), pool.half(), table, lengths)
    with pytest.raises(NotImplementedError):
        big = torch.zeros(2, 1, 512, device=DEV)
        paged_attention(big, torch.zeros(2, 16, 1024, device=DEV), table, lengths)


def test_outputs_apart_from_inputs():
    q, pool, table, lengths = make([5, 6], 4, 4, 64, 16, torch.bfloat16)
    w = torch.zeros(2, 40, device=DEV)
    for out in (q, pool[0, 0].as_strided(q.shape, q.stride()),
                torch.empty(1, 4, 64, dtype=q.dtype, device=DEV).expand(2, 4, 64)):
        with pytest.raises(ValueError):
            paged_attention(q, pool, table, lengths, out=out)
    with pytest.raises(ValueError):  # shifted against the input
        paged_attention(q, pool, table, lengths, weights=w[:, :20], weights_out=w[:, 1:21])
    with pytest.raises(ValueError):
        paged_attention(q, pool, table, lengths, weights=w[:1].expand(2, 40),
                        weights_out=w[:1].expand(2, 40))
    got = paged_attention(q, pool, table, lengths, weights=w, weights_out=w)
    assert got[1] is w


@pytest.mark.parametrize("dtype,H", [(torch.bfloat16, 8), (torch.float32, 8), (torch.bfloat16, 3)])
def test_rows_past_four_gigabytes(dtype, H):
    """Pages whose elements lie more than 2^31 elements from the pool's start."""
    Dh, page = (64, 16) if H == 8 else (20, 16)
    q, pool, table, lengths = make([700, 33, 1], H, H, Dh, page, dtype)
    o, tol, w, wtol = want(q, pool, table, lengths)
    width, n = pool.shape[2], len(pool)
    first = 2 ** 31 // (page * width) + 5
    big = torch.empty(first + n, page, width, dtype=dtype, device=DEV)
    big[first:] = pool
    live = table < n
    got, gw = paged_attention(q, big, torch.where(live, table + first, table), lengths,
                              weights=torch.zeros(w.shape, device=DEV))
    check(got, o, tol)
    check(gw, w, wtol)


def test_a_valid_call_after_a_refused_one():
    """A scale of NaN is refused; the same shapes with a valid one are not."""
    q, pool, table, lengths = make([30, 77], 2, 2, 64, 16, torch.bfloat16, seed=8)
    w = torch.zeros(2, table.shape[1] * 16, device=DEV)
    with pytest.raises(ValueError):
        paged_attention(q, pool, table, lengths, weights=w, scale=float("nan"))
    o, tol, ws, wtol = want(q, pool, table, lengths)
    out, got = paged_attention(q, pool, table, lengths, weights=w)
    check(out, o, tol)
    check(got, ws, wtol + U * ws)
    assert L.device_status()[0] == 0


@pytest.mark.parametrize("lens,H,Hkv,Dh", [
    ([300], 8, 8, 64), ([900, 17, 0, 256], 4, 4, 64), ([700, 64], 8, 2, 128),
    ([1000, 5], 3, 3, 32), ([800, 40], 16, 1, 64), ([500], 24, 2, 128), ([400, 33], 4, 2, 96),
])
def test_probabilities_keep_sixteen_bits(lens, H, Hkv, Dh):
    """bf16, flat probabilities, values of both signs: the output is far smaller than
    A = sum p |v|, so that its own rounding hides nothing. p = p1 + p2 in bf16, p1 cut off
    after 8 bits: off by 2^-8 of p2 < 2^-7 p, and 2^-23 p added, (2^-15 + 2^-23) A. Layouts
    outside the streaming kernel keep p in fp32."""
    q, pool, table, lengths = make(lens, H, Hkv, Dh, 16, torch.bfloat16, seed=12)
    q = q * 0.125
    o, tol, _, _ = want(q, pool, table, lengths)
    A = want_magnitudes(q, pool, table, lengths)
    check(paged_attention(q, pool, table, lengths), o, tol - (2.0 ** -8 - 2.0 ** -15 - 2.0 ** -23) * A)
    w = torch.zeros(len(lens), table.shape[1] * 16, device=DEV)
    check(paged_attention(q, pool, table, lengths, weights=w)[0], o,
          tol - (2.0 ** -8 - 2.0 ** -15 - 2.0 ** -23) * A)


def want_magnitudes(q, pool, table, lengths):
    """sum_j p_j |v_j| in float64: the output of the same scores over |V|."""
    Dh = q.shape[2]
    Hkv = pool.shape[2] // (2 * Dh)
    mag = pool.clone()
    mag[:, :, Hkv * Dh:] = mag[:, :, Hkv * Dh:].abs()
    return want(q, mag, table, lengths)[0]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("Dh,H,Hkv", [(32, 3, 3), (64, 16, 1), (128, 4, 2), (96, 2, 2)])
def test_infinite_values_that_are_alive(dtype, Dh, H, Hkv):
    """An infinite element of V makes its column infinite, not NaN, at any probability."""
    q, pool, table, lengths = make([300, 40, 7], H, Hkv, Dh, 16, dtype, seed=5, nan=False)
    q = q * 0.25  # (no probability vanishes)
    for b, j, d, value in ((0, 0, 1, float("inf")), (0, 131, Dh - 1, -float("inf")),
                           (1, 39, 0, -float("inf")), (2, 3, 5, float("inf"))):
        pool[table[b, j // 16], j % 16, Hkv * Dh + d] = value  # head 0 of the K|V heads
        got = paged_attention(q, pool, table, lengths)[b, :H // Hkv]
        assert bool((got[:, d] == value).all())
    got = paged_attention(q, pool, table, lengths)
    assert int((~torch.isfinite(got)).sum()) == 4 * (H // Hkv) and not bool(torch.isnan(got).any())
