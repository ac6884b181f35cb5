"""lora_linear on the GPU against its definition in 64 bits.

Tolerance, with u = 2^-24: every sum is fp32 over K, rank or both in some
order, so its error is at most (K + rank + 4) u times the sum of the terms'
magnitudes P = |W||x| + |s||B||A||x| + |bias|; the result is rounded once (2^-8
|y| for bf16, u |y| for fp32). bf16 calls whose rows go through the tensor-core
tiles round h = s A x to bf16 for the second product: 2^-8 |B||h|, and s A x
itself is within (K + 1) u |s||A||x| (inside the first term).
"""

from __future__ import annotations

import pytest
import torch

from cortex import _lib as L
from cortex.kernels.lora import lora_linear

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24


def make(M, K, N, rank, n, dtype, seed=0, pattern="random"):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(M, K, generator=g)
    w = torch.randn(N, K, generator=g) * K ** -0.5
    a = torch.randn(n, rank, K, generator=g) * K ** -0.5
    b = torch.randn(n, N, rank, generator=g) * rank ** -0.5
    ids = {"random": lambda: torch.randint(-1, n, (M,), generator=g),
           "runs": lambda: torch.arange(M) // 37 % (n + 1) - 1,
           "one": lambda: torch.full((M,), n - 1),
           "none": lambda: torch.full((M,), -3)}[pattern]()
    scaling = torch.randn(n, generator=g)
    bias = torch.randn(N, generator=g)
    return ([t.to(dtype).to(DEV) for t in (x, w, a, b)] + [ids.int().to(DEV), scaling.to(DEV),
                                                           bias.to(dtype).to(DEV)])


def want(x, w, a, b, ids, scaling, bias):
    x, w, a, b = (t.double().cpu() for t in (x, w, a, b))
    ids = ids.cpu().long()
    M, K = x.shape
    s = torch.ones(len(a)).double() if scaling is None else scaling.double().cpu()
    y = x @ w.t()
    P = x.abs() @ w.abs().t()
    H = torch.zeros_like(y)
    for i in range(len(a)):
        r = (ids == i).nonzero().flatten()
        if len(r):
            h = s[i] * (x[r] @ a[i].t())
            y[r] += h @ b[i].t()
            P[r] += s[i].abs() * (x[r].abs() @ a[i].abs().t()) @ b[i].abs().t()
            H[r] = h.abs() @ b[i].abs().t()
    if bias is not None:
        y += bias.double().cpu()
        P += bias.double().cpu().abs()
    tol = (K + a.shape[1] + 4) * U * P
    return y, tol, H


def check(got, state, scaling=True, bias=True):
    x, w, a, b, ids, s, bi = state
    y, tol, H = want(x, w, a, b, ids, s if scaling else None, bi if bias else None)
    half = 2.0 ** -8 if x.dtype == torch.bfloat16 else U
    tol = tol + half * y.abs() + (2.0 ** -8 * H if x.dtype == torch.bfloat16 else 0)
    err = (got.double().cpu() - y).abs()
    assert bool((err <= tol).all()), float((err / tol.clamp(min=1e-30)).max())


BF, F = torch.bfloat16, torch.float32
CASES = [
    # M, K, N, rank, adapters, dtype, pattern
    (1, 512, 1536, 16, 4, BF, "one"),
    (1, 64, 8, 1, 1, BF, "one"),
    (2, 256, 100, 8, 3, BF, "random"),
    (1, 4096, 1000, 8, 3, BF, "one"),
    (3, 72, 40, 5, 4, BF, "random"),
    (5, 520, 264, 3, 2, BF, "random"),
    (16, 64, 2304, 16, 7, BF, "random"),
    (16, 128, 77, 16, 7, BF, "runs"),
    (1, 192, 256, 256, 2, BF, "one"),
    (1, 200, 20000, 4, 2, BF, "one"),
    (2, 8, 9, 1, 1, BF, "one"),
    (7, 512, 512, 16, 5, BF, "random"),
    (8, 4096, 256, 16, 8, BF, "random"),
    (17, 520, 264, 24, 9, BF, "random"),
    (48, 768, 2304, 64, 64, BF, "random"),
    (63, 1000, 77, 12, 5, BF, "random"),
    (64, 256, 768, 4, 2, BF, "runs"),
    (65, 256, 768, 32, 70, BF, "random"),
    (128, 512, 256, 16, 3, BF, "none"),
    (129, 512, 1536, 16, 8, BF, "runs"),
    (300, 256, 768, 16, 200, BF, "random"),
    (777, 768, 1000, 48, 24, BF, "runs"),
    (1025, 512, 2048, 128, 7, BF, "runs"),
    (513, 264, 520, 200, 3, BF, "random"),
    (2000, 512, 1536, 16, 8, BF, "one"),
    (400, 72, 77, 5, 6, BF, "runs"),
    (300, 256, 1600, 16, 200, BF, "random"),
    (300, 256, 1600, 32, 50, BF, "random"),
    (300, 128, 1600, 64, 50, BF, "random"),
    (300, 256, 1600, 100, 9, BF, "random"),
    (33, 512, 1000, 33, 40, BF, "random"),
    (200, 520, 77, 12, 5, BF, "random"),
    (512, 64, 512, 16, 3, BF, "runs"),
    (33, 70, 97, 3, 4, BF, "random"),
    (200, 70, 97, 16, 4, BF, "runs"),
    (1, 256, 768, 8, 5, F, "one"),
    (301, 256, 768, 8, 5, F, "runs"),
    (100, 1024, 264, 40, 9, F, "random"),
    (45, 520, 77, 3, 1, F, "one"),
    (64, 2050, 129, 7, 30, F, "random"),
    (130, 70, 97, 3, 4, F, "random"),
    (1500, 512, 264, 64, 9, F, "random"),
    (40, 1024, 64, 256, 2, F, "random"),
]


@pytest.mark.parametrize("M,K,N,rank,n,dtype,pattern", CASES)
def test_against_definition(M, K, N, rank, n, dtype, pattern):
    state = make(M, K, N, rank, n, dtype, pattern=pattern)
    x, w, a, b, ids, s, bias = state
    check(lora_linear(x, w, a, b, ids, scaling=s, bias=bias), state)
    check(lora_linear(x, w, a, b, ids), state, scaling=False, bias=False)
    assert L.device_status()[0] == 0


@pytest.mark.parametrize("M", [1, 8, 20, 100, 700])
def test_same_inputs_same_bits(M):
    x, w, a, b, ids, s, bias = make(M, 512, 768, 16, 6, BF)
    y = lora_linear(x, w, a, b, ids, scaling=s, bias=bias)
    for _ in range(5):
        assert torch.equal(y, lora_linear(x, w, a, b, ids, scaling=s, bias=bias))


@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("M", [3, 40, 200, 600])
def test_strides_and_leading_shape(M, dtype):
    state = make(M, 512, 256, 16, 5, dtype)
    x, w, a, b, ids, s, bias = state
    wide = torch.full((M, 520), float("nan"), dtype=dtype, device=DEV)
    wide[:, :512] = x
    ww = torch.full((256, 528), float("nan"), dtype=dtype, device=DEV)
    ww[:, 8:520] = w
    out = torch.full((M, 300), 7.0, dtype=dtype, device=DEV)
    got = lora_linear(wide[:, :512], ww[:, 8:520], a, b, ids, scaling=s, bias=bias,
                      out=out[:, 8:264])
    check(got, state)
    assert bool((out[:, :8] == 7).all()) and bool((out[:, 264:] == 7).all())
    odd = torch.full((M, 513), float("nan"), dtype=dtype, device=DEV)
    odd[:, 1:] = x
    oo = torch.full((M, 257), 7.0, dtype=dtype, device=DEV)
    check(lora_linear(odd[:, 1:], w, a, b, ids, scaling=s, bias=bias, out=oo[:, 1:]), state)
    assert bool((oo[:, 0] == 7).all())
    if M % 4 == 0:
        y = lora_linear(x.view(4, M // 4, 512), w, a, b, ids.view(4, -1), scaling=s, bias=bias)
        assert y.shape == (4, M // 4, 256)
        check(y.reshape(M, 256), state)
    # adapters that are slices of a larger store, transposed weight
    store = torch.full((5, 20, 512), float("nan"), dtype=dtype, device=DEV)
    store[:, :16] = a
    check(lora_linear(x, w.t().contiguous().t(), store[:, :16], b, ids, scaling=s, bias=bias), state)


@pytest.mark.parametrize("M", [2, 5, 64, 300, 2000])
def test_rows_do_not_mix(M):
    """NaN and infinities in one row, or in an adapter that no row names, stay there."""
    x, w, a, b, ids, s, bias = state = make(M, 512, 256, 16, 5, BF)
    ids[ids == 2] = -1
    y = lora_linear(x, w, a, b, ids, scaling=s, bias=bias)
    a2, b2, s2 = a.clone(), b.clone(), s.clone()
    a2[2], b2[2], s2[2] = float("nan"), float("inf"), float("nan")
    assert torch.equal(y, lora_linear(x, w, a2, b2, ids, scaling=s2, bias=bias))
    x2 = x.clone()
    x2[M // 2, 3] = float("inf")
    y2 = lora_linear(x2, w, a, b, ids, scaling=s, bias=bias)
    rest = torch.arange(M, device=DEV) != M // 2
    assert torch.equal(y[rest], y2[rest])
    assert not bool(torch.isfinite(y2[M // 2]).any())
    # an adapter with NaN reaches its own rows only
    a3 = a.clone()
    a3[1, 0, 0] = float("nan")
    y3 = lora_linear(x, w, a3, b, ids, scaling=s, bias=bias)
    mine = ids == 1
    assert torch.equal(y[~mine], y3[~mine]) and bool(torch.isnan(y3[mine]).all())


@pytest.mark.parametrize("M", [5, 300])
def test_bad_ids_are_recorded(M):
    x, w, a, b, ids, s, bias = make(M, 512, 256, 16, 5, BF)
    ids[::2] = 0
    bad = ids.clone()
    bad[1] = 5
    bad[3] = 2 ** 31 - 1
    none = ids.clone()
    none[1] = none[3] = -1
    got = lora_linear(x, w, a, b, bad, scaling=s, bias=bias)
    with pytest.raises(IndexError):
        L.check_device_status("lora_linear")
    assert torch.equal(got, lora_linear(x, w, a, b, none, scaling=s, bias=bias))
    none[:] = -2 ** 31
    y = lora_linear(x, w, a[:0], b[:0], none, bias=bias)
    assert torch.equal(y, lora_linear(x, w, a, b, none, scaling=s, bias=bias))
    assert L.device_status()[0] == 0


@pytest.mark.parametrize("M", [1, 4, 300, 1100])
def test_capture_replay_and_streams(M):
    x, w, a, b, ids, s, bias = state = make(M, 512, 768, 16, 6, BF)
    lora_linear(x, w, a, b, ids, scaling=s, bias=bias)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(st):
        with torch.cuda.graph(graph, stream=st):
            y = lora_linear(x, w, a, b, ids, scaling=s, bias=bias)
    for i in range(2):
        x.normal_()
        ids.copy_(torch.randint(-1, 6, (M,)))
        graph.replay()
        torch.cuda.synchronize()
        check(y, state)
    other = make(M, 512, 768, 16, 6, BF, seed=9)
    ox, ow, oa, ob, oids, os_, obias = other
    s2 = torch.cuda.Stream()
    s2.wait_stream(torch.cuda.current_stream())
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        one = [lora_linear(x, w, a, b, ids, scaling=s, bias=bias) for _ in range(20)]
    with torch.cuda.stream(s2):
        two = [lora_linear(ox, ow, oa, ob, oids, scaling=os_, bias=obias) for _ in range(20)]
    torch.cuda.synchronize()
    for p, q in zip(one, two):
        check(p, state)
        check(q, other)
    assert L.device_status()[0] == 0


def test_empty():
    x, w, a, b, ids, s, bias = make(4, 64, 32, 8, 3, BF)
    assert lora_linear(x[:0], w, a, b, ids[:0], scaling=s).shape == (0, 32)
    assert lora_linear(x, w[:0], a, b[:, :0], ids).shape == (4, 0)


def test_refusals():
    x, w, a, b, ids, s, bias = make(4, 64, 32, 8, 3, BF)
    with pytest.raises(ValueError):
        lora_linear(x, w[:, :60], a, b, ids)
    with pytest.raises(ValueError):
        lora_linear(x, w, a[:, :, :60], b, ids)
    with pytest.raises(ValueError):
        lora_linear(x, w, a, b[:2], ids)
    with pytest.raises(ValueError):
        lora_linear(x, w, a, b[:, :, :4], ids)
    with pytest.raises(ValueError):
        lora_linear(x, w, a, b, ids[:3])
    with pytest.raises(TypeError):
        lora_linear(x, w, a, b, ids.long())
    with pytest.raises(TypeError):
        lora_linear(x.float(), w, a, b, ids)
    with pytest.raises(ValueError):
        lora_linear(x, w, a, b, ids, scaling=s.double())
    with pytest.raises(ValueError):
        lora_linear(x, w, a, b, ids, bias=bias[:3])
    with pytest.raises(ValueError):
        lora_linear(x, w, a, b, ids, out=torch.empty(4, 31, dtype=BF, device=DEV))
    with pytest.raises(RuntimeError):
        lora_linear(x.cpu(), w, a, b, ids)
    with pytest.raises(NotImplementedError):
        lora_linear(x.half(), w.half(), a.half(), b.half(), ids)
    with pytest.raises(NotImplementedError):
        lora_linear(x, w, torch.zeros(3, 300, 64, dtype=BF, device=DEV),
                    torch.zeros(3, 32, 300, dtype=BF, device=DEV), ids)


@pytest.mark.parametrize("M", [1, 6, 200])
def test_expanded_and_single_rows(M):
    """Rows that share memory, and size-one dimensions whose strides are arbitrary."""
    x, w, a, b, ids, s, bias = make(M, 512, 264, 16, 5, BF)
    row = x[:1].expand(M, 512)
    check(lora_linear(row, w, a, b, ids, scaling=s, bias=bias), (row, w, a, b, ids, s, bias))
    odd = torch.as_strided(x, (1, 512), (3, 1))
    state = (odd, w, a, b, ids[:1], s, bias)
    check(lora_linear(odd, w, a, b, ids[:1], scaling=s, bias=bias), state)
    w1 = torch.as_strided(w, (1, 512), (5, 1))
    b1 = b[:, :1].contiguous()
    check(lora_linear(x, w1, a, b1, ids, scaling=s, bias=bias[:1]), (x, w1, a, b1, ids, s, bias[:1]))
    if M > 1:
        with pytest.raises(ValueError):
            lora_linear(x, w, a, b, ids, out=torch.empty(264, dtype=BF, device=DEV).expand(M, 264))


@pytest.mark.parametrize("M", [3, 200])
def test_outputs_apart_from_inputs(M):
    x, w, a, b, ids, s, bias = make(M, 256, 256, 16, 5, BF)
    wide = torch.empty(M, 512, dtype=BF, device=DEV)
    for out in (x, w[:M], torch.empty(1, 256, dtype=BF, device=DEV).expand(M, 256)):
        with pytest.raises(ValueError):
            lora_linear(x, w, a, b, ids, out=out)
    wide[:, :256] = x
    with pytest.raises(ValueError):  # columns beside x: inside the memory that x spans
        lora_linear(wide[:, :256], w, a, b, ids, out=wide[:, 256:])


@pytest.mark.parametrize("dtype", [BF, F])
def test_rows_past_four_gigabytes(dtype):
    """x, then y, with more than 2^31 elements; the rows at both ends are checked."""
    K, N = 2048, 16
    M = 2 ** 31 // K + 700
    small = make(900, K, N, 8, 5, dtype, pattern="runs")
    x, w, a, b, ids, s, bias = small
    big = torch.zeros(M, K, dtype=dtype, device=DEV)
    big[:450], big[-450:] = x[:450], x[450:]
    far = torch.full((M,), -1, dtype=torch.int32, device=DEV)
    far[:450], far[-450:] = ids[:450], ids[450:]
    y = lora_linear(big, w, a, b, far, scaling=s, bias=bias)
    check(torch.cat([y[:450], y[-450:]]), small)
    del big, y
    K, N = 16, 2048
    small = make(900, K, N, 8, 5, dtype, pattern="runs")
    x, w, a, b, ids, s, bias = small
    big = torch.zeros(M, K, dtype=dtype, device=DEV)
    big[:450], big[-450:] = x[:450], x[450:]
    y = lora_linear(big, w, a, b, far, scaling=s, bias=bias)
    check(torch.cat([y[:450], y[-450:]]), small)


@pytest.mark.parametrize("M,rank", [(1, 16), (2, 16), (16, 2), (32, 1)])
def test_bad_ids_of_few_rows(M, rank):
    x, w, a, b, ids, s, bias = make(M, 512, 300, rank, 5, BF)
    bad, none = ids.clone(), ids.clone()
    bad[-1], none[-1] = 5, -1
    got = lora_linear(x, w, a, b, bad, scaling=s, bias=bias)
    with pytest.raises(IndexError):
        L.check_device_status("lora_linear")
    assert torch.equal(got, lora_linear(x, w, a, b, none, scaling=s, bias=bias))
    none[:] = -1
    y = lora_linear(x, w, a[:0], b[:0], none, bias=bias)
    assert torch.equal(y, lora_linear(x, w, a, b, none, scaling=s, bias=bias))
    assert L.device_status()[0] == 0


@pytest.mark.parametrize("M", [5, 40, 700])
def test_adapters_past_the_types_range(M):
    """h near the end of fp32's range, beyond bf16's largest number, and infinite. The
    result's rounding takes 2^-8, the sums far less than that again."""
    x, w, a, b, ids, s, bias = make(M, 512, 256, 16, 5, BF)
    ids[:] = torch.arange(M, device=DEV) % 3
    x[:, 1:], w[:], a[:, :, 0] = 0, 0, 1.0
    x[:, 0] = 3.3895e38  # bf16's largest
    b[:] = 2.0 ** -10
    s[:3] = torch.tensor([1.0, 1.003, 4.0])  # in range; beyond bf16's, in fp32's; infinite
    y = lora_linear(x, w, a, b, ids, scaling=s).float().cpu()
    big = float(x[0, 0]) * 16 * 2.0 ** -10
    assert bool(((y[0::3] / big - 1).abs() <= 1.001 * 2.0 ** -8).all())
    assert bool(((y[1::3] / (1.003 * big) - 1).abs() <= 1.001 * 2.0 ** -8).all())
    assert bool(torch.isposinf(y[2::3]).all())


@pytest.mark.parametrize("M,K,N,rank,n,pattern,tiles", [
    (1, 512, 256, 16, 3, "one", False),  # one launch
    (2, 256, 100, 8, 3, "random", False),
    (20, 512, 256, 24, 5, "random", False),  # rows, h in a launch before
    (48, 768, 2304, 16, 64, "random", False),
    (129, 512, 256, 16, 5, "random", False),
    (300, 256, 1600, 8, 200, "random", True),  # tiles, rank within 16, 32, 64, beyond
    (2000, 512, 1536, 16, 8, "runs", True),
    (300, 256, 768, 32, 50, "random", True),
    (700, 256, 1600, 20, 3, "runs", True),
    (777, 768, 1000, 48, 24, "runs", True),
    (300, 128, 1600, 64, 50, "random", True),
    (1025, 512, 2048, 128, 7, "runs", True),
    (513, 264, 520, 200, 3, "random", True),
    (400, 72, 77, 5, 6, "runs", False),
    (200, 70, 97, 16, 4, "runs", False),  # rows that TMA does not take
])
def test_adapters_are_not_rounded_on_the_way(M, K, N, rank, n, pattern, tiles):
    """The adapters alone (w = 0, so that nothing hides them): h = s A x counts in fp32, or
    in the tiles' two bf16 parts: the first cut off after 8 bits of h leaves less than
    2^-7 |h|, which the second holds up to its rounding, 2^-8 of that, with 2^-23 |h|
    added: (2^-15 + 2^-23) |B||h|. Beside that the sums over K and twice the rank in
    fp32, and the result's one rounding."""
    x, w, a, b, ids, s, _ = make(M, K, N, rank, n, BF, seed=4, pattern=pattern)
    w = torch.zeros_like(w)
    y, tol, H = want(x, w, a, b, ids, s, None)
    if tiles:
        tol = tol * (K + 2 * rank + 4) / (K + rank + 4) + (2.0 ** -15 + 2.0 ** -23) * H
    tol = tol + 2.0 ** -8 * y.abs()
    err = (lora_linear(x, w, a, b, ids, scaling=s).double().cpu() - y).abs()
    assert bool((err <= tol).all()), float((err / tol.clamp(min=1e-30)).max())


@pytest.mark.parametrize("M", [5, 40, 700])
@pytest.mark.parametrize("rank", [16, 32, 100])
def test_infinities_of_an_adapter(M, rank):
    """An infinite element of B_i makes the outputs it reaches infinite, with the sign of
    h, whether h is a bf16 number or not; a row of zeros stays 0 times the rest."""
    x, w, a, b, ids, s, bias = make(M, 256, 264, rank, 5, BF)
    ids[:] = torch.arange(M, device=DEV) % 5
    w[:], a[:], s[:] = 0, 0, 1.0
    a[:, 0, 0] = 1.0
    x[:, 0] = torch.where(torch.arange(M, device=DEV) % 2 == 0, 1.0, -0.75).to(BF)
    s[1], s[3] = 0.7, 1.0 / 3.0  # h with more bits than bf16 holds
    b[2:4, 7, 0] = float("inf")
    y = lora_linear(x, w, a, b, ids, scaling=s).cpu()
    ids = ids.cpu()
    hit = (ids == 2) | (ids == 3)
    assert torch.equal(y[hit, 7].sign(), x[:, 0].cpu()[hit].sign()) and bool(y[hit, 7].isinf().all())
    y[hit, 7] = 0
    assert bool(torch.isfinite(y).all())
    x[:] = 0
    b[2:4, 7, 0] = 1
    assert bool((lora_linear(x, w, a, b, ids.to(DEV), scaling=s) == 0).all())
