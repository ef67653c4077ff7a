"""The 8-bit linear map (lowbit.int8_linear): exact INT32 sums against an integer product, outputs against the epilogue in
64 bits, at the sizes, strides, types and offsets where a kernel can go wrong, on every kernel; and what it refuses.

Tolerances. The sums are exact. The epilogue rounds at most five times in FP32 (conversion, token scale, channel scale and
bias, residual scale, residual sum): with |terms| <= S, the sum of the magnitudes added up, the error is at most
5 * 2^-24 * S. SiLU uses the low-bit epilogue's approximate instructions: rtol 2e-6 on top. A shorter type adds half a unit
in its last place (2^-11 or 2^-8 relative, 2^-25 absolute below FP16's normal range)."""
from __future__ import annotations

import pytest
import torch

from kea_kernels import _lib, lowbit

pytestmark = pytest.mark.gpu
DEV = "cuda"
KERNELS = [0, _lib.INT8_KERNEL_REG, _lib.INT8_KERNEL_TILE64, _lib.INT8_KERNEL_TILE128, _lib.INT8_KERNEL_PAIR,
           _lib.INT8_KERNEL_SPLIT]


def _codes(rows, k, gen, low=-128, pad=0):
    """INT8 [rows, k] in rows 16-byte aligned, with junk in the columns past k."""
    ld = -(-k // 16) * 16 + 16 * pad
    store = torch.randint(low, 128, (rows, ld), generator=gen, dtype=torch.int8)
    return store.to(DEV)[:, :k]


def _problem(m, n, k, seed=0, pad=0):
    g = torch.Generator().manual_seed(seed)
    q, w = _codes(m, k, g, pad=pad), _codes(n, k, g, pad=2 * pad)
    qs = (torch.rand(m, generator=g) * 0.015 + 0.005).to(DEV)
    alpha = (torch.rand(n, generator=g) * 0.04 + 0.01).to(DEV)
    bias = torch.randn(n, generator=g).to(DEV)
    return q, qs, w, alpha, bias


def _sums(q, w):
    return (q.cpu().double() @ w.cpu().double().t()).to(torch.int64)   # integers far below 2^53: exact


def _check(y, sums, qs, alpha, bias=None, silu=False, residual=None, scale=1.0):
    v = sums.double() * qs.cpu().double()[:, None] * alpha.cpu().double()
    size = v.abs()
    if bias is not None:
        v, size = v + bias.cpu().double(), size + bias.cpu().double().abs()
    tol = 5 * 2.0 ** -24 * size
    if silu:
        tol = 1.1 * tol + 2e-6 * v.abs() + 1e-6
        v = v * torch.sigmoid(v)
    if residual is not None:
        v, tol = v * scale, tol * abs(scale)
        r = residual.cpu().double()
        tol = tol + 2 * 2.0 ** -24 * (v.abs() + r.abs())
        v = r + v
    if y.dtype != torch.float32:
        bits = 11 if y.dtype == torch.float16 else 8
        tol = tol + 2.0 ** -bits * (v.abs() + tol) + (2.0 ** -25 if y.dtype == torch.float16 else 0.0)
    off = (y.cpu().double() - v).abs()
    assert bool((off <= tol).all()), f"off by {float((off - tol).max())} more than {float(tol.max())}"


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 4096, 1024), (3, 17, 16), (5, 33, 100), (8, 64, 64), (16, 100, 65), (17, 96, 4096),
                                   (31, 1030, 640), (33, 129, 255), (64, 8, 2048), (125, 1024, 1024), (125, 257, 129),
                                   (127, 128, 128), (128, 256, 384), (129, 300, 1000), (200, 1030, 640), (257, 512, 1040),
                                   (300, 255, 513), (513, 640, 512), (1000, 264, 320)])
def test_sums_and_outputs(m, n, k, kernel):
    q, qs, w, alpha, bias = _problem(m, n, k, seed=m + n + k)
    acc = torch.full((m, n), -7, device=DEV, dtype=torch.int32)
    y = lowbit.int8_linear(q, qs, w, alpha, bias, acc=acc, kernel=kernel)
    sums = _sums(q, w)
    assert torch.equal(acc.cpu().long(), sums)
    _check(y, sums, qs, alpha, bias)
    assert _lib.read_device_error() == 0


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("bias,silu,scale", [(False, False, 0.0), (True, True, 0.0), (True, False, 0.5), (False, True, 1.0)])
@pytest.mark.parametrize("m,n,k", [(2, 70, 96), (125, 200, 640), (260, 512, 256)])
def test_types_and_epilogues(m, n, k, dtype, bias, silu, scale, kernel):
    q, qs, w, alpha, b = _problem(m, n, k, seed=7)
    b = b if bias else None
    res = torch.randn(m, n, generator=torch.Generator().manual_seed(3)).to(DEV, dtype) if scale else None
    y = lowbit.int8_linear(q, qs, w, alpha, b, dtype=dtype, silu=silu, residual=res, residual_scale=scale, kernel=kernel)
    assert y.dtype == dtype
    _check(y, _sums(q, w), qs, alpha, b, silu, res, scale)


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("m", [4, 125, 300])
def test_strides_offsets_and_in_place(m, kernel):
    """Padded rows of every operand, an output inside a larger matrix at an odd offset (no 16-byte rows), the skip
    connection in place; what lies around the output stays as it was."""
    n, k = 150, 200
    q, qs, w, alpha, bias = _problem(m, n, k, seed=11, pad=1)
    store = torch.randn(m + 2, n + 13, device=DEV)
    before = store.clone()
    out = store[1:m + 1, 5:5 + n]
    accs = torch.full((m, n + 3), -7, device=DEV, dtype=torch.int32)
    lowbit.int8_linear(q, qs, w, alpha, bias, out, residual=out, residual_scale=0.5, acc=accs[:, :n], kernel=kernel)
    sums = _sums(q, w)
    assert torch.equal(accs[:, :n].cpu().long(), sums) and bool((accs[:, n:] == -7).all())
    _check(out, sums, qs, alpha, bias, residual=before[1:m + 1, 5:5 + n], scale=0.5)
    before[1:m + 1, 5:5 + n] = out
    assert torch.equal(store, before)


@pytest.mark.parametrize("kernel", KERNELS)
def test_columns_past_k_do_not_count(kernel):
    q, qs, w, alpha, _ = _problem(40, 48, 96, seed=5)
    y = lowbit.int8_linear(q, qs, w, alpha, k=81, kernel=kernel)
    _check(y, _sums(q[:, :81], w[:, :81]), qs, alpha)


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("m", [2, 150])
def test_largest_sums_stay_in_int32(m, kernel):
    """-128 * -128 over the longest K that is allowed, and its opposite."""
    n, k = 16, 131071
    q = torch.full((m, 131072), -128, device=DEV, dtype=torch.int8)
    w = torch.full((n, 131072), -128, device=DEV, dtype=torch.int8)
    w[1::2] = 127
    acc = torch.empty(m, n, device=DEV, dtype=torch.int32)
    lowbit.int8_linear(q, torch.ones(m, device=DEV), w, torch.ones(n, device=DEV), k=k, acc=acc, kernel=kernel)
    assert bool((acc[:, 0::2] == 128 * 128 * k).all()) and bool((acc[:, 1::2] == -128 * 127 * k).all())


def test_kernels_agree_bit_for_bit():
    q, qs, w, alpha, bias = _problem(300, 512, 768, seed=2)
    res = torch.randn(300, 512, device=DEV)
    ys = [lowbit.int8_linear(q, qs, w, alpha, bias, silu=True, residual=res, residual_scale=0.5, kernel=k) for k in KERNELS]
    for y in ys[1:]:
        assert torch.equal(y.view(torch.int32), ys[0].view(torch.int32))


@pytest.mark.parametrize("m", [3, 125, 600])
def test_graph_streams_and_programmatic_launch(m):
    """Two maps in a row, the second on the first one's codes, with programmatic dependent launch, captured once and
    replayed on new inputs, on a stream of its own."""
    n, k = 256, 512
    q, qs, w, alpha, bias = _problem(m, n, k, seed=21)
    _, _, w2, alpha2, _ = _problem(m, 96, n, seed=22)
    plain = lambda q: lowbit.int8_linear(*(lambda t: (t[0][0], t[1][0]))(  # noqa: E731
        lowbit.quantize(lowbit.int8_linear(q, qs, w, alpha, bias), (0, n, 1, m), m, n, 1)), w2, alpha2)
    plain(q)
    stream = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=stream):
        y1 = lowbit.int8_linear(q, qs, w, alpha, bias, pdl=True)
        c, s, _ = lowbit.quantize(y1, (0, n, 1, m), m, n, 1, pdl=True)
        y2 = lowbit.int8_linear(c[0], s[0], w2, alpha2, pdl=True)
    for seed in (1, 2):
        q.copy_(torch.randint(-128, 128, (m, k), generator=torch.Generator().manual_seed(seed), dtype=torch.int8))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y2.view(torch.int32), plain(q).view(torch.int32))


def test_refusals():
    q, qs, w, alpha, bias = _problem(4, 32, 64)
    call = lowbit.int8_linear
    y = torch.empty(4, 32, device=DEV)
    for bad in (lambda: call(q.float(), qs, w, alpha), lambda: call(q, qs, w.short(), alpha),
                lambda: call(q[:, :48], qs, w, alpha), lambda: call(q, qs, w, alpha, k=65), lambda: call(q, qs, w, alpha, k=0),
                lambda: call(q.t(), qs, w, alpha), lambda: call(q, qs[:3], w, alpha), lambda: call(q, qs.double(), w, alpha),
                lambda: call(q, qs, w, alpha[:31]), lambda: call(q, qs, w, alpha, bias.half()),
                lambda: call(q, qs, w, alpha, dtype=torch.float64), lambda: call(q, qs, w, alpha, out=y[:3]),
                lambda: call(q, qs, w, alpha, out=y.t().contiguous().t()),
                lambda: call(q, qs, w, alpha, residual=y.half()), lambda: call(q, qs, w, alpha, residual=y[:, :31]),
                lambda: call(q, qs, w, alpha, acc=y), lambda: call(q, qs, w, alpha, kernel=99),
                lambda: call(q, qs, w.cpu(), alpha), lambda: call(q.cpu(), qs, w, alpha), lambda: call(q, qs.cpu(), w, alpha),
                lambda: call(torch.zeros(4, 65, device=DEV, dtype=torch.int8)[:, 1:], qs, w, alpha),   # rows not aligned
                lambda: call(torch.zeros(2, 131072, device=DEV, dtype=torch.int8), qs[:2],
                             torch.zeros(2, 131072, device=DEV, dtype=torch.int8), alpha[:2])):
        with pytest.raises(ValueError):
            bad()
    assert call(q[:0], qs[:0], w, alpha).shape == (0, 32)
