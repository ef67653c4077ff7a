"""The gated norm step between two blocks (lowbit.residual_norm, residual_norm_quantized) against its formula in 64 bits.

Tolerances. A row's sums run over at most 32 values per thread and 14 levels of adding up, so a mean, a mean square or the
value normed with it is off by at most about 50 * 2^-24 = 3e-6 of the row's largest value; two norms and the step between
make that 1e-5 where the second norm does not enlarge what reaches it by more than 4: it divides by the row's spread, so
where the terms of r are more than 4 times that (rows of one value, near zero by cancellation) the bound on h grows with
them (`_enlarged`). A shorter type adds half
a unit in its last place. INT8 codes may differ by one where the value lies within that of the middle between two."""
from __future__ import annotations

import pytest
import torch
from torch import nn

from kea_kernels import _lib, lowbit

pytestmark = pytest.mark.gpu
DEV = "cuda"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def _norm(kind, d, gen):
    if kind is None:
        return None
    module = nn.LayerNorm(d, eps=1e-5, bias=kind != "layer without bias") if kind.startswith("layer") else nn.RMSNorm(d, eps=1e-6)
    with torch.no_grad():
        for p in module.parameters():
            p.copy_(torch.randn(d, generator=gen) * 0.2 + (1.0 if p is module.weight else 0.0))
    return module.to(DEV)


def _exact_norm(v, module):
    if module is None:
        return v
    w = module.weight.detach().cpu().double()
    if isinstance(module, nn.LayerNorm):
        v = v - v.mean(-1, keepdim=True)
    v = v / ((v * v).mean(-1, keepdim=True) + module.eps).sqrt() * w
    return v if getattr(module, "bias", None) is None else v + module.bias.detach().cpu().double()


def _exact(x, y, post, gate, act, scale, pre):
    u = _exact_norm(y.cpu().double(), post)
    if gate is not None:
        g = gate.cpu().double()
        g = torch.sigmoid(g) if act == "sigmoid" else g
        u = u * (g[:, None] if gate.dim() == 2 and x.dim() == 3 and gate.shape != x.shape else g)
    r = x.cpu().double() + scale * u
    return r, _exact_norm(r, pre)


def _enlarged(x, r, pre):
    """How much more than 4 times pre enlarges an error of r's terms, per row."""
    x = x.cpu().double()
    size = (x.abs() + (r - x).abs()).amax(-1, keepdim=True)
    v = r - r.mean(-1, keepdim=True) if isinstance(pre, nn.LayerNorm) else r
    return (size / ((v * v).mean(-1, keepdim=True) + pre.eps).sqrt() / 4.0).clamp_min(1.0)


def _near(got, want, enlarged=1.0):
    tol = 1e-5 * want.abs().amax(-1, keepdim=True).clamp_min(1.0) * enlarged
    if got.dtype != F32:
        tol = tol + 2.0 ** (-11 if got.dtype == F16 else -8) * (want.abs() + tol) + (2.0 ** -25 if got.dtype == F16 else 0.0)
    off = (got.cpu().double() - want).abs()
    assert bool((off <= tol).all()), f"off by {float((off - tol).max())} more than allowed"


def _inputs(shape, tx, ty, seed=0, gate=None):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(*shape, generator=g) * 2).to(DEV, tx)
    y = (torch.randn(*shape, generator=g) * (0.3 + torch.rand(*shape[:-1], 1, generator=g)) + 0.2).to(DEV, ty)
    of = {None: None, "channel": shape[-1:], "clip": (shape[0], shape[-1]), "row": shape}[gate]
    return x, y, None if of is None else (0.5 + torch.randn(*of, generator=g)).to(DEV, ty), g


@pytest.mark.parametrize("tx,ty", [(F32, F32), (F32, F16), (F16, F16), (BF16, BF16), (F32, BF16), (BF16, F32)])
@pytest.mark.parametrize("post,pre,gate,act", [("layer", "layer", "channel", "none"), ("rms", "rms", "row", "sigmoid"),
                                               (None, "layer without bias", "clip", "none"), ("rms", None, None, "none"),
                                               (None, None, "clip", "sigmoid")])
@pytest.mark.parametrize("shape", [(3, 5, 64), (2, 7, 1024), (2, 3, 1001), (1, 9, 640)])
def test_step(shape, post, pre, gate, act, tx, ty):
    x, y, gt, g = _inputs(shape, tx, ty, seed=shape[-1], gate=gate)
    post, pre = _norm(post, shape[-1], g), _norm(pre, shape[-1], g)
    r, h = lowbit.residual_norm(x, y, post_norm=post, gate=gt, gate_act=act, scale=0.5, pre_norm=pre)
    want_r, want_h = _exact(x, y, post, gt, act, 0.5, pre)
    assert r.dtype == tx and h.dtype == ty
    _near(r, want_r)
    _near(h, want_h)


@pytest.mark.parametrize("d", [1, 2, 7, 8, 31, 33, 256, 257, 300, 511, 512, 1000, 1032, 2048, 4100, 8192, 16384, 16383])
@pytest.mark.parametrize("rows", [1, 3, 700])
def test_widths_and_row_counts(rows, d):
    x, y, gt, g = _inputs((1, rows, d), F32, F32, seed=rows + d, gate="row")
    post, pre = _norm("rms", d, g), _norm("rms" if d < 8 else "layer", d, g)
    r, h = lowbit.residual_norm(x, y, post_norm=post, gate=gt, pre_norm=pre)
    want_r, want_h = _exact(x, y, post, gt, "none", 1.0, pre)
    _near(r, want_r)
    _near(h, want_h)


@pytest.mark.parametrize("tx,ty,th", [(F32, F32, F32), (F32, BF16, BF16), (BF16, F16, BF16), (F16, F32, F16)])
@pytest.mark.parametrize("shape,gate", [((1, 9001, 1), "row"), ((3, 1667, 7), "channel"), ((2, 2501, 33), "clip"), ((1, 4999, 100), "row"),
                                        ((5, 600, 257), "row"), ((1, 2999, 513), "channel"), ((3, 1001, 1001), "clip"),
                                        ((1, 2400, 1023), "row"), ((1, 1501, 2047), None), ((7, 101, 4095), "clip"), ((1, 9001, 1024), "row")])
def test_many_rows(shape, gate, tx, ty, th):
    """Rows enough for every SM, of widths that no vector fits, the last group of rows short; in place and not."""
    d = shape[-1]
    x, y, gt, g = _inputs(shape, tx, ty, seed=d, gate=gate)
    post, pre = _norm("rms", d, g), _norm("layer" if d > 8 else "rms", d, g)
    want_r, want_h = _exact(x, y, post, gt, "sigmoid", 0.5, pre)
    r, h = lowbit.residual_norm(x, y, post_norm=post, gate=gt, gate_act="sigmoid", scale=0.5, pre_norm=pre, dtype=th)
    _near(r, want_r)
    more = _enlarged(x, want_r, pre)
    _near(h, want_h, more)
    q, qs = lowbit.residual_norm_quantized(x, y, post_norm=post, gate=gt, gate_act="sigmoid", scale=0.5, pre_norm=pre, out=x)[1:]
    assert torch.equal(x, r)
    steps = want_h.reshape(-1, d) / qs.cpu().double()[:, None]
    assert bool(((q.cpu().double() - steps).abs() <= 0.5 + 127 * 2e-5 * 4 * more.reshape(-1, 1)).all())
    assert _lib.read_device_error() == 0


@pytest.mark.parametrize("d", [96, 100, 1001])
def test_strides_in_place_and_types(d):
    """Rows inside wider matrices at offsets that leave no alignment, the stream in place, h of a third type, a gate that
    is a slice of a wider projection."""
    b, t = 3, 4
    g = torch.Generator().manual_seed(d)
    wide = torch.randn(b * t, d + 5, generator=g).to(DEV)
    ys = torch.randn(b * t, 2 * d + 3, generator=g).to(DEV)
    x, y, gate = wide[:, 1:d + 1], ys[:, 2:d + 2], ys[:, d + 2:2 * d + 2]
    pre = _norm("layer", d, g)
    want_r, want_h = _exact(x, y, None, gate, "sigmoid", 0.25, pre)
    left, right = wide[:, :1].clone(), wide[:, d + 1:].clone()
    r, h = lowbit.residual_norm(x, y, gate=gate, gate_act="sigmoid", scale=0.25, pre_norm=pre, out=x, dtype=F16)
    assert r.data_ptr() == x.data_ptr() and h.dtype == F16
    _near(r, want_r)
    _near(h, want_h)
    assert torch.equal(wide[:, :1], left) and torch.equal(wide[:, d + 1:], right)


@pytest.mark.parametrize("shape", [(2, 5, 64), (4, 125, 1024), (1, 3, 1001), (3, 7, 24)])
@pytest.mark.parametrize("tx,ty", [(F32, F32), (BF16, F16)])
def test_codes(shape, tx, ty):
    """The codes are h's by the quantizer's formula, the columns past the width zeros."""
    x, y, gt, g = _inputs(shape, tx, ty, seed=5, gate="channel")
    d = shape[-1]
    post, pre = _norm("layer", d, g), _norm("layer", d, g)
    r, q, qs = lowbit.residual_norm_quantized(x, y, post_norm=post, gate=gt, scale=0.5, pre_norm=pre)
    want_r, want_h = _exact(x, y, post, gt, "none", 0.5, pre)
    _near(r, want_r)
    want_h = want_h.reshape(-1, d)
    amax = want_h.abs().amax(1)
    assert bool(((qs.cpu().double() - amax / 127).abs() <= 1e-5 * amax.clamp_min(1.0) / 127 * 4).all())
    assert q.stride(0) % 16 == 0 and q.shape == want_h.shape
    whole = q.as_strided((q.shape[0], q.stride(0)), (q.stride(0), 1))
    assert bool((whole[:, d:] == 0).all())
    steps = want_h / qs.cpu().double()[:, None]
    assert bool(((q.cpu().double() - steps).abs() <= 0.5 + 127 * 2e-5 * 4).all())
    # and the same codes as h in FP32 followed by the quantizer
    _, h = lowbit.residual_norm(x, y, post_norm=post, gate=gt, scale=0.5, pre_norm=pre, dtype=F32)
    q2, qs2, _ = lowbit.quantize(h.view(-1, d), (0, d, 1, h.numel() // d), h.numel() // d, d, 1)
    assert torch.equal(qs, qs2[0]) and torch.equal(q, q2[0][:, :d])


def test_rows_of_zeros_and_special_values():
    """A constant row has no spread, a row of zeros no size: finite through eps. An infinity or a NaN stays in its own row."""
    d = 128
    x, y = torch.zeros(1, 4, d, device=DEV), torch.zeros(1, 4, d, device=DEV)
    x[0, 1], y[0, 1] = 3.0, -2.0
    x[0, 2, 5], y[0, 3, 7] = float("inf"), float("nan")
    pre, post = nn.LayerNorm(d).to(DEV), nn.RMSNorm(d, eps=1e-6).to(DEV)
    r, h = lowbit.residual_norm(x, y, post_norm=post, pre_norm=pre)
    assert bool((r[0, 0] == 0).all()) and bool((h[0, 0] == 0).all())
    assert bool((r[0, 1] - 2.0).abs().max() < 1e-5) and bool(h[0, 1].abs().max() < 1e-2)
    assert bool(h[0, 2].isnan().all()) and bool(h[0, 3].isnan().all()) and bool(r[0, 2, 5].isinf())
    _, q, qs = lowbit.residual_norm_quantized(x[:, :1], y[:, :1], pre_norm=pre)
    assert bool((q == 0).all()) and bool((qs == 1e-30).all())


def test_graph_with_programmatic_launch():
    x, y, gt, g = _inputs((2, 60, 512), F32, F32, gate="row")
    pre = _norm("layer", 512, g)
    w = torch.randint(-128, 128, (96, 512), generator=g, dtype=torch.int8).to(DEV)
    alpha = torch.rand(96, generator=g).to(DEV)
    run = lambda pdl: lowbit.int8_linear(*lowbit.residual_norm_quantized(x, y, gate=gt, pre_norm=pre, pdl=pdl)[1:], w, alpha, pdl=pdl)  # noqa: E731
    run(False)
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=stream):
        out = run(True)
    for seed in (3, 4):
        y.copy_(torch.randn(y.shape, generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, run(False))


def test_refusals():
    x, y, gt, g = _inputs((2, 3, 64), F32, F16, gate="row")
    pre = _norm("layer", 64, g)
    call = lowbit.residual_norm
    for bad in (lambda: call(x.cpu(), y), lambda: call(x, y[:, :2]), lambda: call(x.double(), y), lambda: call(x, y.long()),
                lambda: call(x, y, gate=gt.float()), lambda: call(x, y, gate=gt[..., :32]), lambda: call(x, y, gate=gt[:1]),
                lambda: call(x, y, gate=gt[0]), lambda: call(x, y, gate_act="relu"), lambda: call(x, y, pre_norm=nn.BatchNorm1d(64).to(DEV)),
                lambda: call(x, y, pre_norm=nn.LayerNorm(32).to(DEV)), lambda: call(x, y, pre_norm=nn.LayerNorm(64)),
                lambda: call(x, y, pre_norm=nn.LayerNorm(64, elementwise_affine=False).to(DEV)),
                lambda: call(x, y, pre_norm=nn.LayerNorm(64).half().to(DEV)), lambda: call(x, y, out=x.half()),
                lambda: call(x, y, dtype=torch.int8), lambda: call(x, y.cpu()), lambda: call(x[0, 0], y[0, 0]),
                lambda: call(x.transpose(0, 1), y.transpose(0, 1)),   # rows at two strides
                lambda: call(x[..., ::2], y[..., ::2]),
                lambda: call(torch.zeros(1, 1, 16385, device=DEV), torch.zeros(1, 1, 16385, device=DEV))):
        with pytest.raises(ValueError):
            bad()
    r, h = call(x[:, :0], y[:, :0], pre_norm=pre)
    assert r.shape == h.shape == (2, 0, 64)
    assert _lib.read_device_error() == 0


@pytest.mark.parametrize("ty", [F32, F16, BF16])
@pytest.mark.parametrize("clips,frames,d,pad,offset", [(5, 501, 1001, 0, 0), (3, 1001, 519, 0, 0), (2, 1500, 2047, 3, 0), (5, 601, 1003, 5, 8),
                                                       (4, 700, 997, 1, 3), (1, 2999, 1001, 0, 0), (9, 300, 517, 2, 16), (3, 900, 4089, 0, 0)])
def test_gates_of_clips_beside_rows_of_odd_width(clips, frames, d, pad, offset, ty):
    """A gate per clip inside a wider buffer that holds NaN beside it: each alignment against the rows, the buffer's end
    right after the last value, and bases that leave no alignment."""
    x, y, _, g = _inputs((clips, frames, d), F32, ty, seed=d + pad)
    values = (0.5 + torch.randn(clips, d, generator=g)).to(DEV, ty)
    flat = torch.full((offset + (clips - 1) * (d + pad) + d,), float("nan"), device=DEV, dtype=ty)
    gate = flat[offset:].as_strided((clips, d), (d + pad, 1))
    gate.copy_(values)
    post, pre = _norm("rms", d, g), _norm("rms", d, g)
    want_r, want_h = _exact(x, y, post, values, "none", 0.5, pre)
    r, h = lowbit.residual_norm(x, y, post_norm=post, gate=gate, scale=0.5, pre_norm=pre)
    _near(r, want_r)
    _near(h, want_h, _enlarged(x, want_r, pre))
    assert torch.equal(gate, values) and _lib.read_device_error() == 0
