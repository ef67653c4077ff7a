"""The operators around an 8-bit model where a call can go wrong without a word: offsets past 32 bits, scores that tie, norms
that are not what their class says, buffers that overlap, rows that are not numbers, labels that are masked.

Tolerances stand at each test; where none is named the values have to be equal."""
from __future__ import annotations

import ctypes

import pytest
import torch
from torch import nn

from kea_kernels import _lib, lowbit
from kea_kernels.decoder import BeamDecoder
from kea_kernels.int8 import Int8Linear
from test_operators_cpu import ResidualNormDesc

pytestmark = pytest.mark.gpu
DEV = "cuda"


def test_codes_past_32_bit_offsets():
    """Rows whose codes lie 2^31 bytes and more from the first: the last ones are those of a call of their own. Without
    norms r is one rounded sum and a code one rounded quotient, so the two calls agree bit for bit."""
    d, rows, some = 16384, 131072 + 5, 7
    gen = torch.Generator(device=DEV).manual_seed(1)
    x, y = (torch.zeros(1, rows, d, device=DEV, dtype=torch.float16) for _ in range(2))
    x[:, -some:] = torch.randn(some, d, generator=gen, device=DEV)
    y[:, -some:] = torch.randn(some, d, generator=gen, device=DEV)
    want_r, want_q, want_qs = lowbit.residual_norm_quantized(x[:, -some:].clone(), y[:, -some:].clone())
    r, q, qs = lowbit.residual_norm_quantized(x, y, out=x)
    assert (rows - some) * q.stride(0) < 2 ** 31 < (rows - 1) * q.stride(0)
    assert torch.equal(q[-some:], want_q) and torch.equal(qs[-some:], want_qs) and torch.equal(r[:, -some:], want_r)
    assert bool((qs[:-some] == 1e-30).all()) and not bool(q[:3].any()) and not bool(q[-some - 3:-some].any())
    assert _lib.read_device_error() == 0


def _ulps(base, count, gen):
    """`count` neighbouring FP32 numbers from base up, in a random order."""
    bits = torch.tensor([base], dtype=torch.float32).view(torch.int32) + torch.randperm(count, generator=gen).int()
    return bits.view(torch.float32)


@pytest.mark.parametrize("clips", [1, 2, 40, 300])
@pytest.mark.parametrize("vocab", [40, 1025, 30000])
def test_a_hypothesis_labels_come_by_logit(vocab, clips):
    """Logits a rounding apart at scores where dozens of them have one score: a hypothesis' labels come by logit, equal
    logits by label, whatever number of clips (and with it the split of a row) and whatever the width; a narrower choice is
    the beginning of a wider one."""
    gen = torch.Generator().manual_seed(vocab)
    one = torch.randn(3, vocab, generator=gen).clamp(-3, 3)
    for k in range(3):
        at = torch.randperm(vocab, generator=gen)[:38]
        one[k, at] = _ulps(5.0, 19, gen).repeat(2)                      # every logit twice
    x = one.to(DEV).expand(clips, 3, vocab).contiguous()
    # the other hypotheses' best are 100 and more below the first one's: all 32 places are its own
    s = torch.tensor([-300.0, -400.0, -500.0], device=DEV).expand(clips, 3).contiguous()
    order = torch.sort(one[0], descending=True, stable=True)[1]
    wide = lowbit.beam_select(x, s, 32)
    assert torch.equal(wide.tokens.cpu().long(), order[:32].expand(clips, 32)) and not bool(wide.parents.any())
    assert len(wide.scores[0].unique()) < 8                             # they do tie
    for width in (1, 2, 5, 31):
        step = lowbit.beam_select(x, s, width)
        assert torch.equal(step.tokens, wide.tokens[:, :width]) and torch.equal(step.parents, wide.parents[:, :width])


@pytest.mark.parametrize("clips", [1, 40, 300])
@pytest.mark.parametrize("vocab", [64, 1024, 30000])
def test_hypotheses_that_tie_come_by_index(vocab, clips):
    """Three hypotheses with the same logits and scores: of equal scores the lower hypothesis' come first, within it the
    larger logit, then the lower label."""
    gen = torch.Generator().manual_seed(vocab + 1)
    one = torch.randn(vocab, generator=gen).clamp(-3, 3)
    at = torch.randperm(vocab, generator=gen)[:38]
    one[at] = _ulps(5.0, 38, gen)
    x = one.to(DEV).expand(clips, 3, vocab).contiguous()
    step = lowbit.beam_select(x, torch.full((clips, 3), -300.0, device=DEV), 32)
    scores, parents, tokens = step.scores.tolist(), step.parents.tolist(), step.tokens.tolist()
    order = torch.sort(one, descending=True, stable=True)[1].tolist()
    for b in range(clips):
        places = [(-scores[b][j], parents[b][j], -float(one[tokens[b][j]]), tokens[b][j]) for j in range(32)]
        assert places == sorted(places)
        for k in range(3):
            mine = [tokens[b][j] for j in range(32) if parents[b][j] == k]
            assert mine == order[:len(mine)]
        assert 0 in parents[b] and len(set(scores[b])) < 8


def test_a_score_below_the_range_is_not_offered():
    """A score that FP32 does not hold is -inf, as what is masked: the places go by label."""
    x = torch.zeros(1, 1, 6, device=DEV)
    x[0, 0, 0], x[0, 0, 3], x[0, 0, 4], x[0, 0, 5] = -float("inf"), 2.9e38, -3e38, 3e38
    step = lowbit.beam_select(x, torch.zeros(1, 1, device=DEV), 5)             # label 4: -3e38 - 3e38
    assert step.tokens[0].tolist() == [5, 3, 1, 2, 0] and step.scores[0].isfinite().tolist() == [True] * 4 + [False]
    step = lowbit.beam_select(x, torch.full((1, 1), -1e38, device=DEV), 5)     # labels 1 and 2: -3e38 - 1e38
    assert step.tokens[0].tolist() == [5, 3, 0, 1, 2] and step.scores[0].isfinite().tolist() == [True] * 2 + [False] * 3


def _selection_us(x, s, width):
    """The least of five times of one selection, launches back to back."""
    for _ in range(3):
        lowbit.beam_select(x, s, width)
    least = float("inf")
    for _ in range(5):
        a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        a.record()
        for _ in range(20):
            lowbit.beam_select(x, s, width)
        b.record()
        b.synchronize()
        least = min(least, 50.0 * a.elapsed_time(b))
    return least


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_of_one_value_take_no_longer(dtype):
    """Every logit of such a row reaches the bound of its best. Offered one by one they take several times a usual row's
    time; time between runs moves by a tenth, so 1.6 tells the two apart."""
    x = torch.randn(8, 8, 262144, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV).to(dtype)
    s = -10.0 * torch.rand(8, 8, device=DEV)
    usual = _selection_us(x, s, 8)
    x[:] = 1.5
    assert _selection_us(x, s, 8) < 1.6 * usual
    x[..., ::2] = 1.0
    assert _selection_us(x, s, 8) < 1.6 * usual



@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_finite_masks_and_log_probabilities_take_one_pass(dtype):
    """Logits far below zero, as a mask or everywhere, are summed in the pass that reads them. A second, scalar pass over the
    masked rows is several times as long as the first; time between runs moves by a tenth, so 1.6 tells the two apart."""
    vocab = 262144
    gen = torch.Generator(device=DEV).manual_seed(1)
    plain = torch.randn(8, 8, vocab, generator=gen, device=DEV)
    s = -10.0 * torch.rand(8, 8, generator=gen, device=DEV)
    usual = _selection_us(plain.to(dtype), s, 8)
    low = torch.finfo(dtype).min
    for mask in (-1e4, max(-1e9, low), low):
        x = plain.clone().to(dtype)
        x[..., :vocab // 2] = mask
        assert _selection_us(x, s, 8) < 1.6 * usual, mask
    assert _selection_us((plain - 110.0).to(dtype), s, 8) < 1.6 * usual


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("level", [0.0, -90.0, -1e4, -1e9, -2.0 ** 27, -1e12, -1e30, -3.3e38])
def test_log_sums_far_below_zero(level, dtype):
    """Rows around any level, some with the lowest value beside: the score is the rounded logit less the log-sum. The
    sum is good to 1e-6; then FP32 numbers of the level's size are subtracted: two roundings of it."""
    gen = torch.Generator().manual_seed(3)
    x = (level + 3.0 * torch.randn(4, 3, 700, generator=gen)).to(dtype)
    x[1, :, 100:600] = torch.finfo(dtype).min
    x[2, :, ::2] = -float("inf")
    x[3, 1, 5:] = torch.finfo(dtype).min
    step = lowbit.beam_select(x.to(DEV), torch.zeros(4, 3, device=DEV), 1)
    want = torch.log_softmax(x.double(), -1).flatten(1).amax(-1)
    assert bool(((step.scores.cpu()[:, 0].double() - want).abs() <= 2e-5 + 2.0 ** -22 * abs(level)).all())


@pytest.mark.parametrize("rows,d", [(3, 1001), (12024, 1001), (12024, 1000), (5, 64)])
def test_a_bias_beside_root_mean_square_norms(rows, d):
    """The C entry point takes a bias with either norm, on every route: many rows of odd width as few of them. A normed value
    is off by 3e-6 of the row's largest (sums of at most 32 values per thread and 14 levels), twice, and r's error is
    enlarged by at most 1 / 0.3 in the second norm: 3e-5 of the largest magnitude."""
    gen = torch.Generator(device=DEV).manual_seed(d)
    x, y = (torch.randn(rows, d, generator=gen, device=DEV) for _ in range(2))
    w1, b1, w2, b2 = (torch.randn(d, generator=gen, device=DEV) + (i % 2 == 0) for i in range(4))
    r, h = torch.empty_like(x), torch.empty_like(x)
    desc = ResidualNormDesc(x=x.data_ptr(), y=y.data_ptr(), ldx=d, ldy=d, frames=rows, post=2, pre=2, scale=0.5, post_eps=1e-6,
                            pre_eps=1e-6, post_weight=w1.data_ptr(), post_bias=b1.data_ptr(), pre_weight=w2.data_ptr(),
                            pre_bias=b2.data_ptr(), r=r.data_ptr(), h=h.data_ptr(), ldr=d, ldh=d, m=rows, d=d)
    _lib.check(_lib.lib().kea_lowbit_residual_norm(ctypes.byref(desc), _lib.stream_handle(x.device)), "residual_norm")
    norm = lambda v, w, b: v / ((v * v).mean(-1, keepdim=True) + 1e-6).sqrt() * w.double() + b.double()  # noqa: E731
    want_r = x.double() + 0.5 * norm(y.double(), w1, b1)
    want_h = norm(want_r, w2, b2)
    for got, want in ((r, want_r), (h, want_h)):
        assert bool(((got.double() - want).abs() <= 3e-5 * want.abs().amax(-1, keepdim=True).clamp_min(1.0)).all())


@pytest.mark.parametrize("rows,d", [(9, 64), (9, 65), (12024, 1001), (4000, 1024)])
@pytest.mark.parametrize("norm", [None, nn.LayerNorm, nn.RMSNorm])
def test_a_row_that_is_not_a_number_has_no_scale(rows, d, norm):
    """INT8 codes hold no NaN, so the row's scale does: the 8-bit map after it returns NaN for that row, as it would in FP32,
    and leaves the others as they were. An infinity gives NaN too (its codes are relative to an infinite scale)."""
    gen = torch.Generator(device=DEV).manual_seed(d)
    x, y = (torch.randn(1, rows, d, generator=gen, device=DEV) for _ in range(2))
    pre = None if norm is None else norm(d, eps=1e-5).to(DEV)
    w = torch.randint(-127, 128, (32, -(-d // 16) * 16), generator=gen, device=DEV).to(torch.int8)
    alpha = torch.rand(32, generator=gen, device=DEV)
    run = lambda: (lambda r, q, qs: (q, qs, lowbit.int8_linear(q, qs, w, alpha, k=d)))(  # noqa: E731
        *lowbit.residual_norm_quantized(x, y, pre_norm=pre))
    q, qs, out = run()
    assert bool(qs.isfinite().all()) and bool(out.isfinite().all())
    y[0, 2, d // 2], x[0, 5, d - 1], y[0, rows - 1, 0] = float("nan"), float("nan"), float("inf")
    q2, qs2, out2 = run()
    bad = torch.zeros(rows, dtype=torch.bool, device=DEV)
    bad[[2, 5, rows - 1]] = True
    assert bool(qs2[[2, 5]].isnan().all()) and bool(out2[bad].isnan().all())
    assert torch.equal(q2[~bad], q[~bad]) and torch.equal(qs2[~bad], qs[~bad]) and torch.equal(out2[~bad], out[~bad])


def test_norms_with_a_forward_of_their_own_are_refused():
    """A norm is read, not called: a class or a module that computes something else, or hooks that would run, are turned
    away; a class that only bears another name is taken."""
    class PlusOne(nn.LayerNorm):
        def forward(self, v):
            return nn.functional.layer_norm(v, self.normalized_shape, self.weight + 1, self.bias, self.eps)

    class Named(nn.RMSNorm):
        pass

    d = 64
    x, y = torch.randn(2, 3, d, device=DEV), torch.randn(2, 3, d, device=DEV)
    own, hooked, before, replaced = PlusOne(d).to(DEV), nn.LayerNorm(d).to(DEV), nn.RMSNorm(d).to(DEV), nn.LayerNorm(d).to(DEV)
    hooked.register_forward_hook(lambda module, args, out: 2 * out)
    before.register_forward_pre_hook(lambda module, args: (2 * args[0],))
    replaced.forward = lambda v: v
    for bad in (own, hooked, before, replaced):
        for option in ("post_norm", "pre_norm"):
            with pytest.raises(ValueError):
                lowbit.residual_norm(x, y, **{option: bad})
            with pytest.raises(ValueError):
                lowbit.residual_norm_quantized(x, y, **{option: bad})
    handle = replaced.register_forward_hook(lambda module, args, out: out)
    del replaced.forward
    handle.remove()
    for fine, like in ((Named(d, eps=1e-6).to(DEV), nn.RMSNorm(d, eps=1e-6).to(DEV)), (replaced, nn.LayerNorm(d).to(DEV))):
        for a, b in zip(lowbit.residual_norm(x, y, pre_norm=fine), lowbit.residual_norm(x, y, pre_norm=like)):
            assert torch.equal(a, b)


def test_reorder_refuses_outputs_that_overlap():
    """All states move in one launch: an output may share no byte with any state, nor with another output or itself.
    Buffers that only interleave are taken."""
    clips, beams = 3, 4
    parents = torch.tensor([[1, 0, 3, 2], [0, 0, 2, 1], [3, 3, 3, 0]], device=DEV, dtype=torch.int32)
    make = lambda *shape: torch.randn(*shape, device=DEV)  # noqa: E731
    a, b, free = make(clips, beams, 8), make(clips, beams, 8), make(clips, beams, 8)
    flat, pair, wide = make(clips * beams * 8 + 8), make(clips, beams, 2, 8), make(clips, beams, 12)
    shifted = [flat[i:i + clips * beams * 8].view(clips, beams, 8) for i in (0, 8)]
    call = lowbit.beam_reorder
    for states, out in (([a, b], [b, a]), ([a, b], [free, a]), ([a], [a]), (shifted[:1], shifted[1:]), (shifted[1:], shifted[:1]),
                        ([a, b], [free, free]), ([a], [make(8).expand(clips, beams, 8)]), ([wide[..., :8]], [wide[..., 4:]]),
                        ([pair[:, :, 0]], [pair.view(clips, 2, beams, 8)[:, 1]]), ([a], [a.view(beams, clips, 8).transpose(0, 1)])):
        with pytest.raises(ValueError):
            call(states, parents, out=out)
    row = torch.arange(clips, device=DEV)[:, None]
    layers, halves = make(clips, 2, beams, 8), make(2, 3, clips, beams, 5)
    for states, out, batch in (([pair[:, :, 0]], [pair[:, :, 1]], 0), ([layers[:, 1]], [layers[:, 0]], 0), ([halves[0]], [halves[1]], 1),
                               ([halves[:, 0], halves[:, 1]], [halves[:, 2], make(2, clips, beams, 5)], 1), ([a, a], [b, free], 0),
                               ([wide[..., :6]], [wide[..., 6:]], 0)):
        want = [s[row, parents.long()] if batch == 0 else s[:, row, parents.long()] for s in states]
        for got, o, w in zip(call(states, parents, batch_dim=batch, out=out), out, want):
            assert got is o and torch.equal(got, w)


def test_weights_are_complete_when_a_layer_is():
    """A layer's product is launched so that it may read the weights while earlier kernels finish; they must not be among
    what those write. The wait keeps the stream busy for some 50 ms before the weights' kernels."""
    weight = torch.randn(256, 128, device=DEV)
    Int8Linear(weight)   # what loads at a first use has loaded
    torch.cuda.synchronize()
    torch.cuda._sleep(100_000_000)
    Int8Linear(weight)
    assert torch.cuda.current_stream().query()


def test_search_refuses_lengths_of_other_clips():
    """One length for three clips would otherwise end all of them there; no clips and no frames are searches too."""
    dec = BeamDecoder(d_model=32, hidden=32, vocab=10, device=DEV)
    enc = torch.randn(3, 4, 32, device=DEV)
    for lengths in (torch.tensor([2]), torch.tensor(2), torch.tensor([[4], [4], [4]]), torch.tensor([4, 4])):
        with pytest.raises(ValueError):
            dec.search(enc, lengths, 2)
    for some in (enc[:0], enc[:, :0]):
        found = dec.search(some, torch.full((some.shape[0],), some.shape[1]), 2)
        assert found.labels.shape == (some.shape[0], 2, some.shape[1]) and found.scores.shape == (some.shape[0], 2)
