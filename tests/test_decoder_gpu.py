"""The 8-bit projections and the beam search that runs the 8-bit map, the residual-norm step, the selection and the
reordering together (kea_kernels.int8, kea_kernels.decoder).

Tolerances. Int8Linear on weights of +-alpha has codes of +-127 and scale alpha / 127, so it equals the 1-bit projection but
for the rounding of that quotient and of the larger sums: four roundings more, 1e-6 of the terms' sum. A search's score is
the sum of T log-probabilities formed twice from the same logits: 2e-5 each (the selection's bound), T of them."""
from __future__ import annotations

import math

import pytest
import torch

from kea_kernels import lowbit
from kea_kernels.decoder import BeamDecoder
from kea_kernels.encoder import FastConformerEncoder, LowBitLinear, RandomLowBitWeights
from kea_kernels.int8 import Int8Linear, quantize_weight

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("n,k", [(96, 128), (1030, 640), (33, 100)])
def test_equals_the_one_bit_projection_on_signs(n, k):
    gen = torch.Generator(device=DEV).manual_seed(n)
    w = RandomLowBitWeights(n, k, 1, gen, keep_dense=True)
    bias = torch.randn(n, generator=gen, device=DEV)
    low = LowBitLinear(w.codes, 1, w.scale, bias, k, parts=1, device=torch.device(DEV))
    eight = Int8Linear(w.dense(), bias)
    x = torch.randn(3, 7, k, generator=gen, device=DEV)
    norm = torch.nn.LayerNorm(k).to(DEV)
    res = torch.randn(3, 7, n, generator=gen, device=DEV)
    with torch.inference_mode():
        for options in ({}, {"norm": norm}, {"input_silu": True}, {"silu": True}, {"residual": res, "residual_scale": 0.5}):
            a, b = low(x, **options), eight(x, **options)
            terms = 4.0 * k * float(w.scale.max()) + 4.0
            assert bool(((a - b).abs() <= 1e-6 * terms).all())


def test_weights_are_quantized_by_channel():
    w = torch.randn(40, 75, device=DEV) * torch.rand(40, 1, device=DEV)
    w[3] = 0.0
    codes, scale = quantize_weight(w)
    assert codes.dtype == torch.int8 and codes.stride(0) % 16 == 0
    assert bool(((codes.float() * scale[:, None] - w).abs() <= 0.5001 * scale[:, None]).all())
    assert bool((codes[3] == 0).all())
    with pytest.raises(ValueError):
        quantize_weight(codes)


def test_step_is_the_two_calls():
    lin = Int8Linear(torch.randn(64, 96, device=DEV))
    x, y = torch.randn(2, 5, 96, device=DEV), torch.randn(2, 5, 96, device=DEV)
    norm = torch.nn.LayerNorm(96).to(DEV)
    r, out = lin.step(x, y, scale=0.5, pre_norm=norm)
    r2, h = lowbit.residual_norm(x, y, scale=0.5, pre_norm=norm)
    assert torch.equal(r, r2) and torch.equal(out, lin(h))


def test_encoder_with_eight_bit_projections():
    """Int8Linear in every place of an encoder: the layer's own calls run on it, and the result stays near the encoder in
    FP32 products (8-bit codes of activations and weights: a few percent after two layers)."""
    make = lambda projections=None: FastConformerEncoder(layers=2, d_model=128, heads=4, ff=256, n_mels=32, sub_channels=8,  # noqa: E731
                                                         seed=3, device=DEV, keep_dense=True, projections=projections)
    plain = make()
    eight = [{name: Int8Linear(w.dense(), bias) for name, (w, bias) in layer.weights.items()} for layer in plain.layers]
    mixed = make()
    for layer, lins in zip(mixed.layers, eight):
        for name, lin in lins.items():
            lin.quant_pdl = layer.lin[name].quant_pdl
            layer.lin[name] = lin
    mel = torch.randn(2, 32, 120, generator=torch.Generator().manual_seed(1)).to(DEV)
    lengths = torch.tensor([15, 9], device=DEV)
    a, b = plain(mel, lengths), mixed(mel, lengths)
    assert bool(b.isfinite().all()) and float((a - b).norm() / a.norm()) < 0.05


@pytest.fixture(scope="module")
def decoder():
    return BeamDecoder(d_model=96, hidden=64, vocab=30, durations=5, seed=2, device=DEV)


def _log_probability(dec, enc, labels, length):
    """A label sequence's score, frame by frame with the same 8-bit network, the log-softmax in 64 bits."""
    frames = dec.enc(enc[None])
    state = dec.start.expand(1, 1, -1).contiguous()
    prediction, total = dec.pred(dec.before(state)), 0.0
    for f, label in enumerate(labels[:length]):
        total += float(torch.log_softmax(dec.logits(frames[:, f], prediction)[0, 0].double(), -1)[label])
        if label != dec.blank:
            state, prediction = dec.advance(state, torch.tensor([[label]], device=DEV, dtype=torch.int32))
    return total


@pytest.mark.parametrize("width", [1, 4, 8])
def test_search(decoder, width):
    """Every hypothesis' score is its labels' log-probability, hypotheses are distinct and in order, padding adds blanks at
    no cost, and a width of one is the greedy path."""
    b, t = 3, 12
    enc = torch.randn(b, t, 96, generator=torch.Generator().manual_seed(7)).to(DEV)
    lengths = torch.tensor([12, 7, 1])
    found = decoder.search(enc, lengths, width)
    assert found.labels.shape == (b, width, t) and found.scores.shape == (b, width)
    with torch.inference_mode():
        for i in range(b):
            n = int(lengths[i])
            rows = [tuple(r) for r in found.labels[i].tolist()]
            assert len(set(rows)) == width and all(v == decoder.blank for r in rows for v in r[n:])
            scores = found.scores[i].tolist()
            assert scores == sorted(scores, reverse=True)
            for row, score in zip(rows, scores):
                assert abs(_log_probability(decoder, enc[i], row, n) - score) <= 2e-5 * n
            if width == 1:
                frames, state = decoder.enc(enc[i:i + 1]), decoder.start.expand(1, 1, -1).contiguous()
                prediction = decoder.pred(decoder.before(state))
                for f in range(n):
                    label = int(decoder.logits(frames[:, f], prediction)[0, 0].argmax())
                    assert label == rows[0][f]
                    if label != decoder.blank:
                        state, prediction = decoder.advance(state, torch.tensor([[label]], device=DEV, dtype=torch.int32))
    assert found.best() == [[v for v in r[0] if v != decoder.blank] for r in found.labels.tolist()]


def test_wider_search_finds_no_worse_path(decoder):
    enc = torch.randn(4, 10, 96, generator=torch.Generator().manual_seed(9)).to(DEV)
    best = [decoder.search(enc, None, w).scores[:, 0] for w in (1, 8)]
    assert bool((best[1] >= best[0] - 2e-4).all())


def test_search_over_an_encoder():
    """Encoder states of padded clips into the search at the Parakeet joint's sizes: a clip's labels do not depend on what it
    is batched with."""
    enc = FastConformerEncoder(layers=1, d_model=128, heads=4, ff=256, n_mels=32, sub_channels=8, device=DEV)
    dec = BeamDecoder(d_model=128, device=DEV)
    mel = torch.randn(2, 32, 160, generator=torch.Generator().manual_seed(4)).to(DEV)
    lengths = torch.tensor([20, 11])
    states = enc(mel, lengths)
    both = dec.search(states, lengths, 4)
    alone = dec.search(states[1:, :11], None, 4)
    assert both.best()[1] == alone.best()[0] and math.isclose(float(both.scores[1, 0]), float(alone.scores[0, 0]), abs_tol=1e-3)
