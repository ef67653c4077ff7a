"""A beam search over the joint network's labels, at 8 bits: what comes after the encoder. Encoder and prediction projections,
the prediction block and the joint's output layer are 8-bit maps (int8.Int8Linear); a hypothesis' prediction state takes one
gated residual step per label, straight into the next projection's codes (lowbit.residual_norm_quantized); each frame's
continuations are chosen over hypotheses and labels (lowbit.beam_select) and the hypotheses' states follow their parents
(lowbit.beam_reorder).

Shapes are the Parakeet TDT joint's (1024 -> 640, 640 -> 640, 640 -> 1024 labels + blank + 5 durations), weights random and the
module's own: they are not encoder.TDTJoint's, and the prediction block is a stand-in that takes a label by a gate, not the
recogniser's LSTM. The search chooses one label per frame, blank leaving the prediction state as it is; the durations' logits
are left aside.
The reference decodes greedily, one clip at a time (src/kea_kernels/ternary/decoder_kernels.py:139-157).
"""
from __future__ import annotations

import dataclasses
import math

import torch
from torch import Tensor, nn

from kea_kernels import lowbit
from kea_kernels.int8 import Int8Linear


@dataclasses.dataclass
class Hypotheses:
    """A search's results, best first: labels int32 [B, width, T] (blank where a frame adds none), scores FP32 [B, width]."""
    labels: Tensor
    scores: Tensor
    blank: int

    def best(self) -> list[list[int]]:
        """Every clip's best hypothesis without its blanks."""
        return [[v for v in row if v != self.blank] for row in self.labels[:, 0].tolist()]


class BeamDecoder(nn.Module):
    def __init__(self, d_model: int = 1024, hidden: int = 640, vocab: int = 1024, durations: int = 5, seed: int = 1, device=None):
        super().__init__()
        device = torch.device(device if device is not None else "cuda")
        gen = torch.Generator().manual_seed(seed)
        rnd = lambda *shape: torch.randn(*shape, generator=gen)  # noqa: E731
        linear = lambda n, k: Int8Linear(rnd(n, k) / math.sqrt(k), 0.02 * rnd(n), device=device)  # noqa: E731
        self.vocab, self.blank, self.hidden = vocab, vocab, hidden
        self.enc, self.pred = linear(hidden, d_model), linear(hidden, hidden)
        self.cell, self.out = linear(hidden, hidden), linear(vocab + 1 + durations, hidden)
        self.after, self.before = nn.LayerNorm(hidden), nn.LayerNorm(hidden)   # of the prediction block, of its projection
        self.register_buffer("gates", rnd(vocab + 1, hidden))                  # a label's gate on the block
        self.register_buffer("start", rnd(hidden))
        self.to(device)

    def logits(self, frame: Tensor, prediction: Tensor) -> Tensor:
        """frame [B, hidden] and prediction [B, W, hidden] projections -> label logits [B, W, vocab + 1] (a view: the
        duration logits lie behind each row)."""
        return self.out((frame[:, None] + prediction).relu())[..., : self.vocab + 1]

    def advance(self, state: Tensor, labels: Tensor) -> tuple[Tensor, Tensor]:
        """The prediction states [B, W, hidden] after `labels` [B, W], and their projections."""
        return self.pred.step(state, self.cell(state), post_norm=self.after, gate=self.gates[labels.long()], gate_act="sigmoid",
                              pre_norm=self.before)

    @torch.inference_mode()
    def search(self, enc: Tensor, lengths: Tensor | None = None, width: int = 4) -> Hypotheses:
        """enc FP32 [B, T, d_model] (with `lengths`, int [B]: frames of each clip, the rest is padding) -> the `width` best
        hypotheses of every clip. Past a clip's end its hypotheses have ended: they add blanks at no cost."""
        b, t, _ = enc.shape
        if lengths is not None and tuple(lengths.shape) != (b,):
            raise ValueError(f"lengths must be [{b}], got {tuple(lengths.shape)}")
        device, blank = enc.device, self.blank
        frames = self.enc(enc)
        labels = torch.full((t, b, width), blank, device=device, dtype=torch.int32)
        parents = torch.zeros_like(labels)
        scores = torch.full((b, width), -math.inf, device=device)
        scores[:, 0] = 0.0                                             # one hypothesis to begin with
        state = self.start.expand(b, width, -1).contiguous()
        prediction = self.pred(self.before(state))
        ends = None if lengths is None else lengths.to(device)
        for f in range(t):
            ended = None if ends is None else (ends <= f)[:, None].expand(b, width).contiguous()
            step = lowbit.beam_select(self.logits(frames[:, f], prediction), scores, end=blank, ended=ended,
                                      out=lowbit.BeamStep(torch.empty_like(scores), parents[f], labels[f], None))
            scores = step.scores
            state, prediction = lowbit.beam_reorder([state, prediction], step.parents)
            moved, projected = self.advance(state, step.tokens)
            keep = (step.tokens == blank)[..., None]
            state, prediction = torch.where(keep, state, moved), torch.where(keep, prediction, projected)
        return Hypotheses(self.trace(parents, labels), scores, blank)

    @staticmethod
    def trace(parents: Tensor, labels: Tensor) -> Tensor:
        """Follows parents [T, B, W] back from the last frame: labels [T, B, W] -> [B, W, T] by hypothesis."""
        t, b, w = labels.shape
        at = torch.arange(w, device=labels.device).expand(b, w)
        out = torch.empty(b, w, t, device=labels.device, dtype=labels.dtype)
        for f in range(t - 1, -1, -1):
            out[:, :, f] = labels[f].gather(1, at)
            at = parents[f].long().gather(1, at)
        return out
