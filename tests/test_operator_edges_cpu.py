"""CPU: the operators around an 8-bit model at the edges of what they take."""
from __future__ import annotations

from kea_kernels import _lib
from test_operators_cpu import BeamDesc, _status


def test_beam_labels_stay_inside_32_bits():
    """Label indices are formed up to 4095 past a row's end before they are compared with it, so the last 4096 numbers of
    32 bits are refused; what is accepted goes on to the check of alignment."""
    good = dict(logits=18, ld_clip=1 << 31, ld_beam=1 << 31, scores=16, out_scores=16, parents=16, labels=16, clips=1, beams=1,
                width=1, end=-1)
    status = lambda **c: _status("kea_lowbit_beam_select", BeamDesc, good, **c)  # noqa: E731
    for beams, vocab in ((1, 2 ** 31 - 1), (1, 2 ** 31 - 4095), (2, 2 ** 30 - 2047), (32, 2 ** 26 - 127)):
        assert status(beams=beams, vocab=vocab) == _lib.UNSUPPORTED
    for beams, vocab in ((1, 2 ** 31 - 4096), (2, 2 ** 30 - 2048), (32, 2 ** 26 - 128)):
        assert status(beams=beams, vocab=vocab) == _lib.ALIGNMENT
