"""The operators around an 8-bit model where a call can go wrong without a word: offsets past 32 bits, scores that tie, norms
that are not what their class says, buffers that overlap, rows that are not numbers, labels that are masked.

Tolerances stand at each test; where none is named the values have to be equal."""
from __future__ import annotations

import pytest
import torch

from kea_kernels import _lib, lowbit

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
