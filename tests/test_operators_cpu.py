"""CPU: the 8-bit linear map, the residual-norm step and the beam search refuse bad descriptors before any device work, and
host tensors are turned away."""
from __future__ import annotations

import ctypes
import re

import pytest
import torch

from conftest import ROOT
from kea_kernels import _lib, lowbit

HEADER = (ROOT / "include" / "kea_lowbit.h").read_text()
KINDS = {"int64_t": ctypes.c_int64, "int32_t": ctypes.c_int32, "float": ctypes.c_float}


def _struct(name):
    """The header's struct as a ctypes one, every pointer a c_void_p."""
    body = HEADER[HEADER.index(f"typedef struct {name} "):HEADER.index(f"}} {name};")]
    body = re.sub(r"/\*.*?\*/", "", body[body.index("{") + 1:], flags=re.S)
    fields = []
    for line in filter(None, (part.strip() for part in body.split(";"))):
        kind = re.match(r"(?:const )?(\w+)", line).group(1)
        for item in line[line.index(kind) + len(kind):].split(","):
            fields.append((item.strip(" *"), ctypes.c_void_p if "*" in item else KINDS[kind]))
    return type(name, (ctypes.Structure,), {"_fields_": fields})


Int8Desc, ResidualNormDesc, BeamDesc, ReorderDesc, ReorderItem = map(
    _struct, ("KeaInt8Desc", "KeaResidualNormDesc", "KeaBeamDesc", "KeaReorderDesc", "KeaReorderItem"))


def _status(entry, desc, good, *more, **changes):
    return getattr(_lib.lib(), entry)(ctypes.byref(desc(**{**good, **changes})), *more, None)


def test_int8_descriptors():
    good = dict(q=16, ldq=64, qs=16, w=16, ldw=64, alpha=16, y=16, ldy=32, m=4, n=32, k=64)
    status = lambda **c: _status("kea_lowbit_int8_gemm", Int8Desc, good, **c)  # noqa: E731
    assert status(m=0) == _lib.OK
    for change in (dict(m=-1), dict(n=0), dict(k=0), dict(q=None), dict(qs=None), dict(w=None), dict(alpha=None), dict(y=None),
                   dict(ldq=48), dict(ldw=48), dict(ldy=31), dict(y_type=3), dict(flags=4), dict(kernel=9),
                   dict(residual=16, ld_residual=8), dict(acc=16, ld_acc=8)):
        assert status(**change) == _lib.INVALID_VALUE, change
    for change in (dict(q=24), dict(w=8), dict(ldq=72), dict(ldw=65), dict(y=18), dict(residual=17, ld_residual=32),
                   dict(qs=18), dict(alpha=17), dict(bias=18), dict(acc=18, ld_acc=32)):
        assert status(**change) == _lib.ALIGNMENT, change
    assert status(k=131072, ldq=131072, ldw=131072) == _lib.UNSUPPORTED
    assert _lib.lib().kea_lowbit_int8_gemm(None, None) == _lib.INVALID_VALUE


def test_residual_norm_descriptors():
    good = dict(x=32, y=32, r=32, h=32, ldx=64, ldy=64, ldr=64, ldh=64, frames=4, m=4, d=64, scale=1.0)
    status = lambda **c: _status("kea_lowbit_residual_norm", ResidualNormDesc, good, **c)  # noqa: E731
    assert status(m=0) == _lib.OK
    for change in (dict(x=None), dict(y=None), dict(r=None), dict(h=None), dict(frames=0), dict(d=0), dict(m=-1), dict(x_type=3),
                   dict(y_type=-1), dict(h_type=5), dict(gate_act=2), dict(post=1), dict(pre=2), dict(pre=3, pre_weight=32),
                   dict(flags=2), dict(ldx=63), dict(ldy=60), dict(ldr=1), dict(ldh=0), dict(q=16, ldq=64), dict(q=16, ldq=32, qs=16)):
        assert status(**change) == _lib.INVALID_VALUE, change
    assert status(x=34) == status(y=33) == status(h=2) == status(gate=34) == _lib.ALIGNMENT
    assert status(d=16385, ldx=16385, ldy=16385, ldr=16385, ldh=16385) == _lib.UNSUPPORTED


def test_beam_descriptors():
    good = dict(logits=16, ld_clip=200, ld_beam=50, scores=16, out_scores=16, parents=16, labels=16, clips=2, beams=4, vocab=50,
                width=4, end=-1)
    status = lambda **c: _status("kea_lowbit_beam_select", BeamDesc, good, **c)  # noqa: E731
    assert status(clips=0) == _lib.OK
    for change in (dict(logits=None), dict(scores=None), dict(out_scores=None), dict(parents=None), dict(labels=None), dict(clips=-1),
                   dict(beams=0), dict(vocab=0), dict(width=0), dict(end=50), dict(end=-2), dict(ended=16), dict(logits_type=3),
                   dict(flags=2)):
        assert status(**change) == _lib.INVALID_VALUE, change
    for change in (dict(beams=33), dict(width=33), dict(vocab=1 << 29), dict(beams=1, vocab=3), dict(clips=1 << 28)):
        assert status(**change) == _lib.UNSUPPORTED, change
    assert status(logits=18) == status(scores=17) == status(parents=18) == _lib.ALIGNMENT


def test_reorder_descriptors():
    good = dict(parents=16, count=1, clips=2, beams=4, width=4)
    item = dict(src=16, dst=4096, src_clip=64, src_beam=16, dst_clip=64, dst_beam=16, row_bytes=16, groups=1)
    status = lambda row={}, **c: _status("kea_lowbit_beam_reorder", ReorderDesc, good,  # noqa: E731
                                         ctypes.byref(ReorderItem(**{**item, **row})), **c)
    assert status(count=0) == status(clips=0) == status(row=dict(row_bytes=0)) == _lib.OK
    for change in (dict(parents=None), dict(count=-1), dict(count=33), dict(beams=0), dict(width=0), dict(flags=2),
                   dict(row=dict(groups=0)), dict(row=dict(row_bytes=-1)), dict(row=dict(src=None)), dict(row=dict(dst=None))):
        assert status(**change) == _lib.INVALID_VALUE, change
    assert status(row=dict(row_bytes=1 << 31)) == status(row=dict(groups=1 << 29)) == _lib.UNSUPPORTED
    assert status(parents=18) == _lib.ALIGNMENT


def test_host_tensors_are_refused():
    q, s = torch.zeros(2, 16, dtype=torch.int8), torch.zeros(2)
    with pytest.raises(ValueError):
        lowbit.int8_linear(q, s, q, s)
    with pytest.raises(ValueError):
        lowbit.residual_norm(torch.zeros(2, 8), torch.zeros(2, 8))
    with pytest.raises(ValueError):
        lowbit.residual_norm_quantized(torch.zeros(2, 8), torch.zeros(2, 8))
    with pytest.raises(ValueError):
        lowbit.beam_select(torch.zeros(1, 2, 8), torch.zeros(1, 2))
    with pytest.raises(ValueError):
        lowbit.beam_reorder([torch.zeros(1, 2, 8)], torch.zeros(1, 2, dtype=torch.int32))
