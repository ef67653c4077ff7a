"""Projections at 8 bits: layers an export leaves unpacked, a joint network, or a whole encoder where the 1- and 2-bit codes
are not wanted. `Int8Linear` takes the place of `encoder.LowBitLinear` wherever that is used (a layer's `projections`, the
joint), with the same calls; its weights are INT8 codes with one scale per output channel, its activations the
quantizer's first INT8 part, its product `lowbit.int8_linear`.

kea-kernels quantises 264 encoder linears to 1 or 2 bits (src/kea_kernels/formats.py:39-46) and keeps the joint in FP32
(src/kea_kernels/ternary/decoder_kernels.py:139-157); 8-bit weights have no counterpart there.
"""
from __future__ import annotations

import torch
from torch import Tensor, nn

from kea_kernels import lowbit


def quantize_weight(weight: Tensor) -> tuple[Tensor, Tensor]:
    """FP32 weights [N, K] -> INT8 codes [N, K] in rows of a multiple of 16 bytes, and FP32 scales [N]: per output channel
    scale = max(amax / 127, 1e-30), code = rint(w / scale), the quantizer's formula for an activation row."""
    if weight.dim() != 2 or not weight.is_floating_point():
        raise ValueError("weight must be a floating-point matrix [N, K]")
    w = weight.float()
    n, k = w.shape
    scale = (w.abs().amax(1) / 127.0).clamp_min(1e-30) if k else torch.full((n,), 1e-30, device=w.device)
    store = torch.zeros(n, -(-k // 16) * 16, device=w.device, dtype=torch.int8)
    store[:, :k] = torch.round(w / scale[:, None]).to(torch.int8)
    return store[:, :k], scale


class Int8Linear(nn.Module):
    """One 8-bit projection: the quantizer (optional fused LayerNorm / input SiLU) into one INT8 part, then the INT8 product
    with token and channel scales, bias, optional SiLU and skip connection. FP32 in, FP32 out, the calls of
    encoder.LowBitLinear."""

    wbits, parts = 8, 1

    def __init__(self, weight: Tensor, bias: Tensor | None = None, *, device: torch.device | None = None, pdl: bool = True):
        super().__init__()
        device = weight.device if device is None else torch.device(device)
        codes, scale = quantize_weight(weight.detach().to(device))
        self.out_features, self.in_features, self.pdl, self.quant_pdl = codes.shape[0], codes.shape[1], pdl, False
        self.register_buffer("panels", codes.as_strided((codes.shape[0], codes.stride(0)), codes.stride()))
        self.register_buffer("scale", scale)
        self.register_buffer("bias", None if bias is None else bias.detach().to(device=device, dtype=torch.float32).contiguous())
        if device.type == "cuda":   # the product may read its weights before earlier kernels of its stream have ended
            torch.cuda.current_stream(device).synchronize()

    def product(self, q: Tensor, qs: Tensor, *, silu: bool = False, residual: Tensor | None = None,
                residual_scale: float = 1.0, dtype: torch.dtype = torch.float32, pdl: bool | None = None) -> Tensor:
        """Codes [m, >= K] and scales [m] of one INT8 part -> [m, N]."""
        return lowbit.int8_linear(q, qs, self.panels, self.scale, self.bias, k=self.in_features, dtype=dtype, silu=silu,
                                  residual=residual, residual_scale=residual_scale, pdl=self.pdl if pdl is None else pdl)

    def forward(self, x: Tensor, *, norm: nn.LayerNorm | None = None, input_silu: bool = False, silu: bool = False,
                residual: Tensor | None = None, residual_scale: float = 1.0, pre_norm: nn.LayerNorm | None = None,
                normed: Tensor | None = None) -> Tensor:
        """x FP32 [B, T, K] (any strides) -> [B, T, N], with LowBitLinear.forward's options."""
        b, t, k = x.shape
        m = b * t
        q, qs, ldq = lowbit.quantize(x, (x.stride(0), x.stride(1), x.stride(2), t), m, k, 1, norm=norm,
                                     input_silu=input_silu, pdl=self.pdl and self.quant_pdl, pre_norm=pre_norm,
                                     normed=None if normed is None else normed.view(m, k))
        return self.from_quantized(q, qs, ldq, b, t, silu=silu, residual=residual, residual_scale=residual_scale)

    def from_quantized(self, q: Tensor, qs: Tensor, ldq: int, b: int, t: int, *, silu: bool = False,
                       residual: Tensor | None = None, residual_scale: float = 1.0) -> Tensor:
        """The product on activations already quantized into one part (q [1, b*t, ldq], qs [1, b*t]) -> FP32 [b, t, N]."""
        res = None if residual is None else residual.reshape(b * t, self.out_features)
        return self.product(q[0], qs[0], silu=silu, residual=res, residual_scale=residual_scale).view(b, t, self.out_features)

    def step(self, x: Tensor, y: Tensor, *, silu: bool = False, dtype: torch.dtype = torch.float32,
             **options) -> tuple[Tensor, Tensor]:
        """The step from a block's output y to this projection: lowbit.residual_norm_quantized(x, y, **options), whose
        INT8 codes go straight into the product -> (the residual stream [..., K], [..., N])."""
        r, q, qs = lowbit.residual_norm_quantized(x, y, **options)
        out = lowbit.int8_linear(q, qs, self.panels, self.scale, self.bias, k=self.in_features, dtype=dtype, silu=silu,
                                 pdl=self.pdl)
        return r, out.view(*x.shape[:-1], self.out_features)
