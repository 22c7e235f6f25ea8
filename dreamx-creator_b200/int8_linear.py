"""``Int8Linear``: ``Fp8Linear``'s interface with weights and activations as 8-bit integers.

The weight is quantised once, per output channel: scale = max(amax / 127, 1e-12), codes
round(w / scale). A call quantises the activation per token (``ops.quant_rows``) and
multiplies the codes, summed exactly in int32, with the bias in the product's epilogue
(``ops.int8_gemm``); ``forward_codes`` takes rows that are quantised already
(``ops.add_rms_quant``). There is no CPU path: without the library or a GPU a call raises.
"""
from __future__ import annotations

import torch
import torch.nn as nn

from . import _lib, ops
from .fp8_linear import TARGETS_ALL, Fp8Linear, convert_linears

INT8_MAX = 127.0


def quantize_weight_int8(weight: torch.Tensor):
    """Per-output-channel int8 of a [N, K] weight -> (codes [N, K] in rows that are a
    multiple of 16 bytes apart, fp32 scale [N]). One-time model preparation, in torch."""
    w = weight.detach().float()
    scale = (w.abs().amax(dim=-1) / INT8_MAX).clamp_min(1e-12)
    q = ops.code_rows(*w.shape, torch.int8, w.device)
    q.copy_(torch.round(w / scale[:, None]).clamp(-INT8_MAX, INT8_MAX))
    return q, scale.contiguous()


class Int8Linear(Fp8Linear):
    """Frozen inference Linear computed as a row-wise scaled int8 product."""

    _FIXED_DTYPE = {"weight_int8": torch.int8, "weight_scale": torch.float32}

    def __init__(self, weight, bias=None):
        nn.Module.__init__(self)
        if weight.dim() != 2:
            raise ValueError(f"Int8Linear needs a 2-D [out, in] weight, got {tuple(weight.shape)}")
        self.out_features, self.in_features = (int(v) for v in weight.shape)
        q, s = quantize_weight_int8(weight)
        # the buffer is the padded rows: a module-wide move copies them densely
        self.register_buffer("weight_int8", q.as_strided((q.shape[0], q.stride(0)), (q.stride(0), 1)),
                             persistent=False)
        self.register_buffer("weight_scale", s, persistent=False)
        # added in the output's type (a module-wide cast of 16 or 32 bits sets it)
        self.register_buffer("bias", None if bias is None else bias.detach().clone().contiguous(),
                             persistent=False)
        # zero-element stand-in: callers read .weight.dtype
        self.register_buffer("weight", weight.new_empty(0), persistent=False)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        """x [..., in_features] (bf16, fp16 or fp32) -> [..., out_features] in x's dtype."""
        if x.shape[-1] != self.in_features:
            raise ValueError(f"Int8Linear expects {self.in_features} input features, "
                             f"got {x.shape[-1]}")
        q, scale = ops.quant_rows(ops.as_rows(x, self.in_features))
        return self.forward_codes(q, scale, x.dtype).view(*x.shape[:-1], self.out_features)

    def forward_codes(self, q, scale, dtype=torch.bfloat16, out=None):
        """The product of rows quantised earlier: codes q [M, in_features], fp32 scale [M]."""
        if q.shape[1] != self.in_features:
            raise _lib.SrditError(f"Int8Linear expects {self.in_features} input features, "
                                  f"got {q.shape[1]}")
        bias = self.bias
        if bias is not None and bias.dtype != dtype:
            bias = bias.to(dtype)
        return ops.int8_gemm(q, scale, self.weight_int8[:, :self.in_features], self.weight_scale,
                             bias, out, out_dtype=dtype)

    def extra_repr(self):
        return (f"in_features={self.in_features}, out_features={self.out_features}, "
                f"bias={self.bias is not None}, int8=per-token x per-channel, backend=b200")


def convert_linears_to_int8(model: nn.Module, targets=TARGETS_ALL, skip_first=0, skip_last=0,
                            blocks_attr="blocks"):
    """``convert_linears_to_fp8`` with ``Int8Linear``."""
    return convert_linears(model, Int8Linear, targets, skip_first, skip_last, blocks_attr)
