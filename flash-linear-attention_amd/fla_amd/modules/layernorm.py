"""RMS norm with the residual's addition in front of it (interface of ``RMSNorm`` / ``rms_norm`` of ``fla.modules``), and rows in 8 bits
with a scale each, which :func:`quant_linear` multiplies."""
from __future__ import annotations

import torch
import torch.nn as nn

from .._native import host


def rms_norm(x, weight, bias=None, residual=None, prenorm=False, residual_in_fp32=False, eps=1e-6, quantize=False):
    """``y = s / sqrt(mean(s^2) + eps) * weight (+ bias)`` over the last dimension, ``s = x + residual``; one launch each way.

    ``prenorm``: returns ``(y, s)``, ``s`` in the residual's dtype (without a residual in x's, or with ``residual_in_fp32`` in fp32): the
    residual stream for the next norm.  ``s`` is summed and normalised in fp32; the backward starts from the ``s`` that is returned.
    ``quantize``: in the place of ``y`` the pair ``(q, scale)``, ``q`` in ``torch.float8_e4m3fn`` and ``scale`` fp32 ``[...]`` without the last
    dimension, ``y ~ q * scale[..., None]`` with ``scale = max(max|y|, 1e-30) / 448``.  It has no gradient and is refused where one is
    wanted.  Rows of at most 16384 elements; weight and bias may be ``None``; the residual is in x's dtype or in fp32."""
    return host().rms_norm(x, weight, bias, residual, eps, prenorm, residual_in_fp32, quantize, True)


def quantize_rows(x):
    """``(q, scale)`` of the rows of ``x``: ``q`` in ``torch.float8_e4m3fn``, ``scale = max(max|x|, 1e-30) / 448`` in fp32 for each row.
    Rows of at most 2^23 elements, as many as :func:`quant_linear` takes."""
    return host().rms_norm(x, None, None, None, 0.0, False, False, True, False)


class RMSNorm(nn.Module):
    """Interface of ``fla.modules.RMSNorm``: ``forward(x, residual=None, prenorm=False, residual_in_fp32=False)``, and ``quantize`` as in
    :func:`rms_norm`."""

    def __init__(self, hidden_size: int, elementwise_affine: bool = True, bias: bool = False, eps: float = 1e-5):
        super().__init__()
        self.hidden_size = hidden_size
        self.elementwise_affine = elementwise_affine
        self.eps = eps
        self.register_parameter("weight", nn.Parameter(torch.ones(hidden_size)) if elementwise_affine else None)
        self.register_parameter("bias", nn.Parameter(torch.zeros(hidden_size)) if elementwise_affine and bias else None)

    def __repr__(self) -> str:
        s = f"{self.__class__.__name__}({self.hidden_size}"
        if not self.elementwise_affine:
            s += f", elementwise_affine={self.elementwise_affine}"
        return s + f", eps={self.eps})"

    def forward(self, x, residual=None, prenorm=False, residual_in_fp32=False, quantize=False):
        return rms_norm(x, self.weight, self.bias, residual=residual, prenorm=prenorm, residual_in_fp32=residual_in_fp32,
                        eps=self.eps, quantize=quantize)
