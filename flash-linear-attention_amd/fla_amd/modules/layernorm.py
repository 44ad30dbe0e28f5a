"""RMS norm and layer norm with the residual's addition in front of them (interfaces of ``RMSNorm`` / ``rms_norm`` and ``LayerNorm`` / ``layer_norm``
of ``fla.modules``), and rows in 8 bits with a scale each, which :func:`quant_linear` multiplies."""
from __future__ import annotations

import torch
import torch.nn as nn

from .._native import host

_ROWS8 = {None: 0, False: 0, True: 1, torch.float8_e4m3fn: 1, torch.int8: 2}     # FLA_ROWS_*
_ROWS_ONLY, _RMS, _LAYER = 0, 1, 2


def _rows8(quantize) -> int:
    try:
        return _ROWS8[quantize]
    except (KeyError, TypeError):
        raise ValueError(f"fla_amd: rows in 8 bits are torch.float8_e4m3fn or torch.int8, not {quantize!r}") from None


def rms_norm(x, weight, bias=None, residual=None, prenorm=False, residual_in_fp32=False, eps=1e-6, quantize=False):
    """``y = s / sqrt(mean(s^2) + eps) * weight (+ bias)`` over the last dimension, ``s = x + residual``; one launch each way.

    ``prenorm``: returns ``(y, s)``, ``s`` in the residual's dtype (without a residual in x's, or with ``residual_in_fp32`` in fp32): the
    residual stream for the next norm.  ``s`` is summed and normalised in fp32; the backward starts from the ``s`` that is returned.
    ``quantize``: in the place of ``y`` the pair ``(q, scale)``, ``scale`` fp32 ``[...]`` without the last dimension and ``y ~ q * scale[..., None]``.
    ``True`` or ``torch.float8_e4m3fn``: ``q`` in that type, ``scale = max(max|y|, 1e-30) / 448``; ``torch.int8``: ``q`` the nearest whole numbers (halves to
    even), ``scale = max(max|y|, 1e-30) / 127``, infinite or NaN where the row holds such a value.  It has no gradient and is refused where one
    is wanted.  Rows of at most 16384 elements; weight and bias may be ``None``; the residual is in x's dtype or in fp32.
    A backward cannot be captured while an eager graph of the default stream holds one of the leaves (torch ends the process); unlike :func:`layer_norm`, this
    function does not look: its forward alone may be captured then."""
    return host().norm(x, weight, bias, residual, eps, prenorm, residual_in_fp32, _rows8(quantize), _RMS)


def layer_norm(x, weight, bias=None, residual=None, prenorm=False, residual_in_fp32=False, eps=1e-6, quantize=False):
    """``y = (s - mean(s)) / sqrt(var(s) + eps) * weight (+ bias)`` over the last dimension, ``s = x + residual``, ``var`` the mean square of
    ``s - mean(s)``; one launch each way.  Arguments, results and limits as those of :func:`rms_norm`.
    Under capture a call with gradients is refused while an eager graph of the default stream holds one of its leaves, or one behind them: a backward could
    not be captured."""
    return host().norm(x, weight, bias, residual, eps, prenorm, residual_in_fp32, _rows8(quantize), _LAYER)


def quantize_rows(x, dtype=torch.float8_e4m3fn):
    """``(q, scale)`` of the rows of ``x``: ``q`` in ``torch.float8_e4m3fn``, ``scale = max(max|x|, 1e-30) / 448`` in fp32 for each row, or ``q`` in
    ``torch.int8`` and ``scale = max(max|x|, 1e-30) / 127``, as in :func:`rms_norm`.  Rows of at most 2^23 elements."""
    rows8 = _rows8(dtype)
    if not rows8:
        raise ValueError("fla_amd quantize_rows: dtype is torch.float8_e4m3fn or torch.int8")
    return host().norm(x, None, None, None, 0.0, False, False, rows8, _ROWS_ONLY)


class _Norm(nn.Module):
    _fn = staticmethod(rms_norm)

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
        return self._fn(x, self.weight, self.bias, residual=residual, prenorm=prenorm, residual_in_fp32=residual_in_fp32,
                        eps=self.eps, quantize=quantize)


class RMSNorm(_Norm):
    """Interface of ``fla.modules.RMSNorm``: ``forward(x, residual=None, prenorm=False, residual_in_fp32=False)``, and ``quantize`` as in
    :func:`rms_norm`."""


class LayerNorm(_Norm):
    """Interface of ``fla.modules.LayerNorm``: ``forward(x, residual=None, prenorm=False, residual_in_fp32=False)``, and ``quantize`` as in
    :func:`rms_norm`.  ``bias=False`` is the default, as there."""
    _fn = staticmethod(layer_norm)
