"""The gated product of a feed-forward block, forward and backward, and the block around it."""
from __future__ import annotations

from typing import Optional

import torch
import torch.nn as nn

from .._native import host

_ACTIVATIONS = {None: 0, "silu": 1, "swish": 1, "gelu": 2, "relu": 3}


def _activation(activation: Optional[str], who: str) -> int:
    try:
        return _ACTIVATIONS[activation]
    except (KeyError, TypeError):
        raise ValueError(f"fla_amd {who}: unknown activation {activation!r}") from None


def gated_linear(x: torch.Tensor, gate_weight: torch.Tensor, up_weight: torch.Tensor, gate_bias: Optional[torch.Tensor] = None,
                 up_bias: Optional[torch.Tensor] = None, activation: Optional[str] = "silu") -> torch.Tensor:
    """``act(x @ gate_weight.T + gate_bias) * (x @ up_weight.T + up_bias)`` for ``x`` ``[..., K]`` and weights ``[F, K]``, all in bf16 or all in fp16;
    ``[..., F]``.  One launch (two where there are few tiles and K is summed in slices); both products, the activation and the product of the two
    are formed in fp32 and rounded once.

    ``activation``: ``"silu"`` (``"swish"``), ``"gelu"`` (of the error function), ``"relu"`` (its slope at 0 is 0) or ``None``; biases in any floating type.
    For a backward both pre-activations are kept in fp32, ``2 F`` values a row; it rounds the gradients of both to x's type, in its range, ahead of the
    products that form those of x and the weights.  Gradients of operands that do not ask for one are not formed.  There are no second derivatives.
    Under capture a call with gradients is refused while an eager graph of the default stream holds one of its leaves, or one behind them (the parameters that
    autocast casts, those of the layers ahead): a backward could not be captured.
    Under autocast the operands are cast to its type, as ``torch.nn.functional.linear`` does."""
    code = _activation(activation, "gated_linear")
    if torch.is_autocast_enabled("cuda") and x.is_cuda:
        dtype = torch.get_autocast_dtype("cuda")
        x, gate_weight, up_weight = x.to(dtype), gate_weight.to(dtype), up_weight.to(dtype)
    return host().gated_linear(x, gate_weight, up_weight, gate_bias, up_bias, code)


class GatedMLP(nn.Module):
    """``down_proj(act(gate_proj(x)) * up_proj(x))``, the first two projections, the activation and the product through :func:`gated_linear`, the last one a
    ``torch.nn.Linear``.  Without ``intermediate_size`` it is ``hidden_size * hidden_ratio * 2 / 3`` rounded up to a multiple of 256."""

    def __init__(self, hidden_size: int, intermediate_size: Optional[int] = None, hidden_ratio: int = 4, hidden_act: Optional[str] = "swish",
                 bias: bool = False, device=None, dtype=None):
        super().__init__()
        _activation(hidden_act, "GatedMLP")
        if intermediate_size is None:
            intermediate_size = -(-int(hidden_size * hidden_ratio * 2 / 3) // 256) * 256
        self.hidden_size, self.intermediate_size, self.hidden_act = hidden_size, intermediate_size, hidden_act
        how = {"bias": bias, "device": device, "dtype": dtype}
        self.gate_proj = nn.Linear(hidden_size, intermediate_size, **how)
        self.up_proj = nn.Linear(hidden_size, intermediate_size, **how)
        self.down_proj = nn.Linear(intermediate_size, hidden_size, **how)

    def extra_repr(self) -> str:
        return f"hidden_act={self.hidden_act}"

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return self.down_proj(gated_linear(x, self.gate_proj.weight, self.up_proj.weight, self.gate_proj.bias, self.up_proj.bias, self.hidden_act))
