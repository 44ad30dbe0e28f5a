"""The elementwise gated recurrence token by token (interface of ``fused_recurrent_hgrn`` of ``fla.ops.hgrn``): the decode step."""
from typing import Optional, Tuple

import torch

from ..._native import host
from ...utils import resolve_offsets
from .chunk import hgrn


def fused_recurrent_hgrn(
    x: torch.Tensor,
    g: torch.Tensor,
    initial_state: Optional[torch.Tensor] = None,
    output_final_state: bool = False,
    offsets: Optional[torch.LongTensor] = None,
    cu_seqlens: Optional[torch.LongTensor] = None,
    use_gate_in_kernel: bool = False,
    lower_bound: Optional[torch.Tensor] = None,
    inplace_state: bool = False,
) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Arguments and results of :func:`chunk_hgrn`.  One token per sequence is a single elementwise launch, which with
    ``inplace_state`` updates the fp32 ``initial_state`` where it lies (its address stays, as a captured step needs); more tokens
    go through the scan."""
    if offsets is None and cu_seqlens is None:   # a decode step: straight to the host extension
        return host().hgrn(x, g, lower_bound, initial_state, output_final_state, None, None, use_gate_in_kernel, inplace_state, None)
    return hgrn(x, g, initial_state, output_final_state, resolve_offsets(offsets, cu_seqlens), use_gate_in_kernel, lower_bound,
                inplace_state)
