"""The elementwise gated recurrence over whole sequences (interface of ``chunk_hgrn`` of ``fla.ops.hgrn``), forward and backward."""
import functools
from typing import Optional, Tuple

import torch

from ... import _backend as be
from ..._native import host
from ...utils import _host_offsets, check_varlen_args, native_plan, resolve_offsets


@functools.lru_cache(maxsize=256)
def _segment(offs: Tuple[int, ...], D: int) -> int:
    """Tokens of the segments a packed batch's sequences are cut into."""
    lens = [b - a for a, b in zip(offs[:-1], offs[1:])]
    if not lens or min(lens) < 0:
        raise ValueError("offsets must be non-decreasing int64 positions")
    return be.lib().fla_hgrn_segment(sum(n > 0 for n in lens), sum(lens), max(lens), D)


def hgrn(x, g, initial_state, output_final_state, offsets, use_gate_in_kernel, lower_bound, inplace_state):
    plan = segment = None
    if offsets is not None:
        if x.dim() != 3:
            raise ValueError(f"fla_amd hgrn: x and g are [B, T, D], not {tuple(x.shape)}")
        check_varlen_args(x, offsets, False, initial_state)
        segment = _segment(_host_offsets(offsets), x.shape[-1])
        plan = native_plan(offsets, segment)
    return host().hgrn(x, g, lower_bound, initial_state, output_final_state, plan, segment, use_gate_in_kernel, inplace_state, offsets)


def chunk_hgrn(
    x: torch.Tensor,
    g: torch.Tensor,
    initial_state: Optional[torch.Tensor] = None,
    output_final_state: bool = False,
    offsets: Optional[torch.LongTensor] = None,
    cu_seqlens: Optional[torch.LongTensor] = None,
    use_gate_in_kernel: bool = False,
    lower_bound: Optional[torch.Tensor] = None,
) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    r"""``h_t = exp(g_t) * h_{t-1} + x_t``, ``o_t = h_t``, channel by channel.

    Args:
        x: ``[B, T, D]`` in bf16, fp16 or fp32.  Slices of a wider projection are read where they lie.
        g: log decays (at most 0), ``[B, T, D]``, in x's type or fp32.  ``-inf`` resets the state.
        initial_state: ``[N, D]`` for ``N`` sequences, or ``None``.
        output_final_state: also return the fp32 final state ``[N, D]``.
        offsets (synonym ``cu_seqlens``): int64 ``[N+1]`` sequence boundaries of a packed batch (batch size 1).  Rows ahead of the
            first and behind the last sequence come back as zeros, and have gradients of zero.
        use_gate_in_kernel: ``x`` and ``g`` are the layer's input and forget pre-activations ``i`` and ``f``; the operator forms
            ``a = lower_bound + (1 - lower_bound) * sigmoid(f)`` and ``h_t = a * h_{t-1} + (1 - a) * silu(i)`` in its own launches,
            forward and backward, so that neither the decays nor the gated inputs are written or read.
        lower_bound: ``[D]``, in ``[0, 1)``, with ``use_gate_in_kernel``; its gradient is formed too.  ``None``: 0.

    Returns ``(o, final_state)``, ``o`` in x's type.  The recurrence is evaluated in fp32.
    """
    return hgrn(x, g, initial_state, output_final_state, resolve_offsets(offsets, cu_seqlens), use_gate_in_kernel, lower_bound, False)
