"""CPU: boundaries of a packed batch on another device than the operands are refused ahead of any launch.

The operands lie on the ``meta`` device, which no kernel can read either: what raises is the check of the devices."""
import pytest
import torch

from fla_amd import _backend as be


def _calls():
    from fla_amd.ops import (chunk_delta_rule, chunk_gated_delta_rule, chunk_gla, chunk_global_cumsum, chunk_hgrn, chunk_local_cumsum,
                             chunk_simple_gla, fused_recurrent_gated_delta_rule, fused_recurrent_gla, fused_recurrent_hgrn,
                             fused_recurrent_simple_gla)
    kw = dict(head_first=False)
    return {
        "chunk_hgrn": lambda t, o: chunk_hgrn(t(1, 8, 64), t(1, 8, 64), cu_seqlens=o),
        "fused_recurrent_hgrn": lambda t, o: fused_recurrent_hgrn(t(1, 8, 64), t(1, 8, 64), cu_seqlens=o),
        "chunk_gla": lambda t, o: chunk_gla(*[t(1, 8, 1, 64) for _ in range(4)], cu_seqlens=o, **kw),
        "chunk_simple_gla": lambda t, o: chunk_simple_gla(*[t(1, 8, 1, 64) for _ in range(3)], t(1, 8, 1), cu_seqlens=o, **kw),
        "chunk_gated_delta_rule": lambda t, o: chunk_gated_delta_rule(*[t(1, 8, 1, 64) for _ in range(3)], t(1, 8, 1), t(1, 8, 1),
                                                                      cu_seqlens=o, **kw),
        "chunk_delta_rule": lambda t, o: chunk_delta_rule(*[t(1, 8, 1, 64) for _ in range(3)], t(1, 8, 1), cu_seqlens=o, **kw),
        "fused_recurrent_gla": lambda t, o: fused_recurrent_gla(*[t(1, 8, 1, 64) for _ in range(4)], cu_seqlens=o, **kw),
        "fused_recurrent_simple_gla": lambda t, o: fused_recurrent_simple_gla(*[t(1, 8, 1, 64) for _ in range(3)], t(1, 8, 1),
                                                                              cu_seqlens=o, **kw),
        "fused_recurrent_gated_delta_rule": lambda t, o: fused_recurrent_gated_delta_rule(
            *[t(1, 8, 1, 64) for _ in range(3)], t(1, 8, 1), t(1, 8, 1), cu_seqlens=o, **kw),
        "chunk_local_cumsum": lambda t, o: chunk_local_cumsum(t(1, 8, 1), 64, offsets=o, **kw),
        "chunk_global_cumsum": lambda t, o: chunk_global_cumsum(t(1, 8, 1), offsets=o, **kw),
    }


@pytest.mark.parametrize("op", list(_calls()))
def test_offsets_on_another_device(op):
    offs = torch.tensor([0, 3, 8])
    with pytest.raises(ValueError, match="offsets on cpu, the operands on meta"):
        _calls()[op](lambda *s: torch.zeros(*s, dtype=torch.bfloat16, device="meta"), offs)


def test_host_addresses_do_not_cross_the_boundary():
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        be.ptr(torch.zeros(4))
    assert be.ptr(None) is None


@pytest.mark.gpu
@pytest.mark.parametrize("op", list(_calls()))
def test_offsets_left_on_the_host(device, op):
    with pytest.raises(ValueError, match="offsets on cpu, the operands on cuda"):
        _calls()[op](lambda *s: torch.zeros(*s, dtype=torch.bfloat16, device=device), torch.tensor([0, 3, 8]))
