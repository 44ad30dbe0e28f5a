"""GPU: a prompt and then single tokens through the recurrence of a layer whose state lies in a ``Cache``.  Every step is held to the formula
from the state that was ahead of it, and three steps and one call of three tokens to the formula from the state that both start from."""
import pytest
import torch

from oracle import hgrn as oracle

pytestmark = pytest.mark.gpu


def _within(name, out, ref, bound):
    got, half = out.detach().double().cpu(), torch.finfo(out.dtype).eps / 2
    over = ((got - ref).abs() / (half * (ref.abs() + bound) + bound + 2.0 ** -126)).max().item()
    print(f"{name}: {over:.3f} of the bound", flush=True)
    assert over <= 1.0, name


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("bounded", [False, True])
def test_prompt_and_steps(device, dtype, bounded):
    from fla_amd.models import Cache
    from fla_amd.ops.hgrn import chunk_hgrn, fused_recurrent_hgrn
    gen = torch.Generator().manual_seed(3)
    B, T, D, more = 2, 300, 136, 3
    # one projection's output, as the layer splits it
    both = torch.randn(B, T + more, 2 * D, generator=gen).to(dtype)
    lb = torch.rand(D, generator=gen) * 0.9 if bounded else None
    i, f = both.chunk(2, -1)
    gi, gf = both.to(device).chunk(2, -1)
    how = dict(use_gate_in_kernel=True, lower_bound=None if lb is None else lb.to(device))
    cache = Cache()
    with torch.no_grad():
        o, state = chunk_hgrn(gi[:, :T], gf[:, :T], output_final_state=True, **how)
        ho, hht, eo, eht = oracle.forward(i[:, :T], f[:, :T], lower_bound=lb, gates=True)
        _within("prompt", o, ho, eo)
        _within("its state", state, hht, eht)
        cache.update(recurrent_state=state, layer_idx=0, offset=T)
        held = cache[0]["recurrent_state"].data_ptr()
        start = cache[0]["recurrent_state"].clone()
        steps = []
        for t in range(T, T + more):
            now = slice(t, t + 1)
            before = cache[0]["recurrent_state"].cpu()
            o, state = fused_recurrent_hgrn(gi[:, now], gf[:, now], cache[0]["recurrent_state"], True, inplace_state=True, **how)
            cache.update(recurrent_state=state, layer_idx=0, offset=1)
            ho, hht, eo, eht = oracle.forward(i[:, now], f[:, now], before, lower_bound=lb, gates=True)
            _within(f"token {t}", o, ho, eo)
            _within(f"state behind token {t}", cache[0]["recurrent_state"], hht, eht)
            steps.append(o)
        assert cache[0]["recurrent_state"].data_ptr() == held and cache.get_seq_length() == T + more
        short, end = chunk_hgrn(gi[:, T:], gf[:, T:], start, True, **how)
    ho, hht, eo, eht = oracle.forward(i[:, T:], f[:, T:], start.cpu(), lower_bound=lb, gates=True)
    for name, a, b in (("steps", torch.cat(steps, 1), cache[0]["recurrent_state"]), ("one call", short, end)):
        _within(name, a, ho, eo)
        _within(f"{name}, state", b, hht, eht)
