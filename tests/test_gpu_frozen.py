"""GPU: gradients of operands that are frozen are not formed, and those of the others are what they were.

What is formed shows in the number of allocations that a backward makes (each gradient and each workspace is one)."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _backward(outputs, leaves, grads):
    """The gradients, and the allocations of the call."""
    torch.autograd.grad(outputs, leaves, grads, retain_graph=True)
    torch.cuda.synchronize()
    before = torch.cuda.memory_stats()["allocation.all.allocated"]
    out = torch.autograd.grad(outputs, leaves, grads, retain_graph=True)
    return out, torch.cuda.memory_stats()["allocation.all.allocated"] - before


@pytest.mark.parametrize("rdtype", [None, torch.bfloat16, torch.float32])
def test_norm(device, rdtype):
    from fla_amd.modules import rms_norm
    gen = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=gen).to(device)
    x, w, b, dy = r(300, 256).bfloat16(), r(256), r(256), r(300, 256).bfloat16()
    res = None if rdtype is None else r(300, 256).to(rdtype)

    def run(*trained):
        leaves = {k: t.detach().requires_grad_(k in trained) for k, t in (("x", x), ("w", w), ("b", b), ("res", res)) if t is not None}
        y = rms_norm(leaves["x"], leaves["w"], leaves["b"], residual=leaves.get("res"))
        out, count = _backward(y, [leaves[k] for k in trained], dy)
        return dict(zip(trained, out)), count

    everything = ("x", "w", "b") + (() if res is None else ("res",))
    want, most = run(*everything)
    for frozen, fewer in ((("w",), 2), (("b",), 2), (("w", "b"), 4), (("res",), int(rdtype == torch.float32))):
        left = [k for k in everything if k not in frozen]
        got, count = run(*left)
        assert count == most - (fewer if set(frozen) <= set(everything) else 0), (frozen, count, most)
        assert all(torch.equal(got[k], want[k]) for k in left)
    # only the weight is trained
    got, _ = run("w")
    assert torch.equal(got["w"], want["w"])


@pytest.mark.parametrize("ends", [None, [0, 100, 300]])
def test_recurrence(device, ends):
    from fla_amd.ops.hgrn import chunk_hgrn
    gen = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=gen).to(device)
    N = 1 if ends is None else len(ends) - 1
    x, g, do = (r(1, 300, 64).bfloat16() for _ in range(3))
    lb, h0 = torch.rand(64, generator=gen).to(device) * 0.9, r(N, 64)
    offs = None if ends is None else torch.tensor(ends, device=device)

    def run(*trained):
        leaves = {k: t.detach().requires_grad_(k in trained) for k, t in (("x", x), ("g", g), ("lb", lb), ("h0", h0))}
        o, _ = chunk_hgrn(leaves["x"], leaves["g"], leaves["h0"], cu_seqlens=offs, use_gate_in_kernel=True, lower_bound=leaves["lb"])
        out, count = _backward(o, [leaves[k] for k in trained], do)
        return dict(zip(trained, out)), count

    want, most = run("x", "g", "lb", "h0")
    for frozen, fewer in ((("lb",), 2), (("h0",), 1), (("lb", "h0"), 3)):
        left = [k for k in want if k not in frozen]
        got, count = run(*left)
        assert count == most - fewer, (frozen, count, most)
        assert all(torch.equal(got[k], want[k]) for k in left)
    got, _ = run("lb")
    assert torch.equal(got["lb"], want["lb"])
