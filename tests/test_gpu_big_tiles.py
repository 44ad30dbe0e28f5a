"""GPU: the 256 x 256 tiles of the large products, each element against the formula in fp64 (the bounds of the smaller cases): workgroups that take several tiles, whose
waits count the stores of the tile before, half tiles, several slices of the contraction in both, ragged edges, results of an odd number of columns.  Which of
that a case goes through stands in tests/test_matrix_plan.py."""
import pytest
import torch

from oracle import gated_linear as oracle
from test_gpu_gated_linear import check, double, everything, inputs
from test_gpu_int8_linear import U, close, pre, rows

pytestmark = pytest.mark.gpu

BF, HF, FL = torch.bfloat16, torch.float16, torch.float32

GATED = [  # M, F, K, type, biases, activation
    (4360, 2200, 4400, BF, None, "silu"), (4360, 2200, 4400, HF, FL, "gelu"), (4357, 2197, 4393, HF, None, "silu"), (4357, 2197, 4393, BF, BF, "relu"),
    (5300, 2500, 5000, BF, BF, "gelu"), (5300, 2500, 5000, HF, None, None), (8200, 4400, 200, BF, None, "silu"), (8200, 4400, 200, HF, HF, "gelu"),
]
INTEGERS = [  # M, N, K, result, bias, residual, activation
    (4360, 4400, 528, BF, BF, None, "silu"), (4360, 4400, 528, HF, None, FL, None), (4357, 4397, 528, HF, FL, None, "gelu"), (4357, 4397, 528, BF, None, BF, "relu"),
    (5300, 5000, 400, BF, None, None, "silu"), (5300, 5000, 400, HF, HF, HF, None), (8200, 8200, 144, BF, None, None, None),
]
GATED_INTEGERS = [  # M, F, K, result, biases, activation
    (4360, 4400, 528, HF, HF, "gelu"), (4357, 4397, 528, BF, None, "silu"), (5300, 2500, 400, BF, FL, "relu"), (5300, 5000, 400, HF, None, None),
]


@pytest.mark.parametrize("M,F,K,dtype,btype,name", GATED)
def test_gated(device, M, F, K, dtype, btype, name):
    print(M, F, K, dtype, btype, name, flush=True)
    leaves, dh = inputs(device, M, F, K, dtype, btype, M + F)
    everything(leaves, dh, name)


@pytest.mark.parametrize("M,F,K,dtype,btype,name", GATED[:3])
def test_one_weight(device, M, F, K, dtype, btype, name):
    """Of one weight the launch has half of the tiles."""
    from fla_amd.modules import gated_linear
    leaves, dh = inputs(device, M, F, K, dtype, None, M)
    args = double(leaves)
    _, _, state = oracle.forward(*args, name=name)
    want = oracle.backward(*args[:3], state, dh.double(), name, torch.finfo(dtype).eps / 2)
    for i, k in ((1, "dwg"), (2, "dwu")):
        own = [None if t is None else t.clone().requires_grad_(i == j) for j, t in enumerate(leaves)]
        (got,) = torch.autograd.grad(gated_linear(*own, activation=name), own[i], dh)
        check(k, got, want[k], want["e_" + k])


@pytest.mark.parametrize("M,N,K,out,btype,rtype,name", INTEGERS)
def test_integers(device, M, N, K, out, btype, rtype, name):
    from fla_amd.modules import quant_linear
    print(M, N, K, out, btype, rtype, name, flush=True)
    gen = torch.Generator(device=device).manual_seed(M + N + K)
    x, w = rows(M, K, gen, device), rows(N, K, gen, device)
    r = lambda *s: torch.randn(*s, generator=gen, device=device)
    bias = None if btype is None else r(N).to(btype)
    res = None if rtype is None else r(M, N).to(rtype)
    y = quant_linear(x, w, bias, activation=name, residual=res, output_dtype=out)
    t, e = pre(x, w, bias)
    ref = oracle.act(name, t)[0]
    if name is not None:
        e = oracle.SLOPE * e + 3e-7 * t.abs() + (t.abs() + 8) * U * ref.abs()
    if res is not None:
        ref = ref + res.double()
        e = e + U * (ref.abs() + res.double().abs())
    close("y", y, ref, e)


@pytest.mark.parametrize("M,F,K,out,btype,name", GATED_INTEGERS)
def test_gated_integers(device, M, F, K, out, btype, name):
    from fla_amd.modules import quant_gated_linear
    print(M, F, K, out, btype, name, flush=True)
    gen = torch.Generator(device=device).manual_seed(M + F + K)
    x, wg, wu = rows(M, K, gen, device), rows(F, K, gen, device), rows(F, K, gen, device)
    # (scales as of weights of a layer, so that gates lie where the activation bends)
    x, wg, wu = ((q, s * (2 / (127 * 127 * 0.0101 ** 2 * K ** 0.5)) ** 0.5 * 1.2) for q, s in (x, wg, wu))
    bias = lambda: None if btype is None else torch.randn(F, generator=gen, device=device).to(btype)
    bg, bu = bias(), bias()
    h = quant_gated_linear(x, wg, wu, bg, bu, activation=name, output_dtype=out)
    (g, eg), (u, eu) = pre(x, wg, bg), pre(x, wu, bu)
    a = oracle.act(name, g)[0]
    ea = oracle.SLOPE * eg + 3e-7 * g.abs() + (g.abs() + 8) * U * a.abs()
    ref = a * u
    close("h", h, ref, u.abs() * ea + a.abs() * eu + ea * eu + 2 * U * ref.abs())


def test_repeated_calls_are_the_same_bits(device):
    """A wait that is too short would not show every time."""
    from fla_amd.modules import gated_linear
    (x, wg, wu, bg, bu), dh = inputs(device, 5300, 2500, 5000, BF, BF, 3)
    leaves = [t.requires_grad_() for t in (x, wg, wu, bg, bu)]
    step = lambda: (lambda h: [h.detach(), *torch.autograd.grad(h, leaves, dh)])(gated_linear(*leaves))
    first = step()
    for _ in range(20):
        assert all(torch.equal(a, b) for a, b in zip(step(), first))
