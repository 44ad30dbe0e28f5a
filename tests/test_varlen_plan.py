"""The tables of packed batches: how long they live, and calls on several streams that share them."""
import gc
import weakref

import pytest
import torch

from fla_amd.utils import VarlenPlan


def test_a_plan_lives_as_long_as_its_offsets():
    """However many other batches pass meanwhile: a captured graph keeps addresses of its plan's tables, and what keeps them is the
    tensor of offsets it was captured with."""
    offs = torch.tensor([0, 5, 9])
    plan = VarlenPlan(offs, 64)
    others = [torch.tensor([0, n]) for n in range(1, 400)]
    for t in others:
        VarlenPlan(t, 64)
    assert VarlenPlan(offs, 64) is plan
    del t, others
    gc.collect()
    size = len(VarlenPlan._cache)
    key = (id(offs), 64)
    assert key in VarlenPlan._cache
    del offs
    gc.collect()
    assert key not in VarlenPlan._cache and len(VarlenPlan._cache) == size - 1


def test_a_captured_plan_outlives_a_change_of_its_offsets():
    """Replays go on reading its tables; plans that no capture has met go with the boundaries they were made from."""
    offs = torch.tensor([0, 5, 90])
    plans = []
    for captured in (False, True, False, True, False):
        offs[1] += 1
        plan = VarlenPlan(offs, 64)
        plan._captured = captured           # (what a call under capture sets)
        plans.append(weakref.ref(plan))
    del plan
    gc.collect()
    assert [p() is not None for p in plans] == [False, True, False, True, True]
    del offs
    gc.collect()
    assert not any(p() for p in plans)


def test_tables():
    offs = torch.tensor([2, 2, 70, 135], dtype=torch.int32)
    plan = VarlenPlan(offs, 64)
    assert (plan.N, plan.NT) == (3, 4) and plan.covers(2, 135) and not plan.covers(0, 135)
    assert plan.indices.tolist() == [[1, 0], [1, 1], [2, 0], [2, 1]] and plan.chunk_offsets.tolist() == [0, 0, 2, 4]
    assert plan.seq_order.tolist() == [1, 2, 0] and plan.offsets.tolist() == [2, 2, 70, 135]
    assert all(t.dtype == torch.int64 and t.is_contiguous() for t in (plan.indices, plan.chunk_offsets, plan.seq_order, plan.offsets))
    offs[1] = 3
    assert VarlenPlan(offs, 64).indices.tolist() == [[0, 0], [1, 0], [1, 1], [2, 0], [2, 1]]


def test_offsets_made_in_inference_mode():
    """They have no version that would show a change: their tables are made by every call."""
    with torch.inference_mode():
        offs = torch.tensor([0, 5, 9])
        assert VarlenPlan(offs, 64).offsets.tolist() == [0, 5, 9]
        offs[1] = 7
        assert VarlenPlan(offs, 64).offsets.tolist() == [0, 7, 9]
    assert (id(offs), 64) not in VarlenPlan._cache


@pytest.mark.gpu
def test_a_packed_call_in_inference_mode(device):
    from fla_amd.ops.gla import chunk_gla
    from fla_amd.ops.hgrn import chunk_hgrn
    x = torch.randn(1, 600, 64, device=device).bfloat16()
    q = x.view(1, 600, 1, 64)
    gk = torch.nn.functional.logsigmoid(q.float())
    bounds = [0, 300, 417, 600]
    outside = torch.tensor(bounds, device=device)
    want, ht = chunk_hgrn(x, x, output_final_state=True, cu_seqlens=outside, use_gate_in_kernel=True)
    o, _ = chunk_gla(q, q, q, gk, cu_seqlens=outside, head_first=False)
    with torch.inference_mode():
        inside = torch.tensor(bounds, device=device)
        for offs in (inside, outside):
            got, gt = chunk_hgrn(x, x, output_final_state=True, cu_seqlens=offs, use_gate_in_kernel=True)
            assert torch.equal(got, want) and torch.equal(gt, ht)
            assert torch.equal(chunk_gla(q, q, q, gk, cu_seqlens=offs, head_first=False)[0], o)


@pytest.mark.gpu
@pytest.mark.parametrize("index_type", [torch.int64, torch.int32])
def test_two_streams_share_the_tables(device, index_type):
    """The first call that meets the offsets queues behind a long product on its stream; a call on another stream, which waits for
    nothing, reads the same tables, and both go on while the offsets are dropped and others take their place."""
    from fla_amd.ops.gla import chunk_gla
    from fla_amd.ops.hgrn import chunk_hgrn
    gen = torch.Generator().manual_seed(0)
    T, ends = 2200, [0, 1, 701, 701, 2137, 2200]
    x, g = (torch.randn(1, T, 128, generator=gen).bfloat16().to(device).requires_grad_() for _ in range(2))
    q, k, v = (torch.randn(1, T, 1, 64, generator=gen).bfloat16().to(device) for _ in range(3))
    gk = torch.nn.functional.logsigmoid(torch.randn(1, T, 1, 64, generator=gen)).to(device)
    do = torch.randn(1, T, 128, generator=gen).bfloat16().to(device)
    a = torch.randn(8192, 8192, generator=gen).bfloat16().to(device)
    offsets = lambda: torch.tensor(ends, device=device, dtype=index_type)

    def step(offs):
        o, _ = chunk_hgrn(x, g, cu_seqlens=offs, use_gate_in_kernel=True)
        with torch.no_grad():
            p, _ = chunk_gla(q, k, v, gk, cu_seqlens=offs, head_first=False)
        return [o.detach(), p, *torch.autograd.grad(o, (x, g), do)]

    want = step(offsets())
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for turn in range(4):
        offs = offsets()
        torch.cuda.synchronize()
        print("two streams", index_type, turn, flush=True)
        got = []
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                if i == 0:
                    for _ in range(4):
                        torch.mm(a, a)
                got.append(step(offs))
        del offs
        others = [VarlenPlan(torch.tensor([0, n], device=device), 64).NT for n in (7, 70, 700)]
        torch.cuda.synchronize()
        assert others == [1, 2, 11]
        for out in got:
            assert all(torch.equal(p, q) for p, q in zip(want, out)), turn


@pytest.mark.gpu
def test_tables_first_met_under_capture_are_refused(device):
    """A capture takes no copy, and tables made by one would be empty for the eager calls that find them."""
    from fla_amd.ops.hgrn import chunk_hgrn
    x = torch.randn(1, 600, 64, device=device).bfloat16()
    offs = torch.tensor([0, 300, 600], device=device)
    torch.cuda.synchronize()
    graph, y = torch.cuda.CUDAGraph(), torch.zeros(8, device=device)
    with torch.no_grad():
        with torch.cuda.graph(graph):
            y += 1
            with pytest.raises(RuntimeError, match="ahead of the capture"):
                chunk_hgrn(x, x, cu_seqlens=offs, use_gate_in_kernel=True)
        want, _ = chunk_hgrn(x, x, cu_seqlens=offs, use_gate_in_kernel=True)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out, _ = chunk_hgrn(x, x, cu_seqlens=offs, use_gate_in_kernel=True)
        for _ in range(3):
            out.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want)


@pytest.mark.gpu
def test_replays_behind_a_change_of_the_offsets(device):
    """A graph goes on with the boundaries it was captured with; eager calls follow the offsets."""
    from fla_amd.ops.hgrn import chunk_hgrn
    x = torch.randn(1, 1500, 64, device=device).bfloat16()
    bounds = [[0, 300, 1500], [0, 900, 1500]]
    offs = torch.tensor(bounds[0], device=device)
    call = lambda o: chunk_hgrn(x, x, cu_seqlens=o, use_gate_in_kernel=True)[0]
    with torch.no_grad():
        want = [call(torch.tensor(b, device=device)) for b in bounds]
        assert not torch.equal(*want)
        call(offs)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call(offs)
        plans = [p for *_, p in VarlenPlan._cache.values() if p._captured]
        assert len(plans) == 1
        kept = weakref.ref(plans.pop())
        for turn in range(3):
            offs.copy_(torch.tensor(bounds[1 - turn % 2]))
            gc.collect()
            assert torch.equal(call(offs), want[1 - turn % 2]) and kept() is not None
            others = [VarlenPlan(torch.tensor([0, n], device=device), 64).NT for n in (7, 70, 700)]
            out.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert others == [1, 2, 11] and torch.equal(out, want[0])
