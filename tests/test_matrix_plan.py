"""CPU: which tiles the rule gives the products of tests/test_gpu_big_tiles.py, so that another rule does not leave a kernel without its test."""
import ctypes

from test_gpu_big_tiles import GATED, GATED_INTEGERS, INTEGERS

FORWARD, FORWARD8, DX, DW, DW1, INT8, INT8_F32 = range(7)      # enum fla_product
CUS = 256


def plan(product, M, N, K):
    from fla_amd import _backend as be
    out = (ctypes.c_int * 5)()
    assert be.lib().fla_selftest_matrix_plan(product, M, N, K, out) == 0
    return dict(zip(("rows", "slices", "workgroups", "whole", "halves"), out))


def kinds(plans):
    """What the launches of 256 x 256 tiles among them go through."""
    found = set()
    for p in plans:
        if p["rows"] != 256:
            continue
        found.add("split" if p["slices"] > 1 else "halves" if p["halves"] else "turns" if p["whole"] > p["workgroups"] else "one")
        if p["whole"] > p["workgroups"]:
            found.add("turns")
        if p["halves"] and p["whole"] > p["workgroups"]:
            found.add("turns and halves")
    return found


def up8(K):
    return -(-K // 8) * 8


def test_gated_cases_cover_the_big_tiles():
    for dtype in {c[3] for c in GATED}:
        cases = [(M, F, up8(K)) for M, F, K, t, *_ in GATED if t == dtype]
        several = [c for c in cases if c[2] >= 256]       # four slices of K and more
        assert {"halves", "turns"} <= kinds(plan(FORWARD, *c) for c in several)
        assert {"halves", "turns", "split"} <= kinds(plan(DX, *c) for c in cases)
        assert {"halves", "turns", "split"} <= kinds(plan(DW, *c) for c in cases)
        assert any(plan(FORWARD, *c)["whole"] >= 3 * CUS for c in cases)
    assert all(plan(DW1, M, F, up8(K))["rows"] == 256 for M, F, K, *_ in GATED[:3])


def test_integer_cases_cover_the_big_tiles():
    for residual in (False, True):
        cases = [c[:3] for c in INTEGERS if (c[5] is not None) == residual]
        assert {"halves", "turns"} <= kinds(plan(INT8, *c) for c in cases)
    assert {"turns and halves", "turns"} <= kinds(plan(FORWARD8, *c[:3]) for c in GATED_INTEGERS)
    assert {"turns"} <= kinds(plan(INT8, *c[:3]) for c in INTEGERS if c[5] is None)
    assert plan(INT8_F32, 8191, 2048, 5632)["rows"] == 128


def test_edges_and_refusals():
    from fla_amd import _backend as be
    lib, out = be.lib(), (ctypes.c_int * 5)()
    assert plan(FORWARD, 64, 128, 64) == dict(rows=0, slices=0, workgroups=0, whole=0, halves=0)
    assert plan(FORWARD, 65, 128, 64)["rows"] > 0 and plan(DX, 1, 128, 64)["rows"] > 0
    assert plan(FORWARD, 65, 128, 8192)["slices"] == lib.fla_gated_linear_splits(65, 128, 8192, 2) > 1
    assert lib.fla_selftest_matrix_plan(7, 1, 1, 1, out) == -1 and lib.fla_selftest_matrix_plan(0, 0, 1, 1, out) == -1
    assert lib.fla_selftest_matrix_plan(0, 1, 1, 1, None) == -1 and lib.fla_selftest_matrix_plan(0, 1, (1 << 22) + 1, 1, out) == -2
