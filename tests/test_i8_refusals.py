"""What the W8A8 linear on packed rows refuses, in Python and at the C entry, without a GPU."""
import ctypes as C

import pytest
import torch

from ingot_b200 import capi
from ingot_b200.linear import I8Linear

W, S = torch.zeros(8, 64, dtype=torch.int8), torch.ones(8)


@pytest.mark.parametrize("w,s,rotate,error", [
    (W.float(), S, 0, TypeError), (W, S.half(), 0, TypeError), (W, S[:7], 0, ValueError), (W.t().contiguous().t(), S, 0, ValueError), (W[:, :24].contiguous(), S, 0, ValueError),
    (torch.zeros(1, 131072, dtype=torch.int8), S[:1], 0, ValueError), (W, S, 64, ValueError), (W, S, 256, ValueError), (W[0], S, 0, TypeError), (W, S, 32, ValueError)])
def test_weights(w, s, rotate, error):
    with pytest.raises(error):  # (the last: nothing wrong but the device)
        I8Linear(w, s, rotate)


@pytest.mark.parametrize("change,error", [
    ({"x": torch.zeros(4, 64)}, TypeError), ({"sx": torch.zeros(4, dtype=torch.float16)}, TypeError), ({"y": torch.zeros(4, 8, dtype=torch.int32)}, TypeError), ({"rows": 5}, ValueError),
    ({"rows": -1}, ValueError), ({"x": torch.zeros(4, 48, dtype=torch.int8)}, ValueError), ({"y": torch.zeros(4, 7)}, ValueError), ({"y": torch.zeros(8, 4).t()}, ValueError),
    ({"x": torch.zeros(4, 72, dtype=torch.int8)[:, :64]}, ValueError), ({"x": torch.zeros(4, 80, dtype=torch.int8)[:, 8:72]}, ValueError), ({"sx": torch.zeros(3)}, ValueError),
    ({"sx": torch.zeros(8)[::2]}, ValueError), ({"x": torch.zeros(64, dtype=torch.int8)}, ValueError), ({}, ValueError)])
def test_calls(change, error):
    m = object.__new__(I8Linear)
    m.w, m.scales, m.N, m.K, m.rotate = W, S, 8, 64, 0
    a = {"x": torch.zeros(4, 64, dtype=torch.int8), "sx": torch.zeros(4), "y": torch.zeros(4, 8), "rows": 4}
    a.update(change)
    if change:
        with pytest.raises(error):
            m._check(a["x"], a["sx"], a["y"], a["rows"])
    with pytest.raises((ValueError, TypeError)):
        m.encode(a["x"], a["sx"], a["y"], a["rows"])


P = 1 << 20  # an address that is never used: the checks come first


@pytest.mark.parametrize("change,status", [
    ({"x": 0}, -1), ({"sx": 0}, -1), ({"w": 0}, -1), ({"sw": 0}, -1), ({"y": 0}, -1), ({"yd": 3}, -1), ({"rows": -1}, -1), ({"n": 0}, -1), ({"k": 0}, -1), ({"k": 40}, -1),
    ({"k": 131072, "ldx": 131072}, -2), ({"ldx": 48}, -1), ({"ldx": 72}, -1), ({"ldy": 7}, -1), ({"x": P + 8}, -1), ({"w": P + 4}, -1), ({"y": P + 2}, -1), ({"flags": 2}, -1), ({}, -1)])
def test_c_entry(change, status):
    a = {"x": P, "ldx": 64, "sx": P, "w": P, "sw": P, "n": 8, "k": 64, "y": P, "yd": 0, "ldy": 8, "rows": 4, "flags": 0}
    a.update(change)
    assert capi.lib().iq_qmm_i8(None, None, *a.values()) == status


@pytest.mark.parametrize("change,rotate,status", [
    ({"w": 0}, 0, -1), ({"biases": 0}, 0, -1), ({"bits": 8}, 0, -2), ({"mode": 1}, 0, -2), ({"experts": 2}, 0, -2), ({"group": 128}, 0, -2), ({"k": 96}, 0, -1), ({"k": 65536}, 0, -1),
    ({"n": 0}, 0, -1), ({}, 64, -1), ({}, 256, -1), ({}, 32, -1)])
def test_pack_entry(change, rotate, status):
    a = {"w": P, "scales": P, "biases": P, "n": 8, "k": 128, "bits": 4, "group": 64, "mode": 0, "experts": 1}
    a.update(change)
    q = capi.QLinear(*a.values())
    assert capi.lib().iq_i8_pack(None, None, C.byref(q), rotate, P, P) == status


def test_the_plan():
    """Every tile is covered once, and each of the ways is taken by some shape that the GPU tests run."""
    seen = set()
    for rows in (1, 9, 17, 64, 128, 129, 160, 256, 300, 700, 2048, 4100):
        for n, k in ((1, 16), (256, 512), (300, 1040), (4096, 4096), (1030, 512), (4096, 14336), (256, 256), (1500, 1024), (704, 9216)):
            p = capi.qmm_i8_plan(rows, n, k)
            assert p.tiles == p.row_tiles * -(-n // (256 if p.pair else 128)) and 1 <= p.tall <= p.row_tiles
            whole = p.row_tiles * p.tile_rows - 32 * (p.row_tiles - p.tall)  # the rows of the tiles
            assert rows <= whole and (whole - rows < 32 if p.pair else p.tall == p.row_tiles and whole - rows < p.tile_rows)
            assert 1 <= p.parts <= (3 if p.pair else 8) and p.parts <= -(-k // 128)
            assert p.tile_rows % 32 == 0 and 32 <= p.tile_rows - 32 * (p.tall < p.row_tiles) and p.tile_rows <= 256 if p.pair else p.tile_rows in (16, 32, 64)
            seen.add((p.pair, p.tile_rows if p.pair else 0, p.parts))
    assert {c[2] for c in seen if not c[0]} == {1, 2, 4, 8} and {c[2] for c in seen if c[0]} == {1, 2, 3} and len({c[1] for c in seen if c[0]}) >= 4
    for bad in ((0, 1, 16), (1, 0, 16), (1, 1, 24), (1, 1, 131072)):
        with pytest.raises(capi.IngotError):
            capi.qmm_i8_plan(*bad)


@pytest.mark.parametrize("change", [{"sx": P + 2}, {"sw": P + 1}, {"y": P + 2}, {"y": P + 1, "yd": 2}])
def test_tensors_begin_on_an_element(change):
    a = {"x": P, "ldx": 64, "sx": P, "w": P, "sw": P, "n": 8, "k": 64, "y": P, "yd": 0, "ldy": 8, "rows": (1 << 30) + 1, "flags": 0}  # (too many rows: later, with another status)
    a.update(change)
    call = lambda: capi.lib().iq_qmm_i8(None, None, *a.values())
    assert call() == -1
    a.update({"sx": P, "sw": P, "y": P})
    assert call() == -2


@pytest.mark.parametrize("change,scales", [({"w": P + 2}, P), ({"scales": P + 1}, P), ({"biases": P + 1}, P), ({}, P + 2)])
def test_packed_tensors_begin_on_an_element(change, scales):
    a = {"w": P, "scales": P, "biases": P, "n": 8, "k": 128, "bits": 8, "group": 64, "mode": 0, "experts": 1}  # (8 bits: later, with another status)
    assert capi.lib().iq_i8_pack(None, None, C.byref(capi.QLinear(*a.values())), 0, P, P) == -2
    a.update(change)
    assert capi.lib().iq_i8_pack(None, None, C.byref(capi.QLinear(*a.values())), 0, P, scales) == -1


@pytest.mark.parametrize("rows,n,k", [((1 << 30) + 1, 8, 64), (8, (1 << 30) + 1, 64), (2**31 - 1, 2**31 - 1, 131056), (1 << 30, 1 << 30, 131056)])
def test_more_than_a_grid_holds(rows, n, k):
    assert capi.lib().iq_qmm_i8(None, None, P, k, P, P, P, n, k, P, 0, max(n, 1), rows, 0) in (-1, -2)
    if max(rows, n) > 1 << 30:
        with pytest.raises(capi.IngotError):
            capi.qmm_i8_plan(rows, n, k)
    else:
        assert capi.qmm_i8_plan(rows, n, k).tiles > 1 << 30  # (refused with a context)


@pytest.mark.parametrize("n", [2**30 + 1, 2**32 + 1])
def test_more_features_than_a_call_takes(n):
    """(they would go to the C entry as 32 bits)"""
    with pytest.raises(ValueError, match="features"):
        I8Linear(torch.empty(n, 16, dtype=torch.int8, device="meta"), torch.empty(n, device="meta"))


def test_a_matrix_with_a_rotation_of_its_own():
    from ingot_b200.linear import DenseQ

    m = object.__new__(DenseQ)
    m.had, m.w, m.s, m.b, m.N, m.K, m.bits, m.gs, m.mode, m.experts = torch.ones(1024), torch.zeros(8, 128, dtype=torch.int32), None, None, 8, 1024, 4, 64, "affine", 1
    with pytest.raises(ValueError, match="rotation of its own"):
        I8Linear.pack(m)
