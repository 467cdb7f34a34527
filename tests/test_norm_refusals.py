"""What add_rmsnorm refuses, in Python and at the C entry, without a GPU."""
import ctypes as C

import pytest
import torch

from ingot_b200 import capi
from ingot_b200.norm import add_rmsnorm


def base(**k):
    a = {"x": torch.zeros(4, 64), "residual": torch.zeros(4, 64), "weight": torch.ones(64), "rows": 4, "out": torch.zeros(4, 64)}
    a.update(k)
    return a


def call(a):
    a = dict(a)
    return add_rmsnorm(a.pop("x"), a.pop("residual"), a.pop("weight"), a.pop("rows"), **a)


I8, S = torch.zeros(4, 64, dtype=torch.int8), torch.zeros(4)


@pytest.mark.parametrize("change,error", [
    ({"rows": 5}, ValueError), ({"rows": -1}, ValueError), ({"eps": -1.0}, ValueError), ({"eps": float("nan")}, ValueError),
    ({"out": None}, ValueError), ({"codes": I8}, ValueError), ({"scales": S}, ValueError), ({"x": None, "residual_out": torch.zeros(4, 64)}, ValueError),
    ({"rotate": 32}, ValueError), ({"rotate": 64, "codes": I8, "scales": S}, ValueError), ({"rotate": 256, "codes": I8, "scales": S}, ValueError),
    ({"x": torch.zeros(4, 32)}, ValueError), ({"x": torch.zeros(4, 64, dtype=torch.float64)}, TypeError), ({"out": torch.zeros(4, 64, dtype=torch.int32)}, TypeError),
    ({"out": torch.zeros(64, 4).t()}, ValueError), ({"weight": torch.ones(63)}, ValueError), ({"weight": torch.ones(128)[::2]}, ValueError),
    ({"residual_out": torch.zeros(4, 64, dtype=torch.bfloat16)}, TypeError), ({"codes": torch.zeros(4, 64, dtype=torch.uint8), "scales": S}, TypeError),
    ({"codes": I8, "scales": torch.zeros(3)}, ValueError), ({"codes": I8, "scales": torch.zeros(8)[::2]}, ValueError), ({"codes": I8[:3], "scales": S}, ValueError),
    ({"residual": torch.zeros(1, 4, 64)}, ValueError), ({"x": None, "residual": torch.zeros(4, 32769), "weight": None, "out": torch.zeros(4, 32769)}, ValueError),
])
def test_python_refuses(change, error):
    with pytest.raises(error):
        call(base(**change))


def test_there_is_no_cpu_path():
    with pytest.raises(ValueError, match="CUDA"):
        call(base())


P = 1 << 20  # an address that is never used: the checks come first


@pytest.mark.parametrize("change,status", [
    ({"rows": -1}, -1), ({"d": 0}, -1), ({"d": 32769, "ldx": 40000, "ldr": 40000, "ldro": 40000, "ldo": 40000}, -2), ({"eps": float("nan")}, -1), ({"r": 0}, -1), ({"rd": 3}, -1), ({"ldr": 63}, -1),
    ({"xd": -1}, -1), ({"ldx": 63}, -1), ({"ro": 0}, -1), ({"ldro": 63}, -1), ({"x": 0}, -1), ({"wd": 7}, -1), ({"out": 0}, -1), ({"od": 5}, -1), ({"ldo": 63}, -1),
    ({"codes": P}, -1), ({"scales": P}, -1), ({"codes": P, "scales": P, "ldc": 63}, -1), ({"rot": 64}, -2), ({"rot": 32}, -1),
    ({"rot": 256, "codes": P, "scales": P, "ldc": 64}, -1), ({}, -1),
])
def test_c_entry_refuses(change, status):
    a = {"x": P, "xd": 0, "ldx": 64, "r": P, "rd": 0, "ldr": 64, "ro": P, "ldro": 64, "w": P, "wd": 0, "off": 0.0, "eps": 1e-6, "rows": 4, "d": 64, "out": P, "od": 0,
         "ldo": 64, "codes": 0, "ldc": 0, "scales": 0, "rot": 0}
    a.update(change)
    assert capi.lib().iq_add_rmsnorm(None, None, *a.values()) == status  # (with nothing wrong: there is no context)


@pytest.mark.parametrize("change", [{"x": P + 2}, {"r": P + 1, "rd": 1}, {"ro": P + 2}, {"w": P + 2}, {"w": P + 1, "wd": 2}, {"out": P + 3}, {"codes": P, "scales": P + 2, "ldc": 64}])
def test_tensors_begin_on_an_element(change):
    a = {"x": P, "xd": 0, "ldx": 64, "r": P, "rd": 0, "ldr": 64, "ro": P, "ldro": 64, "w": P, "wd": 0, "off": 0.0, "eps": 1e-6, "rows": 4, "d": 64, "out": P, "od": 0,
         "ldo": 64, "codes": 0, "ldc": 0, "scales": 0, "rot": 0}
    a.update(change)
    call = lambda: capi.lib().iq_add_rmsnorm(None, None, *a.values())
    a["rot"] = 64  # (refused with another status, and later)
    assert call() == -1
    a.update({k: v & ~3 for k, v in a.items() if k in change and k not in ("rd", "wd", "ldc")})
    assert call() == -2


def test_no_rows_are_no_addresses():
    none = torch.zeros(0, 64)
    with pytest.raises(ValueError, match="CUDA"):  # (nothing but the device is wrong)
        add_rmsnorm(none, none, None, 0, out=none)
