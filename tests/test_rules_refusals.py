"""What LogitRules refuses, in Python and at the C entry, without a GPU."""
import ctypes as C

import pytest
import torch

from ingot_b200 import capi
from ingot_b200.sampling import LogitRules

I, F = (lambda *s: torch.zeros(*s, dtype=torch.int32)), (lambda *s: torch.zeros(*s))
HIST, BIAS = {"tokens": I(4, 10), "lens": I(4)}, {"bias_offsets": I(5), "bias_tokens": I(7), "bias_values": F(7)}


@pytest.mark.parametrize("a", [
    {"tokens": I(4, 10)}, {"lens": I(4)}, {"prompt_lens": I(4)}, {**HIST, "lens": I(3)}, {**HIST, "lens": F(4)}, {**HIST, "tokens": I(3, 10)}, {**HIST, "tokens": F(4, 10)},
    {**HIST, "tokens": I(10, 4).t()}, {**HIST, "prompt_lens": I(8)[::2]}, {"repetition": F(3)}, {"presence": I(4)}, {"frequency": F(8)[::2]}, {"bias_offsets": I(5)},
    {**BIAS, "bias_offsets": I(4)}, {**BIAS, "bias_values": F(6)}, {**BIAS, "bias_tokens": F(7)}, {**BIAS, "bias_tokens": I(14)[::2]}, {"mask_rows": I(4)}, {"mask": I(3, 4)}, {"mask": I(4, 3)},
    {"mask": F(4, 4)}, {"mask": I(0, 4), "mask_rows": I(4)}, {"mask": I(1, 4), "mask_rows": I(3)}, HIST])
def test_construction(a):
    with pytest.raises(ValueError):  # (the last: nothing wrong but the device)
        LogitRules(4, 100, **a)


def test_sizes():
    for rows, vocab in ((0, 10), (1, 0), (1, 262145)):
        with pytest.raises(ValueError):
            LogitRules(rows, vocab)


@pytest.mark.parametrize("change,error", [({"x": F(4, 99)}, ValueError), ({"x": F(3, 100)}, ValueError), ({"x": I(4, 100)}, TypeError), ({"rows": 5}, ValueError), ({"rows": -1}, ValueError),
                                          ({"out": F(4, 101)}, ValueError), ({"out": F(4, 100).half()}, TypeError), ({"out": F(100, 4).t()}, ValueError), ({"x": F(100)}, ValueError), ({}, ValueError)])
def test_calls(change, error):
    a = {"x": F(4, 100), "rows": 4, "out": None}
    a.update(change)
    with pytest.raises(error):
        LogitRules(4, 100).encode(a["x"], a["rows"], a["out"])
    with pytest.raises(TypeError):
        LogitRules(4, 100).__getstate__()


P = 1 << 20  # an address that is never used: the checks come first


@pytest.mark.parametrize("call,rules,status", [
    ({"x": 0}, {}, -1), ({"out": 0}, {}, -1), ({"xd": 3}, {}, -1), ({"rows": -1}, {}, -1), ({"vocab": 0}, {}, -1), ({"ldx": 99}, {}, -1), ({"ldo": 99}, {}, -1),
    ({"vocab": 262145, "ldx": 262145, "ldo": 262145}, {}, -2), ({}, {"tokens": P, "ld_tokens": 8, "max_tokens": 8}, -1), ({}, {"tokens": P, "lens": P, "ld_tokens": 8, "max_tokens": 9}, -1),
    ({}, {"tokens": P, "lens": P, "max_tokens": -1}, -1), ({}, {"bias_offsets": P, "biases": -1}, -1), ({}, {"bias_offsets": P, "biases": 2}, -1),
    ({}, {"mask": P, "masks": 4, "ld_mask": 3}, -1), ({}, {"mask": P, "masks": 0, "ld_mask": 4, "mask_rows": P}, -1), ({}, {"mask": P, "masks": 3, "ld_mask": 4}, -1), ({}, {}, -1)])
def test_c_entry(call, rules, status):
    a = {"x": P, "xd": 0, "ldx": 100, "out": P, "ldo": 100, "rows": 4, "vocab": 100}
    a.update(call)
    assert capi.lib().iq_logits_rules(None, None, *a.values(), C.byref(capi.LogitRules(**rules))) == status
    assert capi.lib().iq_logits_rules(None, None, *a.values(), None) == -1


def test_the_struct_is_the_headers():
    import os
    import re

    text = open(os.path.join(os.path.dirname(__file__), "..", "include", "ingot_qmm.h")).read()
    for name, struct in (("iq_logit_rules", capi.LogitRules), ("iq_qmm_i8_tiling", capi.QmmI8Tiling)):
        body = re.sub(r"/\*.*?\*/", "", text[text.index(f"typedef struct {name} {{"):text.index(f"}} {name};")], flags=re.S)
        assert re.findall(r"(\w+);", body) == [f[0] for f in struct._fields_]


@pytest.mark.parametrize("call,rules", [({"x": P + 2}, {}), ({"x": P + 1, "xd": 2}, {}), ({"out": P + 2}, {})] + [({}, {name: P + 1}) for name in (
    "tokens", "lens", "prompt_lens", "repetition", "presence", "frequency", "bias_offsets", "bias_tokens", "bias_values", "mask", "mask_rows")])
def test_tensors_begin_on_an_element(call, rules):
    a = {"x": P, "xd": 0, "ldx": 262145, "out": P, "ldo": 262145, "rows": 4, "vocab": 262145}  # (refused with another status, and later)
    given = lambda: capi.lib().iq_logits_rules(None, None, *a.values(), C.byref(capi.LogitRules(**rules)))
    a.update(call)
    assert given() == -1
    a.update({"x": P, "out": P})
    rules = {name: P for name in rules}
    assert given() == -2


def meta(*s, dtype=torch.int32):
    return torch.empty(*s, dtype=dtype, device="meta")


@pytest.mark.parametrize("a,what", [({"tokens": meta(4, 2**30 + 1), "lens": meta(4)}, "capacity"), ({"tokens": meta(4, 2**32 + 5), "lens": meta(4)}, "capacity"),
                                    ({"bias_offsets": meta(5), "bias_tokens": meta(2**31), "bias_values": meta(2**31, dtype=torch.float32)}, "bias_tokens has"),
                                    ({"mask": meta(2**32 + 1, 4), "mask_rows": meta(4)}, "mask has")])
def test_lists_beyond_32_bits(a, what):
    """Lengths go to the C entry as 32 bits, and the kernel's steps through a history stay within them."""
    with pytest.raises(ValueError, match=what):
        LogitRules(4, 100, **a)


@pytest.mark.parametrize("tokens,status", [(2**30, -1), (2**30 + 1, -2), (2**31 - 1, -2)])
def test_histories_beyond_the_largest(tokens, status):
    rules = capi.LogitRules(tokens=P, lens=P, ld_tokens=2**31, max_tokens=tokens)  # (without a context the largest is refused as well, for that)
    assert capi.lib().iq_logits_rules(None, None, P, 0, 100, P, 100, 4, 100, C.byref(rules)) == status
