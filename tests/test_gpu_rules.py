"""Rules on logits (iq_logits_rules through sampling.LogitRules): bit for bit against the same operations in fp32, and within their roundings of 64 bits."""
import numpy as np
import pytest
import torch

from ingot_b200 import capi
from ingot_b200.linear import VQMV
from ingot_b200.norm import add_rmsnorm
from ingot_b200.sampling import LogitRules, TopK64, argmax_rows
from oracle import qref
from gpu_util import affine_case

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def some(rng, rows, V, history=0, bias=0, masks=0, loose=0.5, spread=4.0, wild=False):
    """Rules of every kind, rows without some of them among them. wild: tokens, lengths and indexes outside their ranges too."""
    a = {}
    if history:
        a["tokens"] = (rng.random((rows, history)) ** spread * V).astype(np.int32)
        a["lens"] = rng.integers(0, history + 1, rows).astype(np.int32)
        a["prompt_lens"] = (a["lens"] * rng.random(rows)).astype(np.int32)
        a["repetition"] = np.where(rng.random(rows) < 0.7, rng.uniform(0.5, 2, rows), 1).astype(np.float32)
        a["presence"] = np.where(rng.random(rows) < 0.5, rng.normal(size=rows), 0).astype(np.float32)
        a["frequency"] = np.where(rng.random(rows) < 0.5, rng.normal(size=rows), 0).astype(np.float32)
        if wild:
            a["tokens"][rng.random((rows, history)) < 0.1] = rng.choice([-1, V, V + 7, 2**31 - 1, -2**31])
            a["lens"][::3] = rng.choice([-5, history + 9])
            a["prompt_lens"][::2] = rng.choice([-5, 2 * history])
    if bias:
        n = rng.integers(0, bias + 1, rows)
        a["bias_offsets"] = np.concatenate([[0], np.cumsum(n)]).astype(np.int32)
        a["bias_tokens"] = rng.integers(0, V, int(n.sum())).astype(np.int32)
        a["bias_values"] = (5 * rng.normal(size=int(n.sum()))).astype(np.float32)
        if wild and len(a["bias_tokens"]):
            a["bias_tokens"][::4] = rng.choice([-1, V, -2**31])
            a["bias_offsets"][-1] += 50
    if masks:
        a["mask"] = rng.integers(0, 2**32, (masks, (V + 31) // 32 + 1), dtype=np.uint64).astype(np.uint32)
        a["mask"][rng.random(a["mask"].shape) > loose] = 0
        a["mask_rows"] = rng.integers(-1, masks, rows).astype(np.int32)
        if wild:
            a["mask_rows"][::2] = rng.choice([masks, 1000000, -2**31])
    return a


def device(a):
    return {k: torch.from_numpy(v.view(np.int32) if v.dtype == np.uint32 else v).cuda() for k, v in a.items()}


def check(rng, rows, V, a, dtype=F32, pad=0, in_place=False, x=None):
    x = torch.from_numpy(3 * rng.normal(size=(rows, V)).astype(np.float32)).to(dtype) if x is None else x
    wide = torch.full((rows + 1, V + pad), float("nan")).to(dtype)
    wide[:rows, :V] = x
    xd = wide.cuda()
    out = xd if in_place else torch.full((rows + 1, V + pad), 7.0, device="cuda")
    beside = out.cpu().clone()
    rules = LogitRules(rows, V, **device(a))
    got = rules.encode(xd[:, :V], rows, out=out[:, :V])[:rows].cpu().numpy()
    full = out.cpu()
    same = lambda p, q: torch.equal(torch.nan_to_num(p, 99), torch.nan_to_num(q, 99))
    assert same(full[rows:], beside[rows:]) and same(full[:, V:], beside[:, V:])
    want = qref.logit_rules(x.float().numpy(), np.float32, **a)
    assert np.array_equal(got, want, equal_nan=True)
    # in 64 bits: a rounding per operation, each relative to no more than the sum of all magnitudes
    ref = qref.logit_rules(x.double().numpy(), np.float64, **a)
    size = np.abs(x.double().numpy()) * 2 + 1
    ops = 5
    if "tokens" in a:
        size = size + np.abs(a["frequency"][:, None]) * a["tokens"].shape[1] + np.abs(a["presence"][:, None])
    if "bias_values" in a and len(a["bias_values"]):
        size, ops = size + np.abs(a["bias_values"]).sum(), ops + len(a["bias_values"])
    fine = np.isfinite(ref)
    assert np.array_equal(fine, np.isfinite(got)) and (np.abs(got[fine] - ref[fine]) <= ops * 2.0**-24 * size[fine]).all()


@pytest.mark.parametrize("V", [1, 2, 31, 33, 127, 1000, 1024, 1025, 4096, 32768, 50257, 128000, 262144])
@pytest.mark.parametrize("rows", [1, 3])
def test_vocabularies(cuda_device, V, rows):
    rng = np.random.default_rng(V + rows)
    check(rng, rows, V, some(rng, rows, V, history=300, bias=20, masks=2))


@pytest.mark.parametrize("what", [{"history": 50}, {"bias": 9}, {"masks": 3}, {"bias": 9, "masks": 1}, {"history": 1, "masks": 1}, {"history": 4000, "bias": 64}, {}])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("V,pad", [(5000, 0), (5001, 3)])
def test_rules_alone_and_together(cuda_device, what, dtype, V, pad):
    rng = np.random.default_rng(V + len(what))
    check(rng, 5, V, some(rng, 5, V, **what), dtype, pad)


@pytest.mark.parametrize("history,spread", [(1, 1), (513, 1), (4097, 6), (20000, 3), (131072, 2)])
def test_histories(cuda_device, history, spread):
    rng = np.random.default_rng(history)
    a = some(rng, 3, 32000, history=history, spread=spread)
    a["lens"][:] = [history, 0, history - 1]
    a["prompt_lens"][:] = [0, 0, history - 1]
    a["repetition"][:], a["presence"][:], a["frequency"][:] = 1.3, 0.4, 0.01
    check(rng, 3, 32000, a)


def test_one_token_many_times(cuda_device):
    rng = np.random.default_rng(1)
    a = some(rng, 2, 1000, history=70000)
    a["tokens"][0], a["tokens"][1] = 999, 0
    a["lens"][:], a["prompt_lens"][:] = 70000, [0, 35000]
    a["repetition"][:], a["presence"][:], a["frequency"][:] = 1.1, 0.5, 1e-3
    check(rng, 2, 1000, a)


@pytest.mark.parametrize("V", [1000, 1001, 2047, 40000, 40003])
def test_what_lies_outside_is_passed_over(cuda_device, V):
    rng = np.random.default_rng(V)
    for _ in range(4):
        check(rng, 6, V, some(rng, 6, V, history=400, bias=30, masks=3, wild=True))


@pytest.mark.parametrize("V,bias", [(64, 40), (300, 3000), (20000, 9000), (2000, 1100)])
def test_biases_of_the_same_token_add_in_their_order(cuda_device, V, bias):
    """Beyond a list's room too."""
    rng = np.random.default_rng(V)
    a = some(rng, 2, V, bias=bias, masks=1, loose=0.9)
    a["bias_offsets"][:] = [0, bias // 3, bias]
    a["bias_tokens"] = rng.integers(0, V, bias).astype(np.int32)
    a["bias_values"] = (rng.normal(size=bias) * 10.0 ** rng.integers(-3, 4, bias)).astype(np.float32)
    check(rng, 2, V, a)


def test_infinities_nan_and_empty_masks(cuda_device):
    rng = np.random.default_rng(2)
    rows, V = 4, 3000
    a = some(rng, rows, V, history=200, bias=10, masks=2)
    a["mask"][1] = 0
    a["mask_rows"][:] = [0, 1, -1, 0]
    a["bias_values"][::2] = -np.inf
    a["bias_values"][1::4] = np.inf
    x = torch.from_numpy(rng.normal(size=(rows, V)).astype(np.float32))
    for value in (float("nan"), float("inf"), -float("inf"), torch.finfo(F32).max, torch.finfo(F32).min, 0.0, -0.0, 1e-45):
        x[torch.from_numpy(rng.random((rows, V)) < 0.02)] = value
    wide = torch.full((rows, V), 0.0)
    want = qref.logit_rules(x.numpy(), np.float32, **a)
    got = LogitRules(rows, V, **device(a)).encode(x.cuda(), rows, out=wide.cuda()).cpu().numpy()
    assert np.array_equal(got, want, equal_nan=True) and np.isneginf(got[1]).all()
    assert (argmax_rows(torch.from_numpy(got).cuda(), rows).cpu().numpy()[1]) == 0
    idx, val, z = TopK64(rows, V, torch.device("cuda", 0)).encode(torch.from_numpy(got).cuda(), rows, [1.0])
    assert (idx[1] == -1).all() and (val[1] == torch.finfo(F32).min).all()


@pytest.mark.parametrize("V", [2045, 2046, 2047, 2048, 20477, 20478, 20480, 20481, 40957])
def test_the_ends_of_the_blocks_parts(cuda_device, V):
    """Rows that begin anywhere within a group of four, vocabularies next to whole parts."""
    rng = np.random.default_rng(V)
    for rows, pad in ((4, 0), (900, 1)):
        check(rng, rows, V, some(rng, rows, V, history=60, bias=8, masks=3), pad=pad)


def test_results_that_begin_elsewhere(cuda_device):
    """x and out at different places within a group of four: one logit at a time."""
    rng = np.random.default_rng(11)
    rows, V = 3, 4999
    a = some(rng, rows, V, history=100, bias=20, masks=2)
    x = torch.from_numpy(rng.normal(size=(rows, V)).astype(np.float32)).cuda()
    out = torch.full((rows * V + 9,), 7.0, device="cuda")
    for at in (0, 1, 2, 3):
        got = LogitRules(rows, V, **device(a)).encode(x, rows, out=out[at:at + rows * V].view(rows, V))
        assert np.array_equal(got.cpu().numpy(), qref.logit_rules(x.cpu().numpy(), np.float32, **a))


@pytest.mark.parametrize("V,pad", [(9000, 0), (9001, 0), (9000, 6)])
def test_in_place(cuda_device, V, pad):
    rng = np.random.default_rng(V + pad)
    check(rng, 3, V, some(rng, 3, V, history=500, bias=40, masks=2), pad=pad, in_place=True)


@pytest.mark.parametrize("rows,V", [(200, 2000), (33, 151665), (1000, 300)])
def test_many_rows(cuda_device, rows, V):
    rng = np.random.default_rng(rows)
    check(rng, rows, V, some(rng, rows, V, history=600, bias=12, masks=4), BF16)


def test_rows_of_fewer_than_the_rules(cuda_device):
    rng = np.random.default_rng(5)
    a = some(rng, 6, 700, history=90, bias=5, masks=2)
    rules = LogitRules(6, 700, **device(a))
    x = torch.from_numpy(rng.normal(size=(6, 700)).astype(np.float32)).cuda()
    whole = rules.encode(x, 6)
    out = torch.full_like(x, 3)
    rules.encode(x, 2, out=out)
    assert torch.equal(out[:2], whole[:2]) and (out[2:] == 3).all()
    rules.encode(x, 0, out=out)
    assert torch.equal(out[:2], whole[:2])
    assert torch.equal(LogitRules(6, 700).encode(x, 6), x)  # no rule


def test_what_the_tensors_hold_changes_between_replays(cuda_device):
    rng = np.random.default_rng(6)
    rows, V = 3, 2500
    a = some(rng, rows, V, history=64, bias=6, masks=2)
    d = device(a)
    rules = LogitRules(rows, V, **d)
    x = torch.from_numpy(rng.normal(size=(rows, V)).astype(np.float32)).cuda()
    out = torch.empty_like(x)
    rules.encode(x, rows, out=out)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        rules.encode(x, rows, out=out)
    for step in range(3):
        a["lens"] = np.minimum(a["lens"] + 1, 64).astype(np.int32)
        a["frequency"] = rng.normal(size=rows).astype(np.float32)
        a["mask_rows"] = rng.integers(-1, 2, rows).astype(np.int32)
        for k in ("lens", "frequency", "mask_rows"):
            d[k].copy_(torch.from_numpy(a[k]))
        g.replay()
        assert np.array_equal(out.cpu().numpy(), qref.logit_rules(x.cpu().numpy(), np.float32, **a))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    want = out.clone()
    out.zero_()
    torch.cuda.synchronize()
    rules.encode(x, rows, out=out, stream=side)
    side.synchronize()
    assert torch.equal(out, want)


def test_the_end_of_a_decode_step(cuda_device):
    """Residual and last norm, lm_head, rules, then the candidates and arg-max that the sampler takes."""
    rng = np.random.default_rng(7)
    rows, D, V = 5, 2048, 8192
    m, _ = affine_case(rng, V, D, 4, cuda_device)
    x, r, w = (torch.from_numpy(rng.normal(size=s).astype(np.float32)) for s in ((rows, D), (rows, D), (D,)))
    h, logits = torch.empty(rows, D, dtype=BF16, device="cuda"), torch.empty(rows, V, device="cuda")
    a = some(rng, rows, V, history=128, bias=16, masks=2, loose=0.8)
    rules, top = LogitRules(rows, V, **device(a)), TopK64(rows, V, torch.device("cuda", 0))
    rd = r.cuda()
    add_rmsnorm(x.to(BF16).cuda(), rd, w.cuda(), rows, out=h)
    VQMV.encode(h, m, logits, rows)
    raw = logits.clone()
    rules.encode(logits, rows, out=logits)
    idx, val, z = top.encode(logits, rows, [0.7])
    best = argmax_rows(logits, rows)
    assert capi.context(0).device_status() == 0
    want = qref.logit_rules(raw.cpu().numpy(), np.float32, **a)
    assert np.array_equal(logits.cpu().numpy(), want)
    for t in range(rows):
        order = np.lexsort((np.arange(V), -want[t]))[:64]
        order = order[np.isfinite(want[t][order])]
        assert np.array_equal(idx[t, :len(order)].cpu().numpy(), order) and best[t].item() == order[0]
    ref = qref.add_rmsnorm((x.to(BF16).float() + r).numpy(), w.numpy(), 1e-6)[0]
    assert np.abs(h.double().cpu().numpy() - ref).max() <= np.abs(ref).max() * (2.0**-8 + 2.0**-18)


def test_tensors_of_no_rows(cuda_device):
    assert LogitRules(2, 100).encode(torch.empty(0, 100, device="cuda"), 0).shape == (0, 100)


def test_two_streams_at_once(cuda_device):
    rng = np.random.default_rng(21)
    rows, V = 5, 30001
    rules = LogitRules(rows, V, **device(some(rng, rows, V, history=3000, bias=40, masks=3)))
    x = torch.from_numpy(rng.normal(size=(rows, V)).astype(np.float32)).cuda()
    want = rules.encode(x, rows)
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream(), torch.cuda.Stream()], [torch.empty_like(x) for _ in range(2)]
    for _ in range(10):
        for s, o in zip(streams, outs):
            rules.encode(x, rows, out=o, stream=s)
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("rows,V,pad,history", [(160, 2000, 0, 300), (160, 2001, 2, 300), (150, 300, 0, 33000), (149, 301, 1, 33000)])
def test_more_rows_than_multiprocessors(cuda_device, rows, V, pad, history, dtype):
    """Several blocks per multiprocessor, with counters of both widths."""
    rng = np.random.default_rng(rows + V)
    check(rng, rows, V, some(rng, rows, V, history=history, bias=5, masks=3, wild=True), dtype=dtype, pad=pad)


@pytest.mark.parametrize("rows,V", [(1, 1), (1, 1023), (1, 1025), (2, 75777), (5, 250000), (5, 262144), (18, 262144), (37, 131072), (37, 131069), (38, 131072), (148, 32765), (148, 32766)])
def test_blocks_with_a_multiprocessor_to_themselves(cuda_device, rows, V):
    """Up to the largest part, and the first that is too large."""
    rng = np.random.default_rng(rows + V)
    check(rng, rows, V, some(rng, rows, V, history=700, bias=9, masks=2))


def test_what_tensors_on_the_gpu_are_refused_for(cuda_device):
    z = lambda *s, dtype=F32: torch.zeros(*s, dtype=dtype, device="cuda")
    rules = LogitRules(4, 100, repetition=z(4) + 1)
    rules.encode(z(4, 100), 4, out=z(4, 100))
    for change in ({"x": z(4, 99)}, {"x": z(3, 100)}, {"x": z(100)}, {"x": z(4, 100).int()}, {"x": z(100, 4).t()}, {"x": z(4, 100).cpu()}, {"rows": 5}, {"rows": -1}, {"out": z(4, 99)},
                   {"out": z(4, 100, dtype=BF16)}, {"out": z(4, 100).cpu()}, {"out": z(100, 4).t()}):
        a = {"x": z(4, 100), "rows": 4, "out": z(4, 100), **change}
        with pytest.raises((ValueError, TypeError)):
            rules.encode(a["x"], a["rows"], out=a["out"])


@pytest.mark.parametrize("rows,V,history,masks", [(20, 100003, 900, 3), (64, 100001, 0, 5), (18, 100000, 0, 0)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_large_parts_that_begin_anywhere(cuda_device, rows, V, history, masks, dtype):
    """Groups of eight logits: x and out at the same place within them, at the same within four, and elsewhere."""
    rng = np.random.default_rng(V + history)
    a = some(rng, rows, V, history=history, masks=masks, bias=7)
    rules = LogitRules(rows, V, **device(a))
    x = torch.from_numpy(3 * rng.normal(size=(rows, V)).astype(np.float32)).to(dtype)
    want = qref.logit_rules(x.float().numpy(), np.float32, **a)
    for at_x, at_out in ((0, 0), (5, 5), (4, 0), (3, 7), (1, 2)):
        xd = torch.zeros(rows * V + 8, dtype=dtype, device="cuda")[at_x:at_x + rows * V].view(rows, V)
        xd.copy_(x)
        flat = torch.full((rows * V + 16,), 7.0, device="cuda")
        rules.encode(xd, rows, out=flat[at_out:at_out + rows * V].view(rows, V))
        got = flat.cpu().numpy()
        assert np.array_equal(got[at_out:at_out + rows * V].reshape(rows, V), want, equal_nan=True)
        assert (got[:at_out] == 7).all() and (got[at_out + rows * V:] == 7).all()


@pytest.mark.parametrize("history", [0, 300])
@pytest.mark.parametrize("offsets", [[0, 2000, 2**31 - 1, 2**31 - 400, -2**31, 700, 2**31 - 1], [2**31 - 1] * 7, [2**31 - 512, 2**31 - 1024, 2600, 2601, 0, -1, 2600],
                                     [-2**31, -2**31, 2**31 - 1, -2**31, 2**31 - 1, 2600, 2599]])
def test_offsets_of_biases_anywhere(cuda_device, history, offsets):
    """Offsets far beyond the list, at either end of their type too, are cut there: the steps of a list's rounds do not pass 32 bits."""
    rng = np.random.default_rng(len(offsets) + history)
    for V in (900, 40001):
        a = some(rng, 6, V, history=history, masks=2)
        a["bias_tokens"], a["bias_values"] = rng.integers(0, V, 2600).astype(np.int32), rng.normal(size=2600).astype(np.float32)
        a["bias_offsets"] = np.array(offsets, dtype=np.int64).astype(np.int32)
        check(rng, 6, V, a)


@pytest.mark.parametrize("rows,V,history", [(160, 2001, 9000), (160, 2000, 9001), (40, 151665, 16384), (150, 40003, 33000), (149, 40000, 40001), (40, 262143, 33000)])
def test_long_histories_of_many_rows(cuda_device, rows, V, history):
    """Blocks of 512 threads that go through histories by 4096 tokens: two counters in a word and one, rows' parts beyond the first, prompts that end inside a step."""
    rng = np.random.default_rng(rows + V + history)
    a = some(rng, rows, V, history=history, bias=6, masks=2, spread=2.0)
    a["lens"][:] = rng.integers(history // 2, history + 1, rows)
    a["lens"][:5] = [history, 2048, 2049, 6144, 6143]
    a["prompt_lens"][:] = a["lens"] * rng.random(rows)
    a["prompt_lens"][:5] = [2048 + 4096, 2048, 2047, 2048, 3000]
    a["tokens"][5, :] = V - 1 - np.arange(history) % 7  # in a row's last part
    a["repetition"][:9], a["presence"][:9], a["frequency"][:9] = 1.25, 0.5, 0.01
    check(rng, rows, V, a)


@pytest.mark.parametrize("history", [32767, 32768])
def test_the_most_of_one_token(cuda_device, history):
    """Counts up to the last that two counters in a word hold, and the first that they do not: neither reaches its neighbour's, nor the prompt's bit."""
    rng = np.random.default_rng(history)
    rows, V = 160, 2000
    a = some(rng, rows, V, history=history)
    token = np.where(np.arange(rows) % 2, 1001, 1000)
    token[4:8], token[8:12] = [0, 1, V - 2, V - 1], [15, 16, 17, 18]
    a["tokens"][:] = token[:, None]
    a["lens"][:] = history
    a["prompt_lens"][:] = np.where(np.arange(rows) % 4 < 2, 0, rng.integers(0, history + 1, rows))
    a["tokens"][12:16, 7] = [1001, 1000, 999, 1002]  # a single neighbour
    a["repetition"][:], a["presence"][:], a["frequency"][:] = 1.3, 0.4, 1e-3
    check(rng, rows, V, a)
