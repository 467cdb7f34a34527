"""iq_add_rmsnorm through norm.add_rmsnorm: the sum and the codes bit for bit, the norm against 64 bits."""
import numpy as np
import pytest
import torch

from ingot_b200 import capi, norm
from ingot_b200.norm import add_rmsnorm
from oracle import qref

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16

# q's relative error: the fp32 sum of squares adds at most 32 fma per thread and ten levels of two trees (42 * 2^-24, halved by the root),
# division, addition of eps and rsqrt another four; with the weight's addition and two products 21 + 4 + 3 = 28
Q_TOL = 32 * 2.0**-24


def rows_of(gen, rows, d, pad, dtype, scale=1.0):
    """[rows + 1, d] inside wider rows, the rest filled with NaN: nothing of it may be read into a result, nor written."""
    t = torch.full((rows + 1, d + pad), float("nan"))
    t[:rows, :d] = scale * torch.randn(rows, d, generator=gen)
    return t.to(dtype)


def run(gen, rows, d, xt, rt, wt, ot, rotate, pad, offset=0.0, eps=1e-6, device="cuda", want_out=True, want_codes=True, spread=1.0):
    x = None if xt is None else rows_of(gen, rows, d, pad, xt)
    r = rows_of(gen, rows, d, pad, rt, spread)
    w = None if wt is None else (1 - offset + 0.3 * torch.randn(d, generator=gen)).to(wt)
    up = lambda t: None if t is None else t.to(device)
    xd, rd, wd = up(x), up(r), up(w)
    ro = None if x is None else torch.full_like(rd, 7)
    out = torch.full((rows + 1, d + pad), 7, dtype=ot, device=device) if want_out else None
    codes = torch.full((rows + 1, d + pad), 99, dtype=torch.int8, device=device) if want_codes else None
    scales = torch.full((rows + 1,), 7, dtype=F32, device=device) if want_codes else None
    cut = lambda t: None if t is None else t[:, :d]
    add_rmsnorm(cut(xd), cut(rd), wd, rows, eps=eps, weight_offset=offset, residual_out=cut(ro), out=cut(out), codes=cut(codes), scales=scales, rotate=rotate)
    torch.cuda.synchronize()
    for t, fill in ((ro, 7), (out, 7), (codes, 99)):  # what lies beside the rows and behind the last one stays
        if t is not None:
            t = t.float().cpu()
            assert (t[rows] == fill).all() and (t[:rows, d:] == fill).all()
    down = lambda t: None if t is None else t[:rows].cpu() if t.dim() == 1 else t[:rows, :d].cpu()
    return tuple(None if t is None else t[:rows, :d] for t in (x, r)) + (w, down(ro), down(out), down(codes), down(scales))


def check(got, offset, eps, rotate):
    x, r, w, ro, out, codes, scales = got
    total = r if x is None else (r.float() + x.float()).to(r.dtype)
    if x is not None:
        assert torch.equal(ro, total)
    kept = total.float().numpy()
    w32 = np.ones(kept.shape[1], np.float32) if w is None else w.float().numpy() + np.float32(offset)
    ref, q = qref.add_rmsnorm(kept, w32, eps)
    if out is not None:
        half = torch.finfo(out.dtype).eps / 2
        tiny = float(torch.finfo(out.dtype).tiny) * half * 2  # half a step of a subnormal
        assert (np.abs(out.double().numpy() - ref) <= np.abs(ref) * (Q_TOL + half * (1 + Q_TOL)) + tiny).all()
    if codes is not None:
        want, s = qref.norm_codes(kept, w32, max(rotate, 1))
        assert np.array_equal(codes.numpy(), want)
        assert np.allclose(scales.double().numpy(), s.astype(np.float64) * q[:, 0], rtol=Q_TOL, atol=0)


@pytest.mark.parametrize("rows,d,pad", [(1, 1, 0), (3, 7, 1), (1, 64, 0), (2, 256, 8), (5, 2880, 0), (4, 2880, 5), (1, 2048, 0), (37, 4096, 0), (3, 8191, 0),
                                        (2, 8192, 0), (2, 8200, 0), (2, 16384, 16), (2, 16385, 3), (2, 32768, 0), (1, 32767, 0)])
@pytest.mark.parametrize("xt,rt,wt,ot", [(BF16, F32, BF16, BF16), (F16, F16, F32, F32), (F32, BF16, None, F16), (None, F32, F16, F32)])
def test_sum_norm_and_codes(cuda_device, rows, d, pad, xt, rt, wt, ot):
    gen = torch.Generator().manual_seed(rows * 100003 + d + pad)
    check(run(gen, rows, d, xt, rt, wt, ot, 0, pad), 0.0, 1e-6, 0)


@pytest.mark.parametrize("rotate", [32, 256])
@pytest.mark.parametrize("rows,blocks,pad", [(1, 1, 0), (3, 7, 0), (2, 16, 3), (65, 8, 0), (2, 33, 0), (2, 72, 0), (1, 128, 1)])
def test_rotated_codes(cuda_device, rotate, rows, blocks, pad):
    gen = torch.Generator().manual_seed(rotate + rows * 31 + blocks)
    d = 256 * blocks if rotate == 256 else 256 * blocks - 32 * (blocks % 3)
    got = run(gen, rows, d, BF16, F32, BF16, F16, rotate, pad)
    check(got, 0.0, 1e-6, rotate)
    # and against the transform in 64 bits: half a step of the codes, and the butterflies' roundings
    x, r, w, ro, out, codes, scales = got
    v = ro.double().numpy() * w.double().numpy()
    u = (v.reshape(rows, -1, rotate) @ qref.hadamard(rotate)).reshape(rows, d)
    sums = np.repeat(np.abs(v).reshape(rows, -1, rotate).sum(-1), rotate, axis=1)
    s = qref.norm_codes(ro.float().numpy(), w.float().numpy(), rotate)[1].astype(np.float64)[:, None]
    assert (np.abs(codes.numpy() * s - u) <= s * (0.5 + 127 * 2.0**-22) + 10 * 2.0**-24 * sums).all()


def test_one_output_alone_and_the_weights_offset(cuda_device):
    gen = torch.Generator().manual_seed(3)
    check(run(gen, 9, 1408, BF16, BF16, BF16, BF16, 0, 0, offset=1.0, want_codes=False), 1.0, 1e-6, 0)
    check(run(gen, 9, 1408, BF16, BF16, BF16, BF16, 32, 0, offset=1.0, want_out=False), 1.0, 1e-6, 32)
    check(run(gen, 9, 1408, F16, F32, F32, F32, 0, 0, eps=0.5), 0.0, 0.5, 0)


@pytest.mark.parametrize("spread", [1e-3, 1e4])
def test_wide_ranges(cuda_device, spread):
    gen = torch.Generator().manual_seed(4)
    check(run(gen, 5, 768, F32, F32, F32, F32, 256, 0, spread=spread), 0.0, 1e-6, 256)


def test_codes_next_to_a_border(cuda_device):
    """Quotients at and beside halves: the codes are the division's, not those of a product with the reciprocal."""
    d = 4096
    s = np.float32(0.7) / np.float32(127)
    k = np.arange(d) % 253 - 126
    r = (np.float32(0.5) + np.float32(k)) * s
    r[1::3] = np.nextafter(r[1::3], np.float32(9))
    r[2::3] = np.nextafter(r[2::3], np.float32(-9))
    r[0] = 0.7
    t = torch.from_numpy(r)[None].cuda()
    codes, scales = torch.empty(1, d, dtype=torch.int8, device="cuda"), torch.empty(1, device="cuda")
    add_rmsnorm(None, t, None, 1, codes=codes, scales=scales)
    want, _ = qref.norm_codes(r[None], np.ones(d, np.float32), 1)
    assert np.array_equal(codes.cpu().numpy(), want)


def test_rows_of_zeros_infinities_and_nan(cuda_device):
    d = 512
    r = torch.randn(6, d, generator=torch.Generator().manual_seed(5))
    r[0] = 0
    r[1, 17] = float("inf")
    r[2, 300] = float("nan")
    r[3] *= 1e-42  # below the normal numbers
    x = torch.zeros(6, d)
    codes = torch.full((6, d), 99, dtype=torch.int8, device="cuda")
    scales, out, ro = torch.full((6,), 7.0, device="cuda"), torch.empty(6, d, device="cuda"), torch.empty(6, d, device="cuda")
    for rotate in (0, 32, 256):
        add_rmsnorm(x.cuda(), r.cuda(), None, 6, residual_out=ro, out=out, codes=codes, scales=scales, rotate=rotate)
        c, s, o = codes.cpu(), scales.cpu(), out.cpu()
        assert (c[:3] == 0).all() and s[0] == 0 and s[1].isnan() and s[2].isnan()
        assert (o[0] == 0).all() and o[1, 17].isnan() and (o[1, :17] == 0).all() and o[2].isnan().all()
        want, _ = qref.norm_codes(r[3:].numpy(), np.ones(d, np.float32), max(rotate, 1))
        assert np.array_equal(c[3:].numpy(), want)  # a poisoned row is alone


def test_in_place_and_the_rows_alone(cuda_device):
    """residual_out = residual (the default), out = x; a row's codes do not depend on the others."""
    gen = torch.Generator().manual_seed(6)
    rows, d = 33, 2880
    x, r, w = torch.randn(rows, d, generator=gen).to(BF16), torch.randn(rows, d, generator=gen), torch.randn(d, generator=gen)
    sep = {"residual_out": torch.empty(rows, d, device="cuda"), "out": torch.empty(rows, d, dtype=BF16, device="cuda")}
    codes, scales = torch.empty(rows, d, dtype=torch.int8, device="cuda"), torch.empty(rows, device="cuda")
    add_rmsnorm(x.cuda(), r.cuda(), w.cuda(), rows, codes=codes, scales=scales, **sep)
    xi, ri = x.cuda(), r.cuda()
    add_rmsnorm(xi, ri, w.cuda(), rows, out=xi)
    assert torch.equal(xi, sep["out"]) and torch.equal(ri, sep["residual_out"])
    for t in (0, 17, 32):
        c, s = torch.empty(1, d, dtype=torch.int8, device="cuda"), torch.empty(1, device="cuda")
        add_rmsnorm(None, sep["residual_out"][t:t + 1], w.cuda(), 1, codes=c, scales=s)
        assert torch.equal(c[0], codes[t]) and torch.equal(s[0], scales[t])


def test_the_w8a8_gemms_own_conversion(cuda_device):
    """On rows of unit weight the codes are those that the reference's activations' conversion gives to r' itself (the norm's factor is in the scale)."""
    rng = np.random.default_rng(8)
    r = rng.normal(size=(4, 2048)).astype(np.float32)
    codes, scales = torch.empty(4, 2048, dtype=torch.int8, device="cuda"), torch.empty(4, device="cuda")
    add_rmsnorm(None, torch.from_numpy(r).cuda(), None, 4, codes=codes, scales=scales, rotate=256)
    want, _ = qref.quant_i8_rows(qref.fwht(r.reshape(4, 8, 256)).reshape(4, 2048))
    assert np.array_equal(codes.cpu().numpy(), want)


def test_streams_graphs_and_no_rows(cuda_device):
    gen = torch.Generator().manual_seed(9)
    rows, d = 8, 4096
    x, r, w = (torch.randn(*s, generator=gen).cuda() for s in ((rows, d), (rows, d), (d,)))
    out, ro = torch.empty(rows, d, device="cuda"), torch.empty(rows, d, device="cuda")
    codes, scales = torch.zeros(rows, d, dtype=torch.int8, device="cuda"), torch.zeros(rows, device="cuda")
    call = lambda **k: add_rmsnorm(x, r, w, rows, residual_out=ro, out=out, codes=codes, scales=scales, rotate=256, **k)
    call()
    torch.cuda.synchronize()
    want = [t.clone() for t in (out, ro, codes, scales)]
    side = torch.cuda.Stream()
    for t in (out, ro, codes, scales):
        t.zero_()
    side.wait_stream(torch.cuda.current_stream())
    call(stream=side)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip((out, ro, codes, scales), want))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call()
    x2 = torch.randn(rows, d, generator=gen).cuda()
    old = x.clone()
    x.copy_(x2)
    g.replay()
    assert torch.equal(ro, r + x2)
    x.copy_(old)
    g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip((out, ro, codes, scales), want))
    out.fill_(5)
    add_rmsnorm(x, r, w, 0, residual_out=ro, out=out)
    assert (out == 5).all()


def test_long_strides_pass_32_bits(cuda_device):
    """Rows 1.2 G elements apart."""
    d, ld = 256, 1_200_000_000
    buf = torch.empty(2 * ld + d, dtype=F16, device="cuda")
    r = torch.as_strided(buf, (3, d), (ld, 1))
    gen = torch.Generator().manual_seed(10)
    v = torch.randn(3, d, generator=gen).to(F16)
    r.copy_(v)
    out = torch.empty(3, d, device="cuda")
    add_rmsnorm(None, r, None, 3, out=out)
    ref, _ = qref.add_rmsnorm(v.float().numpy(), np.ones(d, np.float32), 1e-6)
    assert (np.abs(out.double().cpu().numpy() - ref) <= np.abs(ref) * (Q_TOL + 2.0**-24)).all()


def test_many_rows(cuda_device):
    """More rows than a second grid dimension would take."""
    rows, d = 70001, 64
    r = torch.randn(rows, d, device="cuda")
    out = torch.empty_like(r)
    add_rmsnorm(None, r, None, rows, out=out)
    ref, _ = qref.add_rmsnorm(r.cpu().numpy(), np.ones(d, np.float32), 1e-6)
    assert (np.abs(out.double().cpu().numpy() - ref) <= np.abs(ref) * (Q_TOL + 2.0**-24)).all()
    assert capi.context(0).device_status() == 0


def test_refusals_reach_no_kernel(cuda_device):
    r = torch.randn(2, 64, device="cuda")
    with pytest.raises(ValueError, match="different devices"):
        add_rmsnorm(None, r, torch.ones(64), 2, out=r.clone())
    assert norm.MAX_WIDTH == 32768


@pytest.mark.parametrize("rows,d,xt,rt,wt,ot,rotate,out,codes", [
    (3300, 512, BF16, BF16, BF16, BF16, 256, True, True), (3300, 520, F16, F32, F32, F16, 0, False, True), (700, 2880, F16, F16, F16, F32, 32, True, True),
    (700, 4096, BF16, F32, BF16, BF16, 256, False, True), (650, 4096, BF16, BF16, BF16, BF16, 0, True, False), (500, 5128, None, F32, None, F16, 0, True, False),
    (460, 7680, F32, F16, BF16, F32, 256, True, True), (300, 8192, F32, F32, F32, F32, 32, False, True), (160, 16384, BF16, BF16, BF16, BF16, 256, False, True),
    (200, 14344, BF16, BF16, F32, BF16, 0, True, True), (200, 16384, BF16, BF16, BF16, BF16, 256, False, True), (160, 16384, F32, F32, F32, F32, 0, True, True)])
def test_the_kernel_of_many_rows(cuda_device, rows, d, xt, rt, wt, ot, rotate, out, codes):
    """More rows than blocks that run at once, up to more than two per block; the bits of a row are those of a call of its own."""
    gen = torch.Generator().manual_seed(rows + d)
    got = run(gen, rows, d, xt, rt, wt, ot, rotate, 32, want_out=out, want_codes=codes)
    check(got, 0.0, 1e-6, rotate)
    x, r, w, ro, o, c, s = got
    for t in (0, rows // 2, rows - 1):
        one = {}
        if out:
            one["out"] = torch.empty(1, d, dtype=ot, device="cuda")
        if codes:
            one.update(codes=torch.empty(1, d, dtype=torch.int8, device="cuda"), scales=torch.empty(1, device="cuda"), rotate=rotate)
        add_rmsnorm(None if x is None else x[t:t + 1].cuda(), r[t:t + 1].cuda(), None if w is None else w.cuda(), 1, **one)
        if out:
            assert torch.equal(one["out"][0].cpu(), o[t])
        if codes:
            assert torch.equal(one["codes"][0].cpu(), c[t]) and torch.equal(one["scales"].cpu()[0], s[t])


def test_many_rows_in_place_and_poisoned(cuda_device):
    rows, d = 1500, 4096
    gen = torch.Generator().manual_seed(12)
    x, r = torch.randn(rows, d, generator=gen).to(F16), torch.randn(rows, d, generator=gen).to(F16)
    r[700, 5], r[701] = float("nan"), 0
    x[701] = 0
    xd, rd = x.cuda(), r.cuda()
    codes, scales = torch.empty(rows, d, dtype=torch.int8, device="cuda"), torch.empty(rows, device="cuda")
    add_rmsnorm(xd, rd, None, rows, out=xd, codes=codes, scales=scales, rotate=256)
    total = (x.float() + r.float()).to(F16)
    assert torch.equal(torch.nan_to_num(rd.cpu(), 99), torch.nan_to_num(total, 99))
    assert (codes[700:702] == 0).all() and scales[700].isnan() and scales[701] == 0 and (xd[701] == 0).all() and xd[700].isnan().all()
    keep = [t for t in range(rows) if t not in (700, 701)]
    want, _ = qref.norm_codes(total[keep].float().numpy(), np.ones(d, np.float32), 256)
    assert np.array_equal(codes[keep].cpu().numpy(), want)


def test_a_weight_that_the_launch_before_wrote(cuda_device):
    """Launches start before their predecessors have ended; what those write is waited for, the weight too. Both kernels."""
    gen = torch.Generator().manual_seed(11)
    for rows, d in ((1, 2048), (1500, 2048)):
        r = torch.randn(rows, d, generator=gen).to(BF16).cuda()
        parts = [torch.randn(1, d, generator=gen).to(BF16).cuda() for _ in range(20)]
        w, out = torch.zeros(1, d, dtype=BF16, device="cuda"), torch.empty(20, rows, d, dtype=BF16, device="cuda")
        for i, part in enumerate(parts):
            add_rmsnorm(None, part, None, 1, out=w)
            add_rmsnorm(None, r, w[0], rows, out=out[i])
        for i, part in enumerate(parts):
            add_rmsnorm(None, part, None, 1, out=w)
            torch.cuda.synchronize()
            want = torch.empty_like(r)
            add_rmsnorm(None, r, w[0].clone(), rows, out=want)
            assert torch.equal(out[i], want)


def test_two_streams_at_once(cuda_device):
    gen = torch.Generator().manual_seed(12)
    r = torch.randn(700, 2880, generator=gen).to(BF16).cuda()
    def call(stream=None):
        out, codes, scales = torch.empty_like(r), torch.empty(700, 2880, dtype=torch.int8, device="cuda"), torch.empty(700, device="cuda")
        return (out, codes, scales), lambda: add_rmsnorm(None, r, None, 700, out=out, codes=codes, scales=scales, rotate=32, stream=stream)
    want, go = call()
    go()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    calls = [call(s) for s in streams]
    for _ in range(10):
        for _, go in calls:
            go()
    torch.cuda.synchronize()
    for got, _ in calls:
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_tensors_of_no_rows(cuda_device):
    none = torch.empty(0, 64, device="cuda")
    add_rmsnorm(none, none, None, 0, out=none, codes=torch.empty(0, 64, dtype=torch.int8, device="cuda"), scales=torch.empty(0, device="cuda"))


@pytest.mark.parametrize("rows,d,pad,rotate", [(3, 1024, 7, 256), (5, 1999, 0, 0), (2, 4103, 2, 0), (3, 6144, 7, 256), (160, 4103, 0, 0), (160, 6144, 7, 32), (2, 14337, 0, 0), (2, 14336, 7, 32), (1500, 480, 7, 32), (1700, 2047, 0, 0)])
@pytest.mark.parametrize("xt,rt,wt,ot", [(BF16, BF16, BF16, BF16), (F16, F32, F16, F16), (F32, F16, BF16, F32)])
def test_rows_that_are_not_aligned(cuda_device, rows, d, pad, rotate, xt, rt, wt, ot):
    """Blocks of every size, one and two 16-bit types."""
    gen = torch.Generator().manual_seed(rows + d + pad)
    check(run(gen, rows, d, xt, rt, wt, ot, rotate, pad), 0.0, 1e-6, rotate)


def test_what_tensors_on_the_gpu_are_refused_for(cuda_device):
    """The conditions are looked at in C; what fails one is an error of Python's and reaches no kernel. No reference is lost or kept."""
    import sys
    z = lambda *s, dtype=F32: torch.zeros(*s, dtype=dtype, device="cuda")
    base = lambda: {"x": z(4, 64), "residual": z(4, 64), "weight": z(64), "rows": 4, "out": z(4, 64), "codes": z(4, 64, dtype=torch.int8), "scales": z(4), "residual_out": z(4, 64)}
    call = lambda a: add_rmsnorm(a.pop("x"), a.pop("residual"), a.pop("weight"), a.pop("rows"), **a)
    call(base())
    for change in ({"rows": 5}, {"rows": -1}, {"eps": -1.0}, {"eps": float("nan")}, {"rotate": 16}, {"rotate": 256}, {"scales": None}, {"codes": None}, {"x": z(4, 63)}, {"x": z(3, 64)},
                   {"x": z(64)}, {"x": z(4, 64).double()}, {"x": z(4, 64).cpu()}, {"x": None}, {"residual": z(64)}, {"residual": z(4, 64).int()}, {"residual": z(64, 4).t()},
                   {"residual_out": z(4, 64, dtype=F16)}, {"residual_out": z(64, 4).t()}, {"weight": z(63)}, {"weight": z(128)[::2]}, {"weight": z(64).long()}, {"weight": z(64).cpu()},
                   {"out": z(4, 64).int()}, {"out": z(3, 64)}, {"codes": z(4, 64, dtype=torch.uint8)}, {"codes": z(4, 65, dtype=torch.int8)}, {"scales": z(3)}, {"scales": z(8)[::2]},
                   {"scales": z(4, dtype=F16)}, {"scales": z(4, 1)}):
        with pytest.raises((ValueError, TypeError)):
            call({**base(), **change})
    with pytest.raises(ValueError):
        add_rmsnorm(None, z(2, 32776), None, 2, out=z(2, 32776))
    before = [sys.getrefcount(t) for t in (F32, F16, BF16, torch.int8)]
    x, a = z(4, 64), base()
    kept = {k: sys.getrefcount(v) for k, v in a.items() if torch.is_tensor(v)}
    for _ in range(500):
        call(dict(a))
        with pytest.raises(ValueError):
            call({**a, "x": x[:, :63]})
    assert all(abs(sys.getrefcount(t) - b) < 50 for t, b in zip((F32, F16, BF16, torch.int8), before))
    assert all(sys.getrefcount(v) - kept[k] < 3 for k, v in a.items() if k in kept)
    # one row has no stride, and a scale of its own lies anywhere
    add_rmsnorm(None, z(1, 64), None, 1, codes=z(1, 64, dtype=torch.int8), scales=z(8)[::2])


@pytest.mark.parametrize("rows,d,pad", [(5, 512, 0), (5, 512, 3), (1000, 512, 0), (1000, 512, 3), (300, 4096, 0), (3, 18432, 0)])
@pytest.mark.parametrize("rotate", [0, 256])
@pytest.mark.parametrize("eps", [1e-6, 0.0])
def test_rows_whose_step_rounds_to_nothing(cuda_device, rows, d, pad, rotate, eps):
    """A largest value of up to 63 * 2^-149 has a step max / 127 of 0 in 32 bits: codes and scale are 0, not 127 and 0 * inf. One of 64 * 2^-149 has a step of 2^-149."""
    r = torch.zeros(rows, d)
    r[0, 5] = 1e-44  # 7 * 2^-149
    r[1 % rows, d - 1] = -63 * 2.0**-149
    r[2 % rows, 7] = 64 * 2.0**-149
    r[rows - 1, 0] = 2.0**-149
    wide = torch.zeros(rows, d + pad)
    wide[:, :d] = r
    codes = torch.full((rows, d), 99, dtype=torch.int8, device="cuda")
    scales = torch.full((rows,), 7.0, device="cuda")
    add_rmsnorm(None, wide.cuda()[:, :d], None, rows, eps=eps, codes=codes, scales=scales, rotate=rotate)
    want, s = qref.norm_codes(r.numpy(), np.ones(d, np.float32), max(rotate, 1))
    assert np.array_equal(codes.cpu().numpy(), want)
    got = scales.cpu().numpy()
    assert (got[s == 0] == 0).all() and (s[[0, 1]] == 0).all() and s[2] > 0 and (want[2] != 0).any()
