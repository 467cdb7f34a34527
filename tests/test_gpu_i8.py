"""W8A8 linears on packed int8 rows (iq_qmm_i8 through linear.I8Linear): bit for bit, since the sums are exact integers and what follows is
a fixed order of fp32 operations. And the packing of 4-bit matrices."""
import ctypes as C

import numpy as np
import pytest
import torch

from ingot_b200 import capi
from ingot_b200.linear import VQMV, I8Linear
from ingot_b200.norm import add_rmsnorm
from oracle import qref
from gpu_util import affine_case, deq

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def codes(gen, rows, k, low=-127):
    return torch.randint(low, 128, (rows, k), generator=gen, dtype=torch.int8)


def reference(x, sx, w, sw, base=None):
    """fp32(fp32(sum) * sx) * sw (+ base), the sums in 64 bits"""
    s = torch.from_numpy(x.numpy().astype(np.float64) @ w.numpy().astype(np.float64).T)  # exact: below 2^53
    y = s.to(F32) * sx[:, None] * sw[None, :]
    return y if base is None else y + base.float()


def run(gen, rows, n, k, dtype=F32, accumulate=False, pad=0, low=-127, x=None, w=None):
    x = codes(gen, rows, k, low) if x is None else x
    w = codes(gen, n, k, low) if w is None else w
    sx, sw = torch.rand(rows, generator=gen) + 0.01, torch.rand(n, generator=gen) * 1e-3 + 1e-5
    wide = torch.full((rows + 1, k + 16 * pad), 55, dtype=torch.int8, device="cuda")  # (what lies beside the rows is not read)
    wide[:rows, :k] = x.cuda()
    base = torch.randn(rows + 2, n + pad, generator=gen).to(dtype)
    y = base.cuda()
    m = I8Linear(w.cuda(), sw.cuda())
    m.encode(wide[:, :k], sx.cuda(), y[:, :n], rows, accumulate=accumulate)
    assert capi.context(0).device_status() == 0
    got = y.cpu()
    want = reference(x, sx, w, sw, base[:rows, :n] if accumulate else None).to(dtype)
    assert torch.equal(got[:rows, :n], want)
    assert torch.equal(got[rows:], base[rows:]) and torch.equal(got[:, n:], base[:, n:])


@pytest.mark.parametrize("rows", [1, 2, 15, 16, 17, 31, 33, 48, 64, 65, 100, 128, 129, 200, 256, 257, 300, 513])
@pytest.mark.parametrize("n,k", [(256, 512), (300, 1040), (129, 4096)])
def test_rows(cuda_device, rows, n, k):
    run(torch.Generator().manual_seed(rows * 7 + n), rows, n, k)


@pytest.mark.parametrize("n,k", [(1, 16), (1, 4096), (3, 48), (127, 128), (128, 144), (2880, 2880), (4097, 640), (1000, 8208), (512, 14336), (9472, 256), (37888, 128)])
@pytest.mark.parametrize("rows", [1, 9, 70])
def test_features_and_inputs(cuda_device, rows, n, k):
    run(torch.Generator().manual_seed(rows + n + k), rows, n, k)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("rows,n,k,pad", [(1, 384, 2048, 0), (5, 130, 2048, 3), (40, 257, 512, 1), (300, 200, 384, 5), (700, 1030, 512, 2)])
def test_types_accumulation_and_strides(cuda_device, dtype, accumulate, rows, n, k, pad):
    run(torch.Generator().manual_seed(rows + n), rows, n, k, dtype, accumulate, pad)


@pytest.mark.parametrize("rows,n,k", [(1100, 1500, 1024), (2048, 4096, 528), (1030, 300, 2064), (4100, 256, 256), (600, 9000, 144)])
def test_many_tiles(cuda_device, rows, n, k):
    run(torch.Generator().manual_seed(rows), rows, n, k, BF16)


@pytest.mark.parametrize("rows,n,k,parts,height,tall", [
    (129, 4730, 1040, 1, 64, 2), (1174, 1280, 1040, 1, 96, 9), (300, 4730, 2064, 1, 128, 1), (600, 4096, 528, 1, 160, 3), (1954, 2560, 384, 1, 160, 6), (1902, 9472, 256, 1, 160, 12),
    (173, 18944, 528, 1, 192, 1), (999, 6144, 528, 1, 192, 2), (600, 4730, 1040, 1, 224, 1), (2160, 9472, 384, 1, 224, 8), (700, 6144, 1040, 1, 256, 1),
    (129, 256, 1040, 2, 64, 2), (173, 256, 1040, 2, 64, 3), (200, 2049, 1040, 2, 96, 1), (300, 2049, 2064, 2, 128, 1), (999, 1280, 4096, 2, 192, 2), (700, 2049, 8208, 2, 256, 1),
    (129, 256, 2064, 3, 64, 2), (470, 640, 2064, 3, 96, 1), (246, 2049, 8208, 3, 128, 2), (1500, 300, 8208, 3, 160, 3), (2048, 300, 8208, 3, 192, 9), (470, 2049, 14336, 3, 256, 1)])
@pytest.mark.parametrize("dtype,accumulate", [(F32, True), (F16, False)])
def test_pairs(cuda_device, rows, n, k, parts, height, tall, dtype, accumulate):
    """Pairs of CTAs on tiles of every height, of one and of two heights, the last of them short, more than one tile per pair; two and three pairs per tile."""
    plan = capi.qmm_i8_plan(rows, n, k)
    assert plan.pair == 1 and (plan.parts, plan.tile_rows, plan.tall) == (parts, height, tall)
    run(torch.Generator().manual_seed(rows), rows, n, k, dtype, accumulate, 1)
    run(torch.Generator().manual_seed(rows), rows, n, k, dtype, accumulate, 0)


def test_the_largest_sums(cuda_device):
    """Every code -128 at the most inputs: 131,056 * 2^14 is below 2^31."""
    k = I8Linear.MAX_K
    full = torch.full((2, k), -128, dtype=torch.int8)
    run(torch.Generator().manual_seed(1), 2, 2, k, x=full, w=full)
    run(torch.Generator().manual_seed(2), 3, 130, k, low=-128)


def test_a_row_does_not_depend_on_the_others(cuda_device):
    gen = torch.Generator().manual_seed(3)
    x, w = codes(gen, 600, 2048).cuda(), codes(gen, 1000, 2048).cuda()
    sx, sw = torch.rand(600, generator=gen).cuda(), torch.rand(1000, generator=gen).cuda()
    m = I8Linear(w, sw)
    y = torch.empty(600, 1000, device="cuda")
    m.encode(x, sx, y, 600)
    for lo, hi in ((0, 1), (17, 33), (100, 140), (500, 600), (0, 257)):
        part = torch.empty(hi - lo, 1000, device="cuda")
        m.encode(x[lo:hi], sx[lo:hi], part, hi - lo)
        assert torch.equal(part, y[lo:hi])


@pytest.mark.parametrize("rows,k", [(3, 1024), (400, 1024), (400, 2048)])
def test_streams_and_graphs(cuda_device, rows, k):
    gen = torch.Generator().manual_seed(4)
    n = 520
    x, w = codes(gen, rows, k).cuda(), codes(gen, n, k).cuda()
    sx, sw = torch.rand(rows, generator=gen).cuda(), torch.rand(n, generator=gen).cuda()
    m, y = I8Linear(w, sw), torch.zeros(rows, n, device="cuda")
    m.encode(x, sx, y, rows)
    want = y.clone()
    side = torch.cuda.Stream()
    y.zero_()
    side.wait_stream(torch.cuda.current_stream())
    m.encode(x, sx, y, rows, stream=side)
    side.synchronize()
    assert torch.equal(y, want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        m.encode(x, sx, y, rows)
        m.encode(x, sx, y, rows, accumulate=True)
    y.zero_()
    g.replay()
    x.neg_()
    torch.cuda.synchronize()
    assert torch.equal(y, want + want)
    g.replay()
    assert torch.equal(y, -want - want)
    y.fill_(5)
    m.encode(x, sx, y, 0)
    assert (y == 5).all()


@pytest.mark.parametrize("N,K,group,rotate", [(64, 1024, 64, 256), (100, 1024, 64, 32), (3, 64, 64, 0), (48, 2880, 64, 32), (130, 768, 32, 256), (16, 128, 32, 0), (3, 49152, 64, 256), (5, 16384, 32, 32)])
def test_packing(cuda_device, N, K, group, rotate):
    rng = np.random.default_rng(N + K)
    m, host = affine_case(rng, N, K, 4, cuda_device, group=group)
    wf = deq(host, 4, group=group)
    got = I8Linear.pack(m, rotate)
    n = max(rotate, 1)
    want, s = qref.quant_i8_rows(qref.fwht(wf.reshape(N, K // n, n)).reshape(N, K))
    assert np.array_equal(got.w.cpu().numpy(), want) and np.array_equal(got.scales.cpu().numpy(), s / np.float32(n)) and got.rotate == rotate


@pytest.mark.parametrize("rows,K,rotate", [(1, 2048, 256), (7, 2880, 32), (130, 1024, 256), (700, 2048, 256)])
def test_codes_into_linear(cuda_device, rows, K, rotate):
    """The step as it is used: residual, norm and codes, then the linear, against the exact norm and weights. Rounding to 127 steps of the largest of a row
    on both sides: each product's error is at most half a step of one side times the other's value, independent and of either sign; for rows of
    normal values (largest some 4 times the root mean square) that is 4 / 127 / sqrt(12) = 0.9 % per side, 1.3 % of the result's root mean square in all,
    and its largest of 10^5 values some 4.5 times that."""
    rng = np.random.default_rng(rows)
    N = 192
    m, host = affine_case(rng, N, K, 4, cuda_device)
    lin = I8Linear.pack(m)
    assert lin.rotate == rotate
    x, r = torch.from_numpy(rng.normal(size=(rows, K)).astype(np.float32)), torch.from_numpy(rng.normal(size=(rows, K)).astype(np.float32))
    g = torch.from_numpy((1 + 0.1 * rng.normal(size=K)).astype(np.float32))
    xq, sx = torch.empty(rows, K, dtype=torch.int8, device="cuda"), torch.empty(rows, device="cuda")
    y, ro = torch.empty(rows, N, device="cuda"), torch.empty(rows, K, device="cuda")
    add_rmsnorm(x.cuda(), r.cuda(), g.cuda(), rows, residual_out=ro, codes=xq, scales=sx, rotate=lin.rotate)
    lin.encode(xq, sx, y, rows)
    ref = qref.add_rmsnorm((x + r).numpy(), g.numpy(), 1e-6)[0] @ deq(host, 4).astype(np.float64).T
    err = y.double().cpu().numpy() - ref
    rms = np.sqrt((ref ** 2).mean())
    assert np.sqrt((err ** 2).mean()) <= 0.02 * rms and np.abs(err).max() <= 0.1 * rms
    # and exactly, from the codes
    want = reference(xq.cpu(), sx.cpu(), lin.w.cpu(), lin.scales.cpu())
    assert torch.equal(y.cpu(), want)


@pytest.mark.parametrize("rows", [5, 300])
def test_weights_packed_by_the_launch_before(cuda_device, rows):
    """The linear reads weights ahead of the launch before it; packing leaves them complete, a buffer that is packed again too, eagerly and in a graph."""
    rng, gen = np.random.default_rng(rows), torch.Generator().manual_seed(rows)
    N, K = 640, 1024
    matrices = [affine_case(rng, N, K, 4, cuda_device)[0] for _ in range(2)]
    w, s = torch.zeros(N, K, dtype=torch.int8, device="cuda"), torch.zeros(N, device="cuda")
    lin = I8Linear(w, s)
    x, sx = codes(gen, rows, K).cuda(), torch.rand(rows, generator=gen).cuda()
    want = [torch.empty(rows, N, device="cuda") for _ in matrices]
    for m, y in zip(matrices, want):
        packed = I8Linear.pack(m, 0)
        torch.cuda.synchronize()
        packed.encode(x, sx, y, rows)
    y = torch.empty(8, rows, N, device="cuda")
    def again():
        for i in range(8):
            q = matrices[i % 2].qlinear()
            st = capi.lib().iq_i8_pack(capi.context(0).handle, torch.cuda.current_stream().cuda_stream, C.byref(q), 0, w.data_ptr(), s.data_ptr())
            assert st == 0
            lin.encode(x, sx, y[i], rows)
    again()
    torch.cuda.synchronize()
    for i in range(8):
        assert torch.equal(y[i], want[i % 2])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        again()
    for _ in range(3):
        y.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(y[i], want[i % 2]) for i in range(8))


def test_streams_at_once(cuda_device):
    """Clusters, pairs and the decode linears' own clusters beside one another: a CTA that waits for the others of its cluster holds no tensor memory."""
    rng, gen = np.random.default_rng(3), torch.Generator().manual_seed(3)
    dense, _ = affine_case(rng, 1024, 4096, 4, cuda_device)
    dx, dy = torch.randn(8, 4096, generator=gen).half().cuda(), torch.empty(8, 1024, device="cuda")
    VQMV.encode(dx, dense, dy, 8)
    dense_want = dy.clone()
    jobs = []
    for rows, n, k in ((1, 1024, 4096), (40, 512, 4096), (300, 1024, 1024), (64, 1000, 2048), (200, 600, 2064), (200, 600, 1040)):
        x, sx = codes(gen, rows, k).cuda(), torch.rand(rows, generator=gen).cuda()
        m = I8Linear(codes(gen, n, k).cuda(), torch.rand(n, generator=gen).cuda())
        want = torch.empty(rows, n, device="cuda")
        m.encode(x, sx, want, rows)
        jobs.append((m, x, sx, torch.empty_like(want), want, rows, torch.cuda.Stream()))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for _ in range(20):
        for m, x, sx, y, _, rows, stream in jobs:
            m.encode(x, sx, y, rows, stream=stream)
        VQMV.encode(dx, dense, dy, 8, stream=side)
    torch.cuda.synchronize()
    assert capi.context(0).device_status() == 0
    assert all(torch.equal(j[3], j[4]) for j in jobs) and torch.equal(dy, dense_want)


def test_tensors_of_no_rows(cuda_device):
    m = I8Linear(torch.zeros(8, 64, dtype=torch.int8, device="cuda"), torch.zeros(8, device="cuda"))
    m.encode(torch.empty(0, 64, dtype=torch.int8, device="cuda"), torch.empty(0, device="cuda"), torch.empty(0, 8, device="cuda"), 0)


def test_what_tensors_on_the_gpu_are_refused_for(cuda_device):
    z = lambda *s, dtype=F32: torch.zeros(*s, dtype=dtype, device="cuda")
    m = I8Linear(z(8, 64, dtype=torch.int8), z(8))
    base = {"x": z(4, 64, dtype=torch.int8), "s": z(4), "y": z(4, 8), "rows": 4}
    call = lambda a: m.encode(a["x"], a["s"], a["y"], a["rows"])
    call(base)
    for change in ({"rows": 5}, {"rows": -1}, {"x": z(4, 64)}, {"x": z(4, 48, dtype=torch.int8)}, {"x": z(64, dtype=torch.int8)}, {"x": z(64, 4, dtype=torch.int8).t()},
                   {"x": z(4, 64, dtype=torch.int8).cpu()}, {"s": z(3)}, {"s": z(4, dtype=F16)}, {"s": z(8)[::2]}, {"s": z(4, 1)}, {"y": z(4, 7)}, {"y": z(4, 8).int()}, {"y": z(8, 4).t()},
                   {"y": z(4, 8).cpu()}, {"y": None}):
        with pytest.raises((ValueError, TypeError, AttributeError)):
            call({**base, **change})
    with pytest.raises(capi.IngotError):  # rows 24 bytes apart
        call({**base, "x": z(4, 72, dtype=torch.int8)[:, :64]})
    m.encode(z(1, 64, dtype=torch.int8), z(8)[::2], z(1, 8), 1)


@pytest.mark.parametrize("rows,n,k,pair,parts", [(200, 600, 1040, 1, 2), (200, 1, 1040, 1, 2), (173, 257, 1040, 1, 2), (300, 2049, 2064, 1, 2), (200, 640, 1040, 1, 2), (200, 641, 1040, 1, 2),
                                                 (129, 257, 2064, 1, 3), (470, 640, 2064, 1, 3), (1500, 384, 8208, 1, 3), (1500, 385, 8208, 1, 3), (40, 129, 2064, 0, 8), (17, 4, 4096, 0, 8),
                                                 (3, 129, 1040, 0, 4), (40, 4097, 2064, 0, 4), (64, 9217, 1552, 0, 2)])
def test_divided_tiles_of_few_features(cuda_device, rows, n, k, pair, parts):
    """The last tile's features are few: of a pair the odd CTA may have none of them, and then takes nothing from its counterparts. Beside other calls, whose CTAs follow at once."""
    plan = capi.qmm_i8_plan(rows, n, k)
    assert (plan.pair, plan.parts) == (pair, parts)
    run(torch.Generator().manual_seed(rows + n), rows, n, k, F16, True, 1)
    gen = torch.Generator().manual_seed(n)
    x, w, sx, sw = codes(gen, rows, k), codes(gen, n, k), torch.rand(rows, generator=gen), torch.rand(n, generator=gen)
    want = reference(x, sx, w, sw)
    m, xd, sd = I8Linear(w.cuda(), sw.cuda()), x.cuda(), sx.cuda()
    torch.cuda.synchronize()
    streams, ys = [torch.cuda.Stream() for _ in range(3)], torch.zeros(3, rows, n, device="cuda")
    torch.cuda.synchronize()
    for _ in range(10):
        for s, y in zip(streams, ys):
            m.encode(xd, sd, y, rows, stream=s)
    torch.cuda.synchronize()
    assert capi.context(0).device_status() == 0
    assert all(torch.equal(y.cpu(), want) for y in ys)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("accumulate", [False, True])
@pytest.mark.parametrize("rows,n,k,pair,parts", [(1, 300, 512, 0, 1), (7, 260, 2064, 0, 8), (64, 9217, 1552, 0, 2), (700, 6144, 1040, 1, 1), (200, 640, 1040, 1, 2), (129, 257, 2064, 1, 3)])
def test_scales_that_are_no_numbers(cuda_device, dtype, accumulate, rows, n, k, pair, parts):
    """A row that has come from infinities or NaN (its scale is NaN) is NaN in every type of result, and the other rows are not touched by it."""
    plan = capi.qmm_i8_plan(rows, n, k)
    assert (plan.pair, plan.parts) == (pair, parts)
    gen = torch.Generator().manual_seed(rows)
    x, w, sx, sw = codes(gen, rows, k), codes(gen, n, k), torch.rand(rows, generator=gen), torch.rand(n, generator=gen) * 1e-3
    x[0], sx[0] = 0, float("nan")
    sx[rows // 2], sw[n // 2] = float("nan"), float("inf")
    base = torch.randn(rows, n, generator=gen).to(dtype)
    y = base.cuda()
    I8Linear(w.cuda(), sw.cuda()).encode(x.cuda(), sx.cuda(), y, rows, accumulate=accumulate)
    want = reference(x, sx, w, sw, base if accumulate else None).to(dtype)
    got = y.cpu()
    assert torch.equal(got.isnan(), want.isnan()) and got[0].isnan().all() and got[rows // 2].isnan().all()
    assert torch.equal(got.nan_to_num(7), want.nan_to_num(7))


@pytest.mark.parametrize("rows", [1, 4, 16, 64, 320])
@pytest.mark.parametrize("n,k", [(512, 1024), (4096, 512)])
def test_nan_in_results_of_16_bits(cuda_device, rows, n, k):
    """A NaN that is added to, or that a linear gives in fp32, is one in fp16 and bf16 as well."""
    m, _ = affine_case(np.random.default_rng(rows), n, k, 4, cuda_device)
    gen = torch.Generator().manual_seed(rows)
    x = torch.randn(rows, k, generator=gen)
    encode = VQMV.encode if rows <= 16 else lambda x, m, y, rows, accumulate: m.encode_qmm_f32(x, y, rows, accumulate)
    for poisoned in (False, True):
        if poisoned:
            x[rows // 2] = float("nan")
        nan = []
        for dtype in (F32, F16, BF16):
            y = torch.ones(rows, n, dtype=dtype, device="cuda")
            y[rows // 2, 5] = float("nan")
            encode(x.half().cuda(), m, y, rows, accumulate=True)
            nan.append(y.isnan().cpu())
        assert nan[0][rows // 2, 5] and (poisoned or nan[0].sum() == 1)
        assert torch.equal(nan[0], nan[1]) and torch.equal(nan[0], nan[2])


@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("rotate", [0, 32, 256])
def test_packing_weights_that_are_no_numbers(cuda_device, value, rotate):
    """A feature with a scale or bias that is no number is none in the result either, and the others are as they were."""
    rng = np.random.default_rng(rotate)
    N, K = 40, 512
    m, _ = affine_case(rng, N, K, 4, cuda_device)
    good = I8Linear.pack(m, rotate)
    m.s.view(N, -1)[3, 2] = value
    m.b.view(N, -1)[39, 7] = value
    got = I8Linear.pack(m, rotate)
    keep = torch.ones(N, dtype=torch.bool)
    keep[[3, 39]] = False
    assert torch.equal(got.w.cpu()[keep], good.w.cpu()[keep]) and torch.equal(got.scales.cpu()[keep], good.scales.cpu()[keep])
    gen = torch.Generator().manual_seed(1)
    x, sx = codes(gen, 5, K).cuda(), torch.rand(5, generator=gen).cuda() + 0.1
    for dtype in (F32, F16, BF16):
        y = torch.empty(5, N, dtype=dtype, device="cuda")
        got.encode(x, sx, y, 5)
        assert y[:, 3].isnan().all() and y[:, 39].isnan().all() and y.isnan().sum() == 10
