"""Products in 8-bit integers: rows quantised (as they are, behind a norm, behind a gate) and multiplied, against their definition."""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
ROUND = {torch.bfloat16: 2.0**-8, torch.float32: 2.0**-24}  # a rounding is off by at most half a step, eps / 2 relative to the value


def _ops():
    from nanospec_amd.kernels import ops

    return ops


def _rand(shape, seed, dtype=torch.float32):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def _defined(x: torch.Tensor):
    """float32 rows -> codes and scales by the definition's own 32-bit operations."""
    most = x.abs().amax(1)
    some = most >= 2.0**-100
    inverse = torch.where(some, torch.full_like(most, 127.0) / most, 0.0)
    codes = torch.round(x * inverse[:, None]).clamp(-127, 127)
    return torch.where(some[:, None], codes, 0.0), torch.where(some, most / torch.full_like(most, 127.0), 0.0)


ROWS = [(1, 1), (3, 8), (2, 513), (5, 2048), (7, 4096), (2, 14336), (1, 28672), (2, 32768), (3, 1001), (1, 32767), (4, 20000)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,k", ROWS)
def test_rows(m, k, dtype):
    """Codes and scales are the definition's, bit for bit, of contiguous rows and of rows inside wider ones, at addresses between 16 bytes too."""
    ops = _ops()
    x = _rand((m, k), m + k, dtype) * torch.exp(_rand((m, 1), 3)).to(dtype)
    codes, scales = _defined(x.float())
    for pad in (0, 8, 3):
        wide = torch.full((m, k + 2 * pad), 50.0, dtype=dtype, device=DEV)
        wide[:, pad : pad + k] = x.to(DEV)
        rows = ops.int8_rows(wide[:, pad : pad + k])
        assert torch.equal(rows.codes().cpu().float(), codes) and torch.equal(rows.scales.cpu(), scales), pad


def test_rows_that_are_zero_tiny_or_not_finite():
    ops = _ops()
    x = _rand((8, 640), 1)
    x[0] = 0
    x[1] *= 2.0**-110
    x[2, 5], x[3, 639], x[4, 0] = math.inf, math.nan, -math.inf
    x[5] *= 2.0**100
    x[6] *= 2.0**-95
    rows = ops.int8_rows(x.to(DEV))
    good = [0, 1, 5, 6, 7]
    codes, scales = _defined(x[good])
    assert torch.equal(rows.codes()[good].cpu().float(), codes) and torch.equal(rows.scales[good].cpu(), scales)
    assert bool(torch.isnan(rows.scales[2:5]).all()) and not bool(rows.codes()[:2].any()) and not bool(rows.codes()[2:5].any())
    w = ops.Int8Weight.from_float(_rand((33, 640), 2).to(DEV))
    y = ops.linear_int8(rows, w, dtype=torch.float32)
    assert bool(torch.isnan(y[2:5]).all()) and bool(torch.isfinite(y[good]).all()) and not bool(y[:2].any())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,k", [(1, 64), (5, 2048), (3, 1001), (2, 32768)])
@pytest.mark.parametrize("form", ["resid and x", "resid", "x", "stored elsewhere"])
def test_rows_behind_the_norm(m, k, dtype, form):
    ops = _ops()
    resid, x, weight, eps = _rand((m, k), 1, dtype) * 3, _rand((m, k), 2, dtype), (1 + 0.2 * _rand((k,), 3)).to(dtype), 1e-5
    r = {"resid": resid, "x": x}.get(form, (resid.float() + x.float()).to(dtype))
    keep = resid.to(DEV)
    args = dict(resid=keep if form != "x" else None, x=x.to(DEV) if form != "resid" else None)
    to = torch.full_like(keep, 9.0)
    if form == "resid and x":
        args["resid_out"] = keep
    elif form == "stored elsewhere":
        args["resid_out"] = to
    rows = ops.rmsnorm_int8(weight.to(DEV), eps, **args)
    if form == "resid and x":
        assert torch.equal(keep.cpu(), r)
    else:
        assert torch.equal(keep.cpu(), resid) and torch.equal(to.cpu(), r if form == "stored elsewhere" else torch.full_like(r, 9.0))
    y = r.double() * (r.double().square().mean(1, keepdim=True) + eps).rsqrt() * weight.double()
    most = y.abs().amax(1)
    # the mean of k squares (sums of a thread, a wave and a workgroup: at most 32 + 6 + 16 roundings of 2^-24 of it, halved by the root), 1 / sqrt to 2 units, two products
    off = (27 + 4) * 2.0**-24 + 2.0**-22
    assert bool(((rows.scales.cpu().double() - most / 127).abs() <= (off + 2.0**-23) * most / 127).all())
    # a code is next to the value, or the one beside it where the value lies half way between the two
    far = (rows.codes().cpu().double() - y * (127 / most)[:, None]).abs()
    assert float(far.max()) <= 0.5 + 127 * (2 * off + 2.0**-22)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,k", [(1, 64), (5, 8192), (3, 1001), (2, 28672), (1, 32768)])
def test_rows_behind_the_gate(m, k, dtype):
    ops = _ops()
    gu = _rand((m, 2 * k), m + k, dtype) * 4
    rows = ops.silu_mul_int8(gu.to(DEV))
    g, u = gu.double().chunk(2, 1)
    y = g * torch.sigmoid(g) * u
    most = y.abs().amax(1)
    off = 8 * 2.0**-24  # exp to 2 units, the sum, the quotient, the product, each 2^-24 of the value (the exponential's argument is exact)
    assert bool(((rows.scales.cpu().double() - most / 127).abs() <= (off + 2.0**-23) * most / 127).all())
    far = (rows.codes().cpu().double() - y * (127 / most)[:, None]).abs()
    assert float(far.max()) <= 0.5 + 127 * (2 * off + 2.0**-22)


def _operands(m, n, k, seed):
    gen = torch.Generator().manual_seed(seed)
    cx = torch.randint(-127, 128, (m, k), generator=gen, dtype=torch.int8)
    cw = torch.randint(-127, 128, (n, k), generator=gen, dtype=torch.int8)
    xs, ws = torch.rand(m, generator=gen) + 0.5, torch.rand(n, generator=gen) + 0.5
    return cx, xs, cw, ws


def _rows(cx, xs):
    """Rows in 8 bits whose padding, beyond their values and behind the last row, holds what must not count."""
    ops = _ops()
    m, k = cx.shape
    codes = torch.full((-(-m // 16) * 16, ops.int8_padded_k(k)), 113, dtype=torch.int8)
    codes[:m, :k] = cx
    rows = ops.Int8Rows.from_codes(codes.to(DEV), torch.ones(codes.shape[0], device=DEV))
    return ops.Int8Rows(rows.data, xs.to(DEV), k)


PRODUCTS = [(1, 1, 1), (1, 2048, 2048), (16, 33, 512), (17, 20, 513), (3, 500, 14336), (33, 130, 4096), (64, 1000, 1100), (65, 4096, 768), (128, 257, 2304), (129, 100, 1024),
            (255, 512, 512), (300, 1023, 3333), (520, 64, 8192), (1100, 2050, 640), (8, 7168, 4096), (61, 4096, 4096), (1300, 13003, 600)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,n,k", PRODUCTS)
def test_product(m, n, k, dtype):
    """The sums are whole numbers below 2^31 and exact; two products with the scales and the conversion round three times in 32-bit, then once to the type.  Nothing beside the result
    is written."""
    ops = _ops()
    cx, xs, cw, ws = _operands(m, n, k, m + n + k)
    w = ops.Int8Weight(cw.to(DEV), ws.to(DEV))
    assert torch.equal(w.codes().cpu(), cw)
    room = torch.full((m + 1, n + 5), 7.0, dtype=dtype, device=DEV)
    y = ops.linear_int8(_rows(cx, xs), w, out=room[:m, :n])
    want = (cx.double().to(DEV) @ cw.double().to(DEV).T).cpu() * xs.double()[:, None] * ws.double()
    assert bool(((y.cpu().double() - want).abs() <= (3 * 2.0**-24 * 1.001 + ROUND[dtype]) * want.abs()).all())
    assert bool((room[m] == 7).all()) and bool((room[:, n:] == 7).all())
    assert torch.equal(ops.linear_int8(_rows(cx, xs), w, dtype=dtype), y)


@pytest.mark.parametrize("form", range(6))
@pytest.mark.parametrize("m,n,k,ranges", [(1, 4, 512, 1), (17, 65, 768, 1), (130, 260, 1280, 2), (300, 516, 2304, 4), (257, 130, 4096, 8), (520, 1027, 1024, 2), (1300, 400, 512, 1)])
def test_product_in_every_tile(m, n, k, ranges, form):
    """Tiles and ranges that the plan would not choose: the same whole numbers, times the scales, at sizes off every edge."""
    import ctypes

    from nanospec_amd.kernels import build

    ops = _ops()
    cx, xs, cw, ws = _operands(m, n, k, m + k)
    w, x = ops.Int8Weight(cw.to(DEV), ws.to(DEV)), _rows(cx, xs)
    out = torch.full((m + 1, n + 3), 7.0, device=DEV)
    parts = torch.full((ranges * m * (n + 3),), -5, dtype=torch.int32, device=DEV)
    i = ctypes.c_int
    status = build.core().ns_gemm_int8_many(ops._ptr(out), ops._ptr(parts), ops._ptr(x.data), ops._ptr(x.scales), ops._ptr(w.data), ops._ptr(w.scales), i(m), i(n), i(w.kp), i(n + 3),
                                            i(form), i(ranges), i(ops.F32), ops._stream())
    assert status == 0
    want = (cx.double() @ cw.double().T) * xs.double()[:, None] * ws.double()
    assert bool(((out[:m, :n].cpu().double() - want).abs() <= 4 * 2.0**-24 * 1.001 * want.abs()).all())
    assert bool((out[m] == 7).all()) and bool((out[:, n:] == 7).all())


@pytest.mark.parametrize("blocks", [1, 2, 4])
@pytest.mark.parametrize("m,n,k", [(1, 4, 512), (17, 65, 768), (33, 30, 4096), (64, 16, 1300), (65, 100, 8192), (130, 260, 1280), (16, 17, 14336)])
def test_product_in_every_row_block(m, n, k, blocks):
    """The kernel for few rows with row blocks that the plan would not choose."""
    import ctypes

    from nanospec_amd.kernels import build

    ops = _ops()
    cx, xs, cw, ws = _operands(m, n, k, m + k)
    w, x = ops.Int8Weight(cw.to(DEV), ws.to(DEV)), _rows(cx, xs)
    out = torch.full((m + 1, n + 3), 7.0, device=DEV)
    i = ctypes.c_int
    status = build.core().ns_gemm_int8(ops._ptr(out), ops._ptr(x.data), ops._ptr(x.scales), ops._ptr(w.data), ops._ptr(w.scales), i(m), i(n), i(w.kp), i(n + 3), i(blocks), i(ops.F32),
                                       ops._stream())
    assert status == 0
    want = (cx.double() @ cw.double().T) * xs.double()[:, None] * ws.double()
    assert bool(((out[:m, :n].cpu().double() - want).abs() <= 4 * 2.0**-24 * 1.001 * want.abs()).all())
    assert bool((out[m] == 7).all()) and bool((out[:, n:] == 7).all())


def test_product_of_the_largest_sums():
    """32,768 products of 127 * 127: 528,515,072, of either sign."""
    ops = _ops()
    k = 32768
    cx = torch.full((130, k), 127, dtype=torch.int8)
    cw = torch.full((70, k), 127, dtype=torch.int8)
    cw[1::2] = -127
    w = ops.Int8Weight(cw.to(DEV), torch.ones(70, device=DEV))
    for m in (1, 40, 130):
        y = ops.linear_int8(_rows(cx[:m], torch.ones(m)), w, dtype=torch.float32).cpu()
        assert bool((y[:, ::2] == 127 * 127 * k).all()) and bool((y[:, 1::2] == -127 * 127 * k).all())


def test_product_of_no_rows():
    ops = _ops()
    w = ops.Int8Weight.from_float(torch.randn(48, 64, device=DEV))
    assert ops.linear_int8(ops.int8_rows(torch.randn(0, 64, device=DEV)), w).shape == (0, 48)


@pytest.mark.parametrize("n,k", [(5, 7), (300, 4096), (64, 14336)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_weight_from_values(n, k, dtype):
    ops = _ops()
    w = _rand((n, k), n, dtype)
    w[n // 2] = 0
    made = ops.Int8Weight.from_float(w.to(DEV))
    codes, scales = made.codes().cpu().double(), made.scales[:n].cpu().double()
    most = w.double().abs().amax(1)
    assert bool(((scales - most / 127).abs() <= 2.0**-23 * most).all())
    assert bool(((codes * scales[:, None] - w.double()).abs() <= scales[:, None] * (0.5 + 127 * 2.0**-22)).all()) and not bool(codes[n // 2].any())


@pytest.mark.parametrize("m,n,k", [(65536, 130, 600), (70001, 200, 520), (1_048_600, 17, 64)])
def test_product_of_more_rows_than_a_grid_has_of_them(m, n, k):
    """Rows beyond 65,535, in tiles and, of a small weight, 16 at a time up to the rows that that kernel's grid has; sums below 2^24 are exact in 32-bit too."""
    ops = _ops()
    codes = torch.randint(-127, 128, (m, k), generator=torch.Generator().manual_seed(1), dtype=torch.int8).to(DEV)
    w = torch.randint(-127, 128, (n, k), generator=torch.Generator().manual_seed(2), dtype=torch.int8).to(DEV)
    y = ops.linear_int8(ops.Int8Rows.from_codes(codes, torch.ones(m, device=DEV)), ops.Int8Weight(w, torch.ones(n, device=DEV)), dtype=torch.float32)
    assert torch.equal(y, codes.float() @ w.float().T)


@pytest.mark.parametrize("m,blocks", [(1_048_560, 1), (1_048_577, 2), (1_048_577, 4), (2_097_200, 4)])
def test_few_columns_of_more_rows_than_16_times_a_grid(m, blocks):
    """What the kernel for few rows takes goes by the rows of its workgroups: 65,535 times 16, 32 or 64 of them, one product by the plan's choice and one by each."""
    ops = _ops()
    n, k = 16, 64
    codes = torch.randint(-127, 128, (m, k), generator=torch.Generator().manual_seed(1), dtype=torch.int8).to(DEV)
    w = torch.randint(-127, 128, (n, k), generator=torch.Generator().manual_seed(2), dtype=torch.int8).to(DEV)
    rows, weight = ops.Int8Rows.from_codes(codes, torch.ones(m, device=DEV)), ops.Int8Weight(w, torch.ones(n, device=DEV))
    want = codes.float() @ w.float().T
    assert torch.equal(ops.linear_int8(rows, weight, dtype=torch.float32), want)
    plan, ops.int8_plan = ops.int8_plan, lambda m, n, k, units: ((n, -blocks, 1),)
    try:
        assert torch.equal(ops.linear_int8(rows, weight, dtype=torch.float32), want)
    finally:
        ops.int8_plan = plan


def test_more_workgroups_of_rows_than_a_grid_has_are_refused():
    ops = _ops()
    m = 16 * 65535 + 1
    rows, weight = ops.Int8Rows.from_codes(torch.zeros((m, 64), dtype=torch.int8, device=DEV), torch.ones(m, device=DEV)), ops.Int8Weight(torch.zeros((16, 64), dtype=torch.int8, device=DEV), torch.ones(16, device=DEV))
    plan, ops.int8_plan = ops.int8_plan, lambda m, n, k, units: ((n, -1, 1),)
    try:
        with pytest.raises(ops.KernelRefused):
            ops.linear_int8(rows, weight)
    finally:
        ops.int8_plan = plan
