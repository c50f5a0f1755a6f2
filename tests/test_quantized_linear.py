"""Rows and weights in 8-bit whole numbers against plain implementations in 64 bits: the numbers, which are exact, their scales, and products."""

from fractions import Fraction

import pytest
import torch

from nkipy_b200 import ops
from nkipy_b200.ops import quantized_linear as ql

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
BF, F32 = torch.bfloat16, torch.float32
EPS = 1e-5
U8, U24 = 2.0 ** -8, 2.0 ** -24             # half a step of bf16 and of fp32, relative


def draws(seed):
    return torch.Generator().manual_seed(seed)


# ------------------------------------------------------------------------------------------------ oracles
def oracle_numbers(x):
    """(numbers, largest magnitude) of rows in 64 bits, from remainders: |x| 127 = k m + r, and r against m / 2."""
    q, tops = [], []
    for row in x.double():
        m = row.abs().max()
        if not torch.isfinite(row.float()).all():
            q.append(torch.zeros_like(row))
            tops.append(float("nan"))
            continue
        tops.append(float(m))
        if m == 0:
            q.append(torch.zeros_like(row))
            continue
        k = torch.floor(127 * row.abs() / m)
        r = (127 * row.abs() - k * m) * 2
        k = k + ((r > m) | ((r == m) & (k % 2 == 1))).double()
        q.append(torch.where(row < 0, -k, k))
    return torch.stack(q).to(torch.int8) if q else x.to(torch.int8), torch.tensor(tops, dtype=torch.float64)


def check_rows(rows, x, factor=None, steps=2):
    """steps: roundings to 32 bits in the scale."""
    q, top = oracle_numbers(x)
    assert rows.values.dtype is torch.int8 and rows.values.shape == x.shape
    assert torch.equal(rows.values.cpu(), q)
    want = top / 127 if factor is None else top / 127 * factor
    got = rows.scale.cpu().double()
    assert torch.equal(got.isnan(), want.isnan())
    fine = ~want.isnan()
    assert bool(((got - want).abs()[fine] <= steps * U24 * want[fine] + 2.0 ** -149).all())


def rows_like_a_layers(g, t, k, dtype=BF):
    return (torch.randn((t, k), generator=g) * torch.exp(0.6 * torch.randn((k,), generator=g))).to(dtype)


def weight_like(g, n, k):
    return (torch.randn((n, k), generator=g) * k ** -0.5).to(BF)


# ------------------------------------------------------------------------------------------------ rows
@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("t,k", [(1, 1), (1, 7), (3, 8), (5, 16), (2, 130), (4, 999), (1, 4096), (33, 2880), (3, 8192), (2, 8200), (2, 16385), (1, 40000)])
def test_rows(device, dtype, t, k):
    x = rows_like_a_layers(draws(t * 100000 + k), t, k, dtype)
    check_rows(ops.quantize_rows(x.to(device)), x, steps=1)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [BF, F32])
def test_rows_of_halves_go_to_the_even_number(device, dtype):
    halves = torch.arange(-64, 64).double() + 0.5                        # of eight bits and fewer: exact in bf16
    x = torch.stack([torch.cat([halves, torch.tensor([127.0 * s], dtype=torch.float64)]) * 2.0 ** e
                     for s in (1, -1) for e in (-120, -60, -3, 0, 5, 60, 110)]).to(dtype)
    rows = ops.quantize_rows(x.to(device))
    check_rows(rows, x, steps=1)
    assert torch.equal(rows.values[0, :128].cpu().double(), halves.round())


@pytest.mark.parametrize("device", DEVICES)
def test_rows_beside_a_half_in_32_bits(device):
    """fp32 numbers one step away from a half of the row's unit."""
    top = torch.tensor(127.0)
    up = torch.nextafter(torch.arange(0, 127) + 0.5, top)
    down = torch.nextafter(torch.arange(0, 127) + 0.5, -top)
    x = torch.stack([torch.cat([up, top[None]]), torch.cat([down, -top[None]])])
    rows = ops.quantize_rows(x.to(device))
    assert rows.values[0, :127].tolist() == list(range(1, 128))
    assert rows.values[1, :127].tolist() == list(range(0, 127))
    check_rows(rows, x, steps=1)
    odd = torch.tensor([[3.0, 1.0, 0.1, 2.9999998]])                      # a maximum that is no power of two
    assert ops.quantize_rows(odd.to(device)).values.tolist() == [[round(127 * Fraction(float(v)) / 3) for v in odd[0]]]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [BF, F32])
def test_rows_of_zeros_of_the_ends_of_the_range_and_not_finite_ones(device, dtype):
    inf, nan, top = float("inf"), float("nan"), float(torch.finfo(dtype).max)
    tiny = 2.0 ** -133
    x = torch.tensor([[0.0] * 5, [-0.0, 0, 0, 0, 0], [1, 2, inf, 3, 4], [nan, 0, 0, 0, 0], [top, -top, top / 2, 1, 0], [tiny, 0, -tiny, 0, 0],
                      [1e-30, 2e-30, 0, 0, -3e-30], [0, -inf, 0, 0, 0]]).to(dtype)
    rows = ops.quantize_rows(x.to(device))
    check_rows(rows, x, steps=1)
    assert rows.scale.isnan().cpu().tolist() == [False, False, True, True, False, False, False, True]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("offset,extra", [(0, 0), (1, 0), (0, 3), (8, 8)])
def test_rows_that_lie_apart_or_off_sixteen_bytes(device, offset, extra):
    g = draws(offset * 10 + extra)
    wide = rows_like_a_layers(g, 6, 48 + offset + extra).to(device)
    x = wide[:, offset:offset + 48]
    check_rows(ops.quantize_rows(x), x.cpu(), steps=1)
    check_rows(ops.quantize_rows(x[::2]), x[::2].cpu(), steps=1)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("t,k", [(1, 1), (1, 64), (3, 50), (2, 2880), (17, 4096), (2, 9000), (1, 17000)])
@pytest.mark.parametrize("parts,bias,residual,x_too", [(0, False, True, True), (0, False, False, True), (3, False, True, False), (1, True, True, True),
                                                       (0, True, False, True), (2, True, False, False)])
def test_normed_rows(device, t, k, parts, bias, residual, x_too):
    g = draws(t * 1000 + k + parts)
    x = rows_like_a_layers(g, t, k) if x_too else None
    r = (2 * rows_like_a_layers(g, t, k).float()).to(BF) if residual else None
    p = torch.randn((parts, t, k), generator=g) if parts else None
    b = rows_like_a_layers(g, 1, k)[0] if bias else None
    w = (1 + 0.2 * torch.randn((k,), generator=g)).to(BF)
    to = lambda v: None if v is None else v.to(device)  # noqa: E731
    h, rows = ops.add_rmsnorm(to(x), to(w), residual_in=to(r), partials=to(p), bias=to(b), eps=EPS, quantize=True)
    total = torch.zeros((t, k), dtype=torch.float64)
    if p is not None:
        total = p.double().sum(0)
    for v in (x, b, r):
        total = total if v is None else total + v.double()
    total = total.to(BF)
    if residual or parts:
        assert torch.equal(h.cpu(), total)
    else:
        assert h is None
    # the norm's factor: squares and their sum in 32 bits (a thread adds up to 16, warps and the block join some 40), the mean, eps, the root
    factor = 1 / torch.sqrt(total.double().square().mean(-1) + EPS)
    check_rows(rows, total.double() * w.double(), factor, steps=64)
    if not bias and not parts and not residual:
        again = ops.rmsnorm(to(x), to(w), EPS, quantize=True)
        assert torch.equal(again.values, rows.values) and torch.equal(again.scale, rows.scale)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("form", ["bf16", "f32", "parts"])
@pytest.mark.parametrize("limit,bias", [(0.0, False), (0.0, True), (7.0, True)])
@pytest.mark.parametrize("t,k", [(1, 1), (3, 24), (2, 500), (5, 2880), (1, 14336)])
def test_gated_rows(device, form, limit, bias, t, k):
    g = draws(t + k)
    x = 2 * torch.randn((3, t, 2 * k) if form == "parts" else (t, 2 * k), generator=g)
    x = x.to(BF) if form == "bf16" else x
    b = (0.3 * torch.randn((2 * k,), generator=g)).to(BF) if bias else None
    rows = ops.silu_mul(x.to(device), limit=limit, bias=None if b is None else b.to(device), quantize=True)
    v = x.double().sum(0) if form == "parts" else x.double()
    v = v if b is None else v + b.double()
    gate, up = v[:, :k], v[:, k:]
    if limit:
        gate, up = gate.clamp(max=limit), up.clamp(-limit, limit)
        y = (up + 1) * gate * torch.special.expit(float(torch.tensor(1.702)) * gate if device == "cuda" else 1.702 * gate)
    else:
        y = gate * torch.special.expit(gate) * up
    check_rows(rows, y, steps=1)


@pytest.mark.parametrize("device", DEVICES)
def test_gated_rows_of_small_and_large_values(device):
    """Gates so negative that 32 bits lose them, rows of zeros, and infinities."""
    g = draws(5)
    rows = [torch.cat([-60 - 20 * torch.rand(64, generator=g), torch.randn(64, generator=g)]),
            torch.cat([-1e-3 * torch.rand(64, generator=g), 1e-4 * torch.randn(64, generator=g)]),
            torch.cat([torch.zeros(64), torch.ones(64)]),
            torch.cat([torch.full((64,), 1e4), torch.full((64,), 1e4)]),
            torch.cat([torch.full((64,), float("inf")), torch.ones(64)]),
            torch.cat([torch.full((64,), -200.0), torch.ones(64)])]
    x = torch.stack(rows)
    got = ops.silu_mul(x.to(device), quantize=True)
    v = x.double()
    check_rows(got, v[:, :64] * torch.special.expit(v[:, :64]) * v[:, 64:], steps=1)


def test_refusals_of_rows():
    x, w = torch.zeros((2, 8), dtype=BF), torch.ones((8,), dtype=BF)
    with pytest.raises(TypeError):
        ops.quantize_rows(x.half())
    with pytest.raises(ValueError):
        ops.quantize_rows(x[0])
    with pytest.raises(ValueError):
        ops.quantize_rows(x.T)
    with pytest.raises(ValueError):
        ops.quantize_rows(torch.zeros((2, 0), dtype=BF))
    with pytest.raises(ValueError):
        ops.add_rmsnorm(x, None, quantize=True)
    with pytest.raises(ValueError):
        ops.add_rmsnorm(x, w, normed_out=torch.empty_like(x), quantize=True)
    with pytest.raises(ValueError):
        ops.rmsnorm(x, w, EPS, out=torch.empty_like(x), quantize=True)
    with pytest.raises(TypeError):
        ops.add_rmsnorm(x.float(), w, quantize=True)
    with pytest.raises(ValueError):
        ops.add_rmsnorm(x, w[:4], quantize=True)
    with pytest.raises(ValueError):
        ops.add_rmsnorm(x, w, residual_in=x[:1], quantize=True)
    with pytest.raises(TypeError):
        ops.add_rmsnorm(None, w, partials=x[None], quantize=True)
    with pytest.raises(ValueError):
        ops.add_rmsnorm(None, w, partials=torch.zeros((0, 2, 8)), quantize=True)
    with pytest.raises(ValueError):
        ops.silu_mul(x[:, :7], quantize=True)
    with pytest.raises(ValueError):
        ops.silu_mul(x, out=x, quantize=True)
    with pytest.raises(TypeError):
        ops.silu_mul(x.half(), quantize=True)


# ------------------------------------------------------------------------------------------------ products
def oracle_product(q, sx, w, sw, gated=False, act="silu", bias=None, residual=None, fp32=False):
    """(result, tolerance) in 64 bits.

    The sum is exact; rounding it to fp32 and both scales take three roundings of 32 bits, each addend one more of the result so far, and bf16
    half a step.  The gate's exponential and quotient are those of the special-function unit: some 2^-20 of the result with arguments below
    a hundred (2^-24 of the argument, which is an absolute error of the exponent, and two steps of each unit)."""
    y = (q.double() @ w.double().T) * sx.double()[:, None] * sw.double()
    tol = 3 * U24 * y.abs()
    if gated:
        n = y.shape[1] // 2
        g, u = y[:, :n], y[:, n:]
        if act == "silu":
            y = g * torch.special.expit(g) * u
        else:
            y = 0.5 * g * (1 + torch.tanh(0.7978845608028654 * (g + 0.044715 * g ** 3))) * u
        # (d/dg of the gate is at most about 1.1; near a gate's zeros the error of g counts, elsewhere that of the exponent)
        tol = 8 * U24 * (g.abs() * u.abs()) * 1.2 + 2.0 ** -16 * y.abs() + (2.0 ** -20 * g.abs() * u.abs() if act != "silu" else 0)
    for v in (bias, residual):
        if v is not None:
            y = y + v.double()
            tol = tol + U24 * y.abs()
    return y, tol + (U24 if fp32 else U8) * 1.001 * y.abs() + 1e-37


def check_product(got, want, tol):
    got = got.cpu().double()
    assert got.shape == want.shape
    off = (got - want).abs() - tol
    assert bool((off <= 0).all()), f"off by {float(off.max()):g} more than it may be, at {int(off.argmax())}"


def made(g, m, n, k, gated=False):
    x = ops.quantize_rows(rows_like_a_layers(g, m, k))
    w = ops.QuantizedWeight.of(weight_like(g, 2 * n if gated else n, k))
    return x, w


def there(x, device):
    return type(x)(x.values.to(device), x.scale.to(device))


SIZES = [(1, 1, 1), (1, 128, 128), (1, 6144, 4096), (2, 130, 100), (15, 1, 4096), (16, 256, 257), (17, 129, 64), (31, 1000, 333), (33, 128, 2880),
         (64, 4096, 14336), (65, 257, 500), (100, 2000, 1000), (127, 64, 128), (128, 300, 640), (129, 256, 128), (129, 1, 16), (200, 700, 300),
         (257, 513, 384), (300, 31, 1000), (414, 512, 2048), (1000, 1025, 129)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("m,n,k", SIZES)
def test_products(device, m, n, k):
    g = draws(m * 7 + n * 3 + k)
    x, w = made(g, m, n, k)
    for fp32 in (False, True):
        want, tol = oracle_product(x.values, x.scale, w.values, w.scale, fp32=fp32)
        check_product(ops.linear(there(x, device), there(w, device), fp32_out=fp32), want, tol)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 128, 128), (3, 200, 1000), (16, 1024, 512), (20, 100, 257), (64, 300, 2048), (65, 129, 640),
                                   (128, 256, 300), (130, 128, 128), (300, 130, 500), (414, 1000, 640)])
def test_gated_products(device, act, m, n, k):
    g = draws(m + n + k)
    x, w = made(g, m, n, k, gated=True)
    want, tol = oracle_product(x.values, x.scale, w.values, w.scale, gated=True, act=act)
    check_product(ops.linear(there(x, device), there(w, device), gated=True, act=act), want, tol)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("m,n,k", [(1, 64, 256), (5, 301, 1024), (64, 256, 4096), (90, 100, 130), (130, 256, 256), (300, 333, 200)])
@pytest.mark.parametrize("bias,residual", [(True, False), (False, True), (True, True)])
def test_products_with_addends(device, m, n, k, bias, residual):
    g = draws(m + n)
    x, w = made(g, m, n, k)
    b = rows_like_a_layers(g, 1, n)[0] if bias else None
    r = rows_like_a_layers(g, m, n) if residual else None
    to = lambda v: None if v is None else v.to(device)  # noqa: E731
    want, tol = oracle_product(x.values, x.scale, w.values, w.scale, bias=b, residual=r)
    got = ops.linear(there(x, device), there(w, device), bias=to(b), residual=to(r))
    check_product(got, want, tol)
    # into part of a wider tensor, the residual in its own place
    wide = torch.full((m, n + 24), 7.0, dtype=BF, device=device)
    out = wide[:, 8:8 + n]
    if residual:
        out.copy_(r.to(device))
    ops.linear(there(x, device), there(w, device), bias=to(b), residual=out if residual else None, out=out)
    assert torch.equal(out, got)
    assert bool((wide[:, :8] == 7).all()) and bool((wide[:, 8 + n:] == 7).all())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("m,n,k,splits", [(1, 256, 1024, 4), (7, 100, 300, 2), (64, 6144, 4096, 3), (64, 130, 640, 8), (1, 64, 64, 8), (200, 300, 520, 3),
                                          (128, 128, 4096, 64)])
def test_partial_sums(device, m, n, k, splits):
    g = draws(m + n + k)
    x, w = made(g, m, n, k)
    b = rows_like_a_layers(g, 1, n)[0]
    parts = ops.linear(there(x, device), there(w, device), splits=splits, bias=b.to(device))
    S = ql.effective_splits(k, splits)
    assert parts.shape == (S, m, n) and parts.dtype is F32
    step = -(-(-(-k // 128)) // S) * 128
    for s in range(S):
        at = slice(s * step, (s + 1) * step)
        want, tol = oracle_product(x.values[:, at], x.scale, w.values[:, at], w.scale, bias=b if s == 0 else None, fp32=True)
        check_product(parts[s], want, tol)


@pytest.mark.gpu
def test_splits_are_the_librarys():
    for k in (1, 100, 128, 129, 1000, 4096, 14336, 30000):
        for s in (1, 2, 3, 5, 8, 64, 1000):
            assert ops._lib.lib().nkb_gemm_i8_splits(k, s) == ql.effective_splits(k, s)


@pytest.mark.parametrize("device", DEVICES)
def test_largest_sums(device):
    """All numbers at their ends, the longest k: the sum is just below 2^31."""
    k = ql.MAX_K
    x = ops.QuantizedRows(torch.full((3, k), 127, dtype=torch.int8), torch.tensor([1.0, 0.5, 2.0]))
    v = torch.full((130, k), 127, dtype=torch.int8)
    v[1::2] = -127
    w = ops.QuantizedWeight(v, torch.ones(130))
    want, tol = oracle_product(x.values, x.scale, w.values, w.scale, fp32=True)
    check_product(ops.linear(there(x, device), there(w, device), fp32_out=True), want, tol)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("m", [1, 64, 200])
def test_rows_that_are_not_finite_and_zeros_stay_among_themselves(device, m):
    g = draws(m)
    x = rows_like_a_layers(g, m, 256)
    x[m // 2] = float("nan")
    x[m - 1] = 0 if m > 1 else x[m - 1]
    w = weight_like(g, 200, 256)
    w[7, 3] = float("inf")
    got = ops.linear(x.to(device), ops.QuantizedWeight.of(w.to(device))).cpu()
    bad = got.isnan()
    assert bool(bad[m // 2].all()) and bool(bad[:, 7].all())
    bad[m // 2], bad[:, 7] = False, False
    assert not bool(bad.any())
    if m > 1:
        assert bool((got[m - 1, :7] == 0).all())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("m,k", [(1, 100), (3, 4096), (64, 2880), (150, 333)])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_products_of_rows_that_come_in_more_bits(device, m, k, dtype):
    g = draws(m * k)
    x, w = rows_like_a_layers(g, m, k, dtype), weight_like(g, 300, k)
    q = ops.QuantizedWeight.of(w.to(device))
    rows = ops.quantize_rows(x.to(device))
    got = ops.linear(x.to(device), q)
    assert torch.equal(got, ops.linear(rows, q))
    # as near to the product in 64 bits as 8 bits say: half a scale of every number against the other's values
    want = x.double() @ w.double().T
    dx, dw = rows.scale.cpu().double() / 2, q.scale.cpu().double() / 2
    may = dx[:, None] * w.double().abs().sum(1) + (x.double().abs().sum(1)[:, None] + k * dx[:, None]) * dw
    assert bool(((got.cpu().double() - want).abs() <= may * 1.001 + U8 * 1.01 * (want.abs() + may)).all())


@pytest.mark.parametrize("device", DEVICES)
def test_nothing_to_do(device):
    w = ops.QuantizedWeight.of(torch.randn((40, 24)).to(device))
    x = torch.zeros((0, 24), dtype=BF, device=device)
    assert ops.linear(x, w).shape == (0, 40)
    assert ops.quantize_rows(x).shape == (0, 24)
    assert ops.silu_mul(x, quantize=True).shape == (0, 12)
    h, rows = ops.add_rmsnorm(x, torch.ones(24, dtype=BF, device=device), residual_in=x, quantize=True)
    assert h.shape == (0, 24) and rows.shape == (0, 24)


@pytest.mark.parametrize("device", DEVICES)
def test_layouts_of_weights(device):
    """Rows off sixteen bytes are laid out anew; rows with room behind them stay where they are."""
    v = torch.randint(-127, 128, (20, 64), dtype=torch.int8, device=device)
    s = torch.rand(20, device=device)
    kept = ops.QuantizedWeight(v[:, :33], s)
    assert kept.values.data_ptr() == v.data_ptr() and kept.ld == 64
    moved = ops.QuantizedWeight(v[:, 1:34], s)
    assert moved.ld % 16 == 0 and torch.equal(moved.values, v[:, 1:34])
    x = ops.quantize_rows(torch.randn((3, 33), device=device))
    assert torch.equal(ops.linear(x, moved), ops.linear(x, ops.QuantizedWeight(v[:, 1:34].contiguous(), s)))
    assert torch.equal(moved.dequantize(), v[:, 1:34].float() * s[:, None])


def test_refusals_of_products():
    w = ops.QuantizedWeight.of(torch.randn((8, 32)))
    x = ops.quantize_rows(torch.randn((2, 32)))
    b = torch.zeros((2, 8), dtype=BF)
    with pytest.raises(TypeError):
        ops.linear(x, torch.zeros((8, 32), dtype=BF))
    with pytest.raises(ValueError):
        ops.linear(ops.quantize_rows(torch.randn((2, 31))), w)
    with pytest.raises(ValueError):
        ops.linear(torch.randn((2, 31)), w)
    with pytest.raises(TypeError):
        ops.linear(torch.zeros((2, 32), dtype=torch.float16), w)
    for kw in (dict(out_act="relu2"), dict(gated=True, bias=b[0, :4]), dict(gated=True, residual=b[:, :4]), dict(gated=True, splits=2),
               dict(gated=True, act="relu"), dict(splits=2, residual=b), dict(bias=b[0, :7]), dict(residual=b[:1]), dict(out=b[:, :7]),
               dict(gated=True, fp32_out=True), dict(out=b.T.contiguous().T)):
        with pytest.raises(ValueError):
            ops.linear(x, w, **kw)
    for kw in (dict(bias=torch.zeros(8)), dict(residual=torch.zeros((2, 8))), dict(out=torch.zeros((2, 8))), dict(fp32_out=True, out=b)):
        with pytest.raises(TypeError):
            ops.linear(x, w, **kw)
    with pytest.raises(ValueError):
        ops.linear(x, ops.QuantizedWeight.of(torch.randn((7, 32))), gated=True)
    with pytest.raises(TypeError):
        ops.QuantizedWeight(torch.zeros((2, 4)), torch.ones(2))
    with pytest.raises(TypeError):
        ops.QuantizedRows(torch.zeros((2, 4), dtype=torch.int8), torch.ones(2).half())
    for v, s in (((2, 4), 3), ((2, 0), 2), ((2, ql.MAX_K + 1), 2), ((2, 4, 1), 2)):
        with pytest.raises(ValueError):
            ops.QuantizedWeight(torch.zeros(v, dtype=torch.int8), torch.ones(s))


# ------------------------------------------------------------------------------------------------ captured, and on other streams
@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 64, 300])
def test_captured_and_replayed(m):
    g = draws(m)
    x, n, k = rows_like_a_layers(g, m, 1024).cuda(), 512, 1024
    w, w2 = (ops.QuantizedWeight.of(weight_like(g, a, b).cuda()) for a, b in ((2 * n, k), (k, n)))
    norm = torch.ones(k, dtype=BF, device="cuda")

    def step(h):
        h, rows = ops.add_rmsnorm(h, norm, residual_in=h, quantize=True)
        return ops.linear(ops.linear(rows, w, gated=True), w2, residual=h)

    want = [step(x), step(x * 2)]
    buf = x.clone()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(buf)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(buf)
    for scale, ref in ((1, want[0]), (2, want[1]), (1, want[0])):
        buf.copy_(x * scale)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ref)


@pytest.mark.gpu
def test_streams_beside_one_another():
    g = draws(1)
    x = [rows_like_a_layers(g, 40, 2048).cuda() for _ in range(4)]
    w = ops.QuantizedWeight.of(weight_like(g, 1000, 2048).cuda())
    want = [ops.linear(v, w) for v in x]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in x]
    for _ in range(5):
        got = []
        for s, v in zip(streams, x):
            with torch.cuda.stream(s):
                got.append(ops.linear(v, w))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 64, 300])
def test_weights_made_right_ahead_of_their_product(m):
    """The product fetches weights ahead of its wait for the kernel before it, which is the one that makes them."""
    g = draws(m)
    x = ops.quantize_rows(rows_like_a_layers(g, m, 2048).cuda())
    ws = [weight_like(g, 4096, 2048).cuda() for _ in range(4)]
    want = []
    for w in ws:
        q = ops.QuantizedWeight.of(w)
        torch.cuda.synchronize()
        want.append(ops.linear(x, q))
    junk = torch.full((4096 * 2048,), 99, dtype=torch.int8, device="cuda")
    for _ in range(5):
        for w, y in zip(ws, want):
            del junk                                                 # (the new weight's memory has other numbers)
            q = ops.QuantizedWeight.of(w)
            got = ops.linear(x, q)
            assert torch.equal(got, y)
            del q
            junk = torch.full((4096 * 2048,), 99, dtype=torch.int8, device="cuda")


@pytest.mark.parametrize("device", DEVICES)
def test_the_lowest_number(device):
    """-128, which no row that was brought into 8 bits here has, counts as what it is."""
    v = torch.randint(-128, 128, (70, 300), dtype=torch.int8, generator=draws(0))
    v[:, ::3] = -128
    x, w = ops.QuantizedRows(v, torch.rand(70)), ops.QuantizedWeight(v.flip(0), torch.rand(70))
    for m in (1, 2, 40, 70):
        rows = ops.QuantizedRows(x.values[:m].contiguous(), x.scale[:m])
        want, tol = oracle_product(rows.values, rows.scale, w.values, w.scale, fp32=True)
        check_product(ops.linear(there(rows, device), there(w, device), fp32_out=True), want, tol)


@pytest.mark.parametrize("device", DEVICES)
def test_normed_rows_in_the_place_of_the_stream(device):
    """The residual stream may be written where it, or what is added, was; narrow rows and ones that are computed twice."""
    for k in (64, 4096, 20000):
        g = draws(k)
        x, r = rows_like_a_layers(g, 3, k), rows_like_a_layers(g, 3, k)
        w = torch.ones(k, dtype=BF)
        want, rows = ops.add_rmsnorm(x.to(device), w.to(device), residual_in=r.to(device), quantize=True)
        for place in (0, 1):
            a, b = x.to(device, copy=True), r.to(device, copy=True)
            h, q = ops.add_rmsnorm(a, w.to(device), residual_in=b, residual_out=(a, b)[place], quantize=True)
            assert h is (a, b)[place] and torch.equal(h, want) and torch.equal(q.values, rows.values) and torch.equal(q.scale, rows.scale)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("offset", [0, 1, 2, 3, 4, 5, 6, 7, 9])
def test_columns_that_start_anywhere(device, offset):
    """Rows whose columns lie across pieces of sixteen bytes, whatever they are moved by, and rows that share their memory."""
    g = draws(offset)
    x = rows_like_a_layers(g, 5, 1030)
    memory = torch.full((offset + 5 * 1030,), float("nan"), dtype=BF, device=device)[offset:].view(5, 1030)
    memory.copy_(x)
    for width in (1030 - offset, 1024, 17, 9):
        check_rows(ops.quantize_rows(memory[:, :width]), x[:, :width], steps=1)
        check_rows(ops.quantize_rows(memory[:, 1030 - width:]), x[:, 1030 - width:], steps=1)
    check_rows(ops.quantize_rows(memory[2:3].expand(4, 1030)), x[2:3].expand(4, 1030), steps=1)
    flat = x.reshape(-1)
    check_rows(ops.quantize_rows(memory.reshape(-1).as_strided((40, 33), (7, 1), memory.storage_offset())), flat.as_strided((40, 33), (7, 1), 0), steps=1)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("m,n,k,gated", [(300, 1001, 96, False), (300, 1001, 96, True), (260, 2050, 130, False), (700, 333, 64, True), (513, 4100, 257, False)])
@pytest.mark.parametrize("fp32,addends", [(False, False), (False, True), (True, False)])
def test_products_into_rows_off_sixteen_bytes(device, m, n, k, gated, fp32, addends):
    if gated and (fp32 or addends):
        return
    g = draws(m + n + k)
    x, w = made(g, m, n, k, gated)
    rows, weight = there(x, device), there(w, device)
    bias = torch.randn((n,), generator=g).to(BF) if addends else None
    residual = torch.randn((m, n), generator=g).to(BF) if addends else None
    base = torch.full((m, n + 3), 7.0, dtype=F32 if fp32 else BF, device=device)
    out = base[:, 1:n + 1]
    kw = dict(gated=True) if gated else dict(fp32_out=fp32)
    if addends:
        kw.update(bias=bias.to(device), residual=residual.to(device))
    want, tol = oracle_product(x.values, x.scale, w.values, w.scale, gated=gated, bias=bias, residual=residual, fp32=fp32)
    for into in (None, out):
        got = ops.linear(rows, weight, out=into, **kw)
        assert into is None or got.data_ptr() == out.data_ptr()
        check_product(got, want, tol)
    assert bool((base[:, 0] == 7).all()) and bool((base[:, n + 1:] == 7).all())


@pytest.mark.gpu
@pytest.mark.parametrize("t,k", [(3, 1), (3, 9), (5, 23), (4, 257), (3, 263), (7, 1030), (5, 2557), (3, 9001), (2, 20003), (11000, 301), (6000, 2557)])
@pytest.mark.parametrize("start", [0, 3])
def test_normed_rows_of_odd_widths_in_place(t, k, start):
    """The stream's rows start anywhere between pieces of sixteen bytes; what lies ahead of it and behind it stays."""
    g = draws(t + k)
    x, r = rows_like_a_layers(g, t, k), rows_like_a_layers(g, t, k)
    w = (1 + 0.2 * torch.randn((k,), generator=g)).to(BF)
    h, q = ops.add_rmsnorm(x, w, residual_in=r, eps=EPS, quantize=True)
    for place in ("new", "x", "stream"):
        memory = [torch.full((start + t * k + 5,), 7.0, dtype=BF, device="cuda") for _ in range(2)]
        a, b = (m[start:start + t * k].view(t, k) for m in memory)
        a.copy_(x), b.copy_(r)
        got, rows = ops.add_rmsnorm(a, w.cuda(), residual_in=b, residual_out={"new": None, "x": a, "stream": b}[place], eps=EPS, quantize=True)
        assert torch.equal(got.cpu(), h) and torch.equal(rows.values.cpu(), q.values)
        assert bool(((rows.scale.cpu().double() - q.scale.double()).abs() <= 64 * U24 * q.scale.double()).all())
        assert all(bool((m[:start] == 7).all()) and bool((m[start + t * k:] == 7).all()) for m in memory)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("t,k", [(5, 9), (3, 263), (9000, 301), (6000, 930), (6000, 928), (3000, 2557), (3000, 5000), (3, 17001)])
def test_many_gated_rows(dtype, t, k):
    g = draws(t + k)
    x = (2 * torch.randn((t, 2 * k), generator=g)).to(dtype)
    q, rows = ops.silu_mul(x, quantize=True), ops.silu_mul(x.cuda(), quantize=True)
    assert torch.equal(rows.values.cpu(), q.values)
    assert bool(((rows.scale.cpu().double() - q.scale.double()).abs() <= 2 * U24 * q.scale.double()).all())


@pytest.mark.gpu
@pytest.mark.parametrize("form", ["plain", "bias", "residual", "fp32", "silu", "gelu_tanh", "parts"])
@pytest.mark.parametrize("n,k,size", [(512, 1024, 1.0), (257, 700, 1.0), (512, 1024, 30.0), (300, 512, 1e-30)])
def test_a_token_has_the_same_bits_in_every_batch(form, n, k, size):
    """One and two tokens on the CUDA cores, few of them on narrow tiles with and without a cluster, prompts on pairs: the tokens that they share are the
    same, for gates of tens too, and for scales that bring results below the normal numbers of 32 bits."""
    g = draws(n + k)
    rows = 700
    gated = form in ("silu", "gelu_tanh")
    x = ops.quantize_rows((size * rows_like_a_layers(g, rows, k).float()).to(BF).cuda())
    w = weight_like(g, 2 * n if gated else n, k)
    w = ops.QuantizedWeight.of((w.float() * (1e-8 if size < 1e-3 else 1.0)).to(BF).cuda())
    bias = rows_like_a_layers(g, 1, n)[0].cuda() if form in ("bias", "residual", "parts") else None
    residual = rows_like_a_layers(g, rows, n).cuda()
    ys = {}
    for m in (1, 2, 3, 16, 30, 64, 128, 300, 700):
        kw = dict(gated=True, act=form) if gated else dict(bias=bias)
        if form == "residual":
            kw["residual"] = residual[:m]
        if form in ("fp32", "parts"):
            kw["fp32_out"] = True
        if form == "parts":
            kw["splits"] = 3
        ys[m] = ops.linear(ops.QuantizedRows(x.values[:m], x.scale[:m]), w, **kw)
    for m, y in ys.items():
        assert torch.equal(y, ys[700][:, :m] if form == "parts" else ys[700][:m]), m
    if form not in ("parts", "residual"):
        # whole products, k in one piece: fp32 rows go the same way
        bf = (size * rows_like_a_layers(draws(n + k), rows, k).float()).to(BF).cuda()
        kw = dict(gated=True, act=form) if gated else dict(bias=bias, fp32_out=form == "fp32")
        for m in (1, 2, 64):
            assert torch.equal(ops.linear(bf[:m], w, **kw), ys[700][:m])


@pytest.mark.parametrize("device", DEVICES)
def test_the_clamped_gates_factors_have_32_bits(device):
    """Columns whose number is another one where alpha has 64: the same on both devices."""
    gate = torch.tensor([[7.0, float.fromhex("-0x1.1edd34p+1"), float.fromhex("-0x1.f4e338p+0"), float.fromhex("0x1.087114p+0")]])
    up = torch.tensor([[7.0, float.fromhex("-0x1.63d0d8p+2"), float.fromhex("0x1.216e64p+1"), float.fromhex("0x1.c09ff8p+0")]])
    alpha = float(torch.tensor(1.702))
    y = (up.double() + 1) * gate.double() / (1 + torch.exp(-alpha * gate.double()))
    rows = ops.silu_mul(torch.cat([gate, up], 1).to(device), limit=7.0, quantize=True)
    check_rows(rows, y, steps=1)
    assert rows.values.tolist() == [[127, 0, 0, 6]]


@pytest.mark.parametrize("device", DEVICES)
def test_the_stream_of_a_norm_is_rounded_once(device):
    """Sums beside the middle of two bf16 numbers, which 32 bits hold as the middle itself."""
    k, middle, off = 16, 2.0 ** -8, 2.0 ** -31
    x = torch.ones((2, k), dtype=BF)
    x[:, 8:] = -1
    parts = torch.full((2, 2, k), off)
    parts[0, :, :8], parts[0, :, 8:] = middle, -middle
    parts[1, 1] = -off
    w = torch.ones(k, dtype=BF)
    h, rows = ops.add_rmsnorm(x.to(device), w.to(device), partials=parts.to(device), eps=EPS, quantize=True)
    up = 1 + 2.0 ** -7
    # above the middle: away from it, below: towards it; -1 - 2^-8 + 2^-31 is nearer to -1
    want = torch.tensor([[up] * 8 + [-1.0] * 8, [1.0] * 8 + [-up] * 8])
    assert torch.equal(h.cpu().float(), want)
    check_rows(rows, want.double(), 1 / torch.sqrt(want.double().square().mean(-1) + EPS), steps=64)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("t,k", [(24, 131000), (3, 24), (5, 1001), (64, 14336), (330, 928), (700, 2880)])
def test_sums_of_gates_far_below_zero(device, t, k):
    """Gates between -80 and -65, which ups of e^65 and more lift to numbers again: the exponential makes 80 roundings of the gate's one."""
    g = draws(t + k)
    x = torch.randn((2, t, 2 * k), generator=g)
    gate = -65 - 15 * torch.rand((t, k), generator=g)
    x[0, :, :k], x[1, :, :k] = gate, 0.1 * x[1, :, :k]
    x[0, :, k:] *= torch.exp(-gate)
    got = ops.silu_mul(x.to(device), quantize=True)
    v = x.double().sum(0)
    check_rows(got, v[:, :k] * torch.special.expit(v[:, :k]) * v[:, k:], steps=1)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("form", ["bf16", "f32", "parts"])
@pytest.mark.parametrize("t,k", [(4, 24), (6, 999), (5, 2880), (64, 14336), (4, 20000), (1300, 300)])
def test_gates_beyond_the_range_of_the_exponential(device, form, t, k):
    """exp(88) is the last one that 32 bits hold: gates down to -100 and ups up to 1e38, ahead of the row's other columns, among them and alone."""
    g = draws(t * k)
    x = torch.randn((t, 2 * k), generator=g)
    far = torch.rand((t, k), generator=g) < 0.1
    far[0], far[1] = True, False
    x[:, :k] = torch.where(far, -80 - 20 * torch.rand((t, k), generator=g), x[:, :k])
    lift = torch.exp2(100 + 26 * torch.rand((t, k), generator=g))
    x[:, k:] = torch.where(far, x[:, k:] * lift * torch.tensor([1.0, 1.0, 1e-4, 1e-12]).repeat(t)[:t, None], x[:, k:])
    x[:, k:] = x[:, k:].clamp(-3e38, 3e38)
    x = x.to(BF) if form == "bf16" else x
    given = torch.stack([x, torch.zeros_like(x)]) if form == "parts" else x
    got = ops.silu_mul(given.to(device), quantize=True)
    v = x.double()
    check_rows(got, v[:, :k] * torch.special.expit(v[:, :k]) * v[:, k:], steps=1)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [BF, F32])
def test_clamped_gates_whose_product_leaves_the_range(device, dtype):
    """(up + 1) * gate is beyond 32 bits where the gate is -1e38; its sigmoid is zero.  A gate of minus infinity is not a number, here as elsewhere."""
    x = torch.tensor([[-1e38, 3.0, -0.5, 2.0, 7.0, 5.0, -1.0, 3.0], [-1e38] * 4 + [7.0] * 4, [-float("inf"), 1, 1, 1, 7, 1, 1, 1], [-30, 1, -16, 2, 7, 1, 1, 1]]).to(dtype)
    alpha = float(torch.tensor(1.702))
    got = ops.silu_mul(x.to(device), limit=7.0, quantize=True)
    v = x.double()
    gate, up = v[:, :4].clamp(max=7), v[:, 4:].clamp(-7, 7)
    y = (up + 1) * gate / (1 + torch.exp(-alpha * gate))
    check_rows(got, y, steps=1)
    assert got.scale.isnan().cpu().tolist() == [False, False, True, False]
