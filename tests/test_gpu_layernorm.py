"""Layer norm (caif_b200/csrc/layernorm.cu) against its definition in 64 bits.

Tolerances: u = 2^-24 is half a step of fp32, `half` half a step of the result's type.  A sum of n terms whose longest chain
of additions is k long is off by at most k u times the sum of the terms' magnitudes; a thread's chain is n / 256 long at
most where a row has more columns than a block keeps in registers, and 64 covers the rest (32 columns a thread, the tree).
"""
import numpy as np
import pytest
import torch

from caif_b200 import native as nv

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
EPS = 1e-5
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
# one column; less than a warp; odd; a row of 16-byte pieces; widths at the ends of the forms that keep rows in registers
DIMS = [1, 7, 32, 40, 129, 1001, 1024, 4096, 5000, 8192, 8200, 16384, 16389, 32768, 33000]


def half(t):
    return torch.finfo(t).eps / 2


def make(rows, dim, dtype, seed=0, offset=0.25):
    g = torch.Generator(device="cuda").manual_seed(1000 * rows + dim + seed)
    x = (torch.randn(rows, dim, generator=g, device="cuda") * 1.5 + offset).to(dtype)
    dy = torch.randn(rows, dim, generator=g, device="cuda").to(dtype)
    gamma = 1.0 + 0.1 * torch.randn(dim, generator=g, device="cuda")
    beta = 0.1 * torch.randn(dim, generator=g, device="cuda")
    return x, dy, gamma, beta


def ref_fwd(x, gamma, beta, eps=EPS):
    x = x.double()
    mean = x.mean(1, keepdim=True)
    rstd = 1.0 / torch.sqrt((x - mean).square().mean(1, keepdim=True) + eps)
    g = gamma.double() if gamma is not None else torch.ones(x.shape[1], device="cuda", dtype=torch.float64)
    b = beta.double() if beta is not None else torch.zeros(x.shape[1], device="cuda", dtype=torch.float64)
    return (x - mean) * rstd * g + b, mean[:, 0], rstd[:, 0]


def check_fwd(x, gamma, beta, got, eps=EPS):
    y, mean, rstd = got
    want, wm, wr = ref_fwd(x, gamma, beta, eps)
    n = x.shape[1]
    k = (n / 256 + 64) * U
    xd = x.double()
    em = k * xd.abs().mean(1) + U * wm.abs()
    assert bool(((mean.double() - wm).abs() <= em).all())
    # the variance: every term off by twice the mean's error times the distance (and its square), the sum's chain, a division,
    # an addition, a root and a division; rstd follows it with half the relative error
    off = xd - wm[:, None]
    ev = 2 * em * off.abs().mean(1) + em ** 2 + (k + 4 * U) * off.square().mean(1)
    er = (0.5 * ev * wr ** 2 + 4 * U) * wr * 1.01
    assert bool(((rstd.double() - wr).abs() <= er).all())
    g = (gamma.double() if gamma is not None else torch.ones(n, device="cuda", dtype=torch.float64)).abs()
    b = (beta.double() if beta is not None else torch.zeros(n, device="cuda", dtype=torch.float64)).abs()
    xh = off.abs() * wr[:, None]
    tol = g * (wr * em)[:, None] * 1.01 + g * xh * (er / wr + 3 * U)[:, None] + U * (g * xh + b)
    tol = tol * 1.01 + half(y.dtype) * (want.abs() + tol) + (2.0 ** -25 if y.dtype == torch.float16 else 0.0)
    assert bool(((y.double() - want).abs() <= tol).all())


def ref_bwd(dy, x, mean, rstd, gamma):
    dy, x, mean, rstd = dy.double(), x.double(), mean.double()[:, None], rstd.double()[:, None]
    xh = (x - mean) * rstd
    g = dy * gamma.double() if gamma is not None else dy
    dx = rstd * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True))
    return dx, (dy * xh).sum(0), dy.sum(0)


def check_bwd(dy, x, mean, rstd, gamma, got, before=(0.0, 0.0)):
    dx, dg, db = got
    wx, wg, wb = ref_bwd(dy, x, mean, rstd, gamma)
    rows, n = x.shape
    k = (n / 256 + 64) * U
    r = rstd.double()[:, None]
    xh = ((x.double() - mean.double()[:, None]) * r).abs()
    g = (dy.double() * gamma.double() if gamma is not None else dy.double()).abs()
    s1, s2 = g.mean(1, keepdim=True), (g * xh).mean(1, keepdim=True)
    tol = r * (4 * U * (g + s1 + xh * s2) + (k + 3 * U) * s1 + (k + 6 * U) * xh * s2)
    tol = tol * 1.01 + half(dx.dtype) * (wx.abs() + tol) + (2.0 ** -25 if dx.dtype == torch.float16 else 0.0)
    assert bool(((dx.double() - wx).abs() <= tol).all())
    # rows are dealt out to 296 slices at least half of which a long call fills; 128 covers the slices' own sums
    kr = (rows / 148 + 128) * U
    for got_c, want, terms, start in ((dg, wg, (dy.double().abs() * xh).sum(0), before[0]), (db, wb, dy.double().abs().sum(0), before[1])):
        tol = (kr + 4 * U) * terms * 1.01 + U * (want + start).abs()
        assert bool(((got_c.double() - (want + start)).abs() <= tol).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("rows", [1, 5, 333])
def test_layernorm(rows, dim, dtype):
    x, dy, gamma, beta = make(rows, dim, dtype)
    got = nv.layernorm_fwd(x, gamma, beta, EPS)
    check_fwd(x, gamma, beta, got)
    _, mean, rstd = got
    check_bwd(dy, x, mean, rstd, gamma, nv.layernorm_bwd(dy, x, mean, rstd, gamma))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,dim", [(2100, 1024), (1500, 4096), (4000, 129), (700, 8192), (3001, 1001), (1100, 4101), (600, 8191),
                                      (500, 8197), (300, 16384), (40001, 5), (9000, 33), (2500, 640), (1700, 3001)])
def test_layernorm_many_rows(rows, dim, dtype):
    x, dy, gamma, beta = make(rows, dim, dtype)
    got = nv.layernorm_fwd(x, gamma, beta, EPS)
    check_fwd(x, gamma, beta, got)
    check_bwd(dy, x, got[1], got[2], gamma, nv.layernorm_bwd(dy, x, got[1], got[2], gamma))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,dim", [(400, 10000), (350, 12288), (260, 12296), (200, 20480), (170, 24584), (120, 24577), (40, 49149),
                                      (60, 65536), (30, 65537), (70, 70000)])
def test_layernorm_wide_rows(rows, dim, dtype):
    x, dy, gamma, beta = make(rows, dim, dtype)
    got = nv.layernorm_fwd(x, gamma, beta, EPS)
    check_fwd(x, gamma, beta, got)
    want = nv.layernorm_bwd(dy, x, got[1], got[2], gamma)
    check_bwd(dy, x, got[1], got[2], gamma, want)
    for a, b in zip(nv.layernorm_bwd(dy, x, got[1], got[2], gamma), want):
        assert torch.equal(a, b)
    # without the columns' sums, and in place
    lib, s = nv.lib(), torch.cuda.current_stream().cuda_stream
    code = {torch.float32: nv.F32, torch.float16: nv.F16, torch.bfloat16: nv.BF16}[dtype]
    assert lib.caifq_layernorm_bwd(dy.data_ptr(), x.data_ptr(), gamma.data_ptr(), got[1].data_ptr(), got[2].data_ptr(), dy.data_ptr(),
                                   None, None, 0, None, code, rows, dim, s) == 0
    assert torch.equal(dy, want[0])


@pytest.mark.parametrize("dim", [40, 1001, 4096])
def test_layernorm_without_gamma_or_beta(dim):
    x, dy, gamma, beta = make(9, dim, torch.bfloat16)
    for g, b in ((None, None), (gamma, None), (None, beta)):
        got = nv.layernorm_fwd(x, g, b, EPS)
        check_fwd(x, g, b, got)
        check_bwd(dy, x, got[1], got[2], g, nv.layernorm_bwd(dy, x, got[1], got[2], g))


@pytest.mark.parametrize("dim", [24, 1001, 4096])
def test_layernorm_rows_far_from_zero(dim):
    """A mean a thousand times the spread: the variance of the squares' difference would be all rounding."""
    x, dy, gamma, beta = make(6, dim, torch.float32, offset=1500.0)
    check_fwd(x, gamma, beta, nv.layernorm_fwd(x, gamma, beta, EPS))


@pytest.mark.parametrize("dim", [40, 1001, 4096])
@pytest.mark.parametrize("dtype", DTYPES)
def test_layernorm_rows_off_a_16_byte_boundary(dim, dtype):
    x, dy, gamma, beta = make(7, dim, dtype)

    def shifted(t):
        flat = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")
        flat[1:] = t.reshape(-1)
        return flat[1:].view(t.shape)

    xs, ds, gs, bs = shifted(x), shifted(dy), shifted(gamma), shifted(beta)
    got = nv.layernorm_fwd(xs, gs, bs, EPS)
    check_fwd(x, gamma, beta, got)
    check_bwd(dy, x, got[1], got[2], gamma, nv.layernorm_bwd(ds, xs, got[1], got[2], gs))


def test_layernorm_gradients_add_onto_given_ones_and_repeat_bit_for_bit():
    x, dy, gamma, beta = make(777, 2048, torch.bfloat16)
    _, mean, rstd = nv.layernorm_fwd(x, gamma, beta, EPS)
    first = nv.layernorm_bwd(dy, x, mean, rstd, gamma)
    for _ in range(3):
        again = nv.layernorm_bwd(dy, x, mean, rstd, gamma)
        assert all(torch.equal(a, b) for a, b in zip(first, again))
    g0, b0 = torch.full_like(gamma, 3.0), torch.full_like(gamma, -2.0)
    got = nv.layernorm_bwd(dy, x, mean, rstd, gamma, g0, b0)
    assert got[1].data_ptr() == g0.data_ptr() and got[2].data_ptr() == b0.data_ptr()
    assert torch.equal(g0, first[1] + 3.0) and torch.equal(b0, first[2] - 2.0)


def test_layernorm_a_bad_row_stays_alone():
    x, dy, gamma, beta = make(64, 1024, torch.bfloat16)
    clean = nv.layernorm_fwd(x, gamma, beta, EPS)
    bad = x.clone()
    bad[5, 17] = float("nan")
    bad[40, 1000] = float("inf")
    got = nv.layernorm_fwd(bad, gamma, beta, EPS)
    rest = [r for r in range(64) if r not in (5, 40)]
    assert all(torch.equal(a[rest], b[rest]) for a, b in zip(clean, got))
    assert bool(torch.isnan(got[0][5]).all()) and bool(torch.isnan(got[0][40]).all())


def test_layernorm_no_rows():
    x = torch.empty(0, 64, device="cuda")
    y, mean, rstd = nv.layernorm_fwd(x)
    assert y.shape == (0, 64) and mean.numel() == 0 and rstd.numel() == 0
    dx, dg, db = nv.layernorm_bwd(x, x, mean, rstd)
    assert dx.shape == (0, 64) and not bool(dg.any()) and not bool(db.any())
    g0 = torch.ones(64, device="cuda")
    nv.layernorm_bwd(x, x, mean, rstd, None, g0, g0.clone())
    assert bool((g0 == 1).all())


def test_layernorm_equal_values_in_a_row():
    """No spread: rstd is 1 / sqrt(epsilon), y is beta."""
    x = torch.full((3, 4096), 2.0, device="cuda")
    beta = torch.linspace(-1, 1, 4096, device="cuda")
    y, mean, rstd = nv.layernorm_fwd(x, None, beta, EPS)
    assert bool((mean == 2.0).all()) and torch.equal(y, beta.expand(3, -1))
    assert bool(((rstd.double() - EPS ** -0.5).abs() <= 4 * U * EPS ** -0.5).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,dim", [(33, 2048), (1900, 1001), (70, 8205), (3, 40000)])
def test_layernorm_in_place(rows, dim, dtype):
    x, dy, gamma, beta = make(rows, dim, dtype)
    y, mean, rstd = nv.layernorm_fwd(x, gamma, beta, EPS)
    dx, dg, db = nv.layernorm_bwd(dy, x, mean, rstd, gamma)
    x2, m2, r2 = x.clone(), torch.empty_like(mean), torch.empty_like(rstd)
    code = nv.dtype_code(x)
    nv._check(nv.lib().caifq_layernorm_fwd(nv._ptr(x2), nv._ptr(gamma), nv._ptr(beta), nv._ptr(x2), nv._ptr(m2), nv._ptr(r2),
                                           EPS, code, rows, dim, nv._stream()), "in place")
    assert torch.equal(x2, y) and torch.equal(m2, mean) and torch.equal(r2, rstd)
    ws = torch.empty(nv.lib().caifq_layernorm_bwd_workspace_bytes(rows, dim), dtype=torch.uint8, device="cuda")
    for over_dy in (True, False):
        d2, x2, g2, b2 = dy.clone(), x.clone(), torch.empty_like(dg), torch.empty_like(db)
        nv._check(nv.lib().caifq_layernorm_bwd(nv._ptr(d2), nv._ptr(x2), nv._ptr(gamma), nv._ptr(mean), nv._ptr(rstd),
                                               nv._ptr(d2 if over_dy else x2), nv._ptr(g2), nv._ptr(b2), 0, nv._ptr(ws), code, rows, dim,
                                               nv._stream()), "in place")
        assert torch.equal(d2 if over_dy else x2, dx) and torch.equal(g2, dg) and torch.equal(b2, db)
    # rows alone, without a workspace
    d3 = torch.empty_like(dy)
    nv._check(nv.lib().caifq_layernorm_bwd(nv._ptr(dy), nv._ptr(x), nv._ptr(gamma), nv._ptr(mean), nv._ptr(rstd), nv._ptr(d3),
                                           None, None, 0, None, code, rows, dim, nv._stream()), "dx alone")
    assert torch.equal(d3, dx)
    # one of the two gradients
    g3 = torch.empty_like(dg)
    nv._check(nv.lib().caifq_layernorm_bwd(nv._ptr(dy), nv._ptr(x), nv._ptr(gamma), nv._ptr(mean), nv._ptr(rstd), nv._ptr(d3),
                                           nv._ptr(g3), None, 0, nv._ptr(ws), code, rows, dim, nv._stream()), "dgamma alone")
    assert torch.equal(g3, dg)


@pytest.mark.parametrize("dim", [37, 256])
def test_layernorm_gradient_against_differences(dim):
    """<dx, v> against central differences of the definition along v, in 64 bits (step 1e-4: truncation below 1e-7 of the
    values' size), within the bounds of check_bwd."""
    x, dy, gamma, beta = make(4, dim, torch.float32)
    _, mean, rstd = nv.layernorm_fwd(x, gamma, beta, EPS)
    dx, dg, db = nv.layernorm_bwd(dy, x, mean, rstd, gamma)
    g = torch.Generator(device="cuda").manual_seed(dim)
    vx, vg = torch.randn(4, dim, generator=g, device="cuda").double(), torch.randn(dim, generator=g, device="cuda").double()
    h = 1e-4

    def loss(sx, sg, sb):
        return float((ref_fwd(x.double() + sx * vx, gamma.double() + sg * vg, beta.double() + sb * vg)[0] * dy.double()).sum())

    for got, diff in ((float((dx.double() * vx).sum()), (loss(h, 0, 0) - loss(-h, 0, 0)) / (2 * h)),
                      (float((dg.double() * vg).sum()), (loss(0, h, 0) - loss(0, -h, 0)) / (2 * h)),
                      (float((db.double() * vg).sum()), (loss(0, 0, h) - loss(0, 0, -h)) / (2 * h))):
        size = float((dy.double().abs().sum())) * 4
        assert abs(got - diff) <= size * (200 * U + 1e-7)


def test_layernorm_captured_and_on_another_stream():
    x, dy, gamma, beta = make(100, 1024, torch.bfloat16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y, mean, rstd = nv.layernorm_fwd(x, gamma, beta, EPS)
        grads = nv.layernorm_bwd(dy, x, mean, rstd, gamma)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cy, cm, cr = nv.layernorm_fwd(x, gamma, beta, EPS)
        cg = nv.layernorm_bwd(dy, x, cm, cr, gamma)
    graph.replay()
    assert torch.equal(cy, y) and all(torch.equal(a, b) for a, b in zip(cg, grads))
    x2, dy2, _, _ = make(100, 1024, torch.bfloat16, seed=9)
    x.copy_(x2)
    dy.copy_(dy2)
    graph.replay()
    y, mean, rstd = nv.layernorm_fwd(x2, gamma, beta, EPS)
    grads = nv.layernorm_bwd(dy2, x2, mean, rstd, gamma)
    assert torch.equal(cy, y) and all(torch.equal(a, b) for a, b in zip(cg, grads))


def test_layernorm_refusals():
    x, dy, gamma, beta = make(4, 64, torch.float32)
    _, mean, rstd = nv.layernorm_fwd(x)
    with pytest.raises(nv.CaifqError, match="contiguous"):
        nv.layernorm_fwd(x.t())
    with pytest.raises(nv.CaifqError, match="gamma has 63"):
        nv.layernorm_fwd(x, gamma[1:])
    with pytest.raises(nv.CaifqError, match="beta must be"):
        nv.layernorm_fwd(x, gamma, beta.half())
    with pytest.raises(nv.CaifqError, match="no CPU fallback"):
        nv.layernorm_fwd(x.cpu())
    with pytest.raises(KeyError):
        nv.layernorm_fwd(x.double())
    with pytest.raises(nv.CaifqError, match="without dimensions"):
        nv.layernorm_fwd(torch.ones((), device="cuda"))
    with pytest.raises(nv.CaifqError, match="dy must be"):
        nv.layernorm_bwd(dy.half(), x, mean, rstd)
    with pytest.raises(nv.CaifqError, match="dy has"):
        nv.layernorm_bwd(dy[:3], x, mean, rstd)
    with pytest.raises(nv.CaifqError, match="rstd has"):
        nv.layernorm_bwd(dy, x, mean, rstd[:3])
    with pytest.raises(nv.CaifqError, match="both"):
        nv.layernorm_bwd(dy, x, mean, rstd, gamma, gamma.clone())
