"""Layer normalisation of rows far from zero and of sums over many terms, to the last digits of float32.

Tolerances.  A row's sums are chains of at most c = ceil(dim / 64) + 8 float32 additions where a wave holds a
row, ceil(dim / 256) + 10 where a workgroup does (beyond 2048 elements), or 12 behind chains in double (beyond
8192): C = c 2^-24 of the sum of magnitudes.  The mean is at first off by C |x|; the mean of the
differences from it, which are exact but for 2^-24 of themselves, takes that away up to
C (mean |d| + C |mean|), so y is off by that times rstd and by |h| times the relative error of rstd,
C (1 + (C |mean| rstd)^2) and a few roundings; the stored result adds u |y|."""
import numpy as np
import pytest
import torch

from mlx_audio_amd.frontends import layer_norm, layer_norm_backward
from oracle import transformer as o
from test_gpu_layer_norm import TYPES, f64, make, tiny, u

pytestmark = pytest.mark.gpu
EPS = 2.0 ** -24


def additions(dim):
    return -(-dim // 64) + 8 if dim <= 2048 else -(-dim // 256) + 10 if dim <= 8192 else 12


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("dim", [100, 640, 1280, 2048, 3000, 8192, 9001, 100_003])
@pytest.mark.parametrize("offset,spread", [(0.0, 1.0), (30.0, 1.0), (1000.0, 0.5), (10000.0, 1.0), (-50000.0, 30.0)])
def test_rows_far_from_zero(gpu, t, dim, offset, spread):
    t = TYPES[t]
    x = make((6, dim), t, dim, offset, spread)
    w, b = make((dim,), torch.float32, 1, 1.0, 0.1), make((dim,), torch.float32, 2, 0.0, 0.1)
    y, mean, rstd = layer_norm(x, w, b, return_stats=True)
    wd, bd = f64(w), f64(b)
    want, wmean, wrstd = o.layer_norm(f64(x), wd, bd)
    C = additions(dim) * EPS
    d = np.abs(f64(x) - wmean[:, None])
    e_mean = C * (d.mean(-1) + 1.5 * C * np.abs(wmean))
    assert (np.abs(f64(mean) - wmean) <= 1.01 * EPS * np.abs(wmean) + 1.1 * e_mean).all()
    rel = (C + 8 * EPS) * (1 + 2 * (C * np.abs(wmean) * wrstd) ** 2)
    assert (np.abs(f64(rstd) - wrstd) <= rel * wrstd).all()
    h = d * wrstd[:, None]
    tol = u(t) * np.abs(want) + tiny(t) + 2 * EPS * np.abs(bd) \
        + np.abs(wd) * (1.1 * e_mean[:, None] * wrstd[:, None] + h * (rel[:, None] + 4 * EPS))
    err = np.abs(f64(y) - want)
    assert (err <= 1.001 * tol).all(), np.max(err / tol)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("value", [0.1, 12345.678, -3e-5])
@pytest.mark.parametrize("dim", [7, 640, 1280, 5000, 20001])
def test_constant_rows(gpu, t, value, dim):
    """Nothing is left of a constant but 2^-24 of the error of its mean, times 1 / sqrt(eps)."""
    x = torch.full((3, dim), value, device="cuda", dtype=TYPES[t])
    value = abs(float(x[0, 0]))
    y, mean, rstd = layer_norm(x, return_stats=True)
    C = additions(dim) * EPS
    assert (f64(y.abs()) <= 1.01 * (2 * C * C * value / 1e-5 ** 0.5 + EPS * C * value)).all()
    assert (np.abs(f64(mean) - f64(x[:, 0])) <= 2 * EPS * value).all()
    assert (f64(rstd) <= 1.0001 / 1e-5 ** 0.5).all() and (f64(rstd) >= 0.9999 / np.sqrt(1e-5 + (C * value) ** 2 * 4 * C)).all()


def test_bad_rows_keep_their_statistics_bad(gpu):
    x = make((5, 1280), torch.float32, 3)
    x[1, 9], x[3, 0] = float("nan"), float("inf")
    y, mean, rstd = layer_norm(x, return_stats=True)
    for bad in (1, 3):
        assert torch.isnan(y[bad]).all() and not torch.isfinite(mean[bad]) and torch.isnan(rstd[bad])
    assert all(torch.isfinite(v[[0, 2, 4]]).all() for v in (y, mean, rstd))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows,dim", [(700, 8200), (200, 20001), (65, 9000), (129, 40_000)])
def test_gradients_of_long_rows(gpu, t, rows, dim):
    """Rows of more than 8192 elements, more of them than the column sums have groups (64).  The sums of dweight
    and dbias and those within a row are chains in double: what is left are the roundings of the terms (h: two
    of 2^-24 of |x - mean| rstd; a product: none in the sum of dy) and of the parts, 4 2^-24 of the magnitudes."""
    t = TYPES[t]
    x, dy = make((rows, dim), t, 4, 3.0), make((rows, dim), t, 5, 0.1)
    w = make((dim,), torch.float32, 6, 1.0, 0.1)
    _, mean, rstd = layer_norm(x, w, return_stats=True)
    dx, dw, db = layer_norm_backward(dy, x, mean, rstd, w)
    xd, gd, wd, md, rd = f64(x), f64(dy), f64(w), f64(mean), f64(rstd)
    ex, ew, eb = o.layer_norm_backward(gd, xd, md, rd, wd)
    h = np.abs(xd - md[:, None]) * rd[:, None]
    assert (np.abs(f64(dw) - ew) <= 6 * EPS * (np.abs(gd) * h).sum(0)).all()
    assert (np.abs(f64(db) - eb) <= 2 * EPS * np.abs(gd).sum(0)).all()
    g = np.abs(gd * wd)
    # 12 additions behind the double chains, and the roundings of the terms
    mag = g * 4 + 18 * g.mean(-1, keepdims=True) + h * (22 * (g * h).mean(-1, keepdims=True))
    tol = u(t) * np.abs(ex) + 1.01 * EPS * rd[:, None] * mag + tiny(t)
    err = np.abs(f64(dx) - ex)
    assert (err <= tol).all(), np.max(err / tol)


@pytest.mark.parametrize("t", TYPES)
def test_column_sums_of_many_long_rows(gpu, t):
    """469 rows in each of the 64 groups, terms of one sign: a chain in float32 would be off by several 2^-24."""
    t = TYPES[t]
    g = torch.Generator(device="cuda").manual_seed(7)
    x = torch.randn((30_000, 8200), generator=g, device="cuda").to(t)
    dy = (torch.rand((30_000, 8200), generator=g, device="cuda") + 0.5).to(t)
    w = torch.ones(8200, device="cuda")
    _, mean, rstd = layer_norm(x, w, return_stats=True)
    _, dw, db = layer_norm_backward(dy * x.sign(), x, mean, rstd, w)
    h = (x.double() - mean.double()[:, None]) * rstd.double()[:, None] * x.sign().double()
    want = (h * dy.double()).sum(0)
    assert ((dw.double() - want).abs() <= 6 * EPS * (h.abs() * dy.double()).sum(0)).all()
    del h
    _, _, db = layer_norm_backward(dy, x, mean, rstd, w)
    want = dy.double().sum(0)
    assert ((db.double() - want).abs() <= 2 * EPS * want).all()
