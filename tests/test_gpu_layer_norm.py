"""Layer normalisation on the GPU against the float64 oracle on the same (rounded) inputs.

Tolerances.  u = eps / 2 of the stored type.  A row's sums are trees of at most 64 float32 additions
per thread and eight joins, so mean and sum of squares are off by at most 72 * 2^-24 relative to the
sums of magnitudes; each result passes a handful of further float32 operations.  E = 100 * 2^-24
times the magnitudes that enter bounds them all; the stored result adds u |y|."""
import numpy as np
import pytest
import torch

from mlx_audio_amd.frontends import layer_norm, layer_norm_backward
from oracle import transformer as o

pytestmark = pytest.mark.gpu

E = 100 * 2.0 ** -24
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def f64(t):
    return t.detach().cpu().double().numpy()


def u(t):
    return torch.finfo(t).eps / 2


def tiny(t):  # half a step of the smallest (subnormal) values
    return torch.finfo(t).tiny * u(t)


def make(shape, t, seed, offset=0.5, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale + offset).to(t).cuda()


def check_forward(x, w, b, eps=1e-5, **kw):
    y, mean, rstd = layer_norm(x, w, b, eps, return_stats=True)
    wd, bd = (None if v is None else f64(v) for v in (w, b))
    want, wmean, wrstd = o.layer_norm(f64(x), wd, bd, eps)
    xa = np.abs(f64(x))
    top = xa.max(-1, keepdims=True) if x.numel() else xa
    assert y.dtype == x.dtype and y.shape == x.shape and mean.shape == x.shape[:-1] == rstd.shape
    assert (np.abs(f64(mean) - wmean) <= E * top[..., 0]).all()
    # the variance's relative error: E on the sum of squares, 2 E top / sd on the centred values
    rel = E * (1 + 2 * top[..., 0] * wrstd)
    assert (np.abs(f64(rstd) - wrstd) <= rel * wrstd).all()
    mag = (xa + top) * wrstd[..., None] * (1.0 if wd is None else np.abs(wd)) * (1 + rel[..., None] / E * 0.5)
    tol = u(x.dtype) * np.abs(want) + E * (mag + (0.0 if bd is None else np.abs(bd))) + tiny(x.dtype)
    assert (np.abs(f64(y) - want) <= tol).all(), np.max(np.abs(f64(y) - want) / tol)
    return y, mean, rstd


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows,dim", [(1, 1), (3, 2), (5, 7), (9, 64), (4, 100), (33, 384), (1500, 512), (70, 513),
                                      (40, 768), (17, 1024), (200, 1280), (11, 1281), (6, 1537), (10, 2048), (10, 2049),
                                      (7, 4096), (5, 5000), (3, 8192), (3, 8193), (2, 20001)])
def test_forward_and_backward(gpu, t, rows, dim):
    t = TYPES[t]
    x, dy = make((rows, dim), t, rows + dim), make((rows, dim), t, 1 + rows + dim, 0.0)
    w, b = make((dim,), t, 2, 1.0, 0.1), make((dim,), t, 3, 0.0, 0.1)
    _, mean, rstd = check_forward(x, w, b)
    dx, dw, db = layer_norm_backward(dy, x, mean, rstd, w)
    xd, gd, wd, md, rd = f64(x), f64(dy), f64(w), f64(mean), f64(rstd)
    ex, ew, eb = o.layer_norm_backward(gd, xd, md, rd, wd)
    h = np.abs((xd - md[:, None]) * rd[:, None]) + (np.abs(xd) + np.abs(md)[:, None]) * rd[:, None] * E
    g = np.abs(gd * wd)
    mag = rd[:, None] * (g + g.mean(-1, keepdims=True) + h * (g * h).mean(-1, keepdims=True))
    # h itself is off by E (|x| + |mean|) rstd, which reaches dx through the last product
    mag += rd[:, None] * (np.abs(xd) + np.abs(md)[:, None]) * rd[:, None] * (g * (1 + h)).mean(-1, keepdims=True)
    tol = u(t) * np.abs(ex) + 2 * E * mag + tiny(t)
    assert dx.dtype == t and (np.abs(f64(dx) - ex) <= tol).all(), np.max(np.abs(f64(dx) - ex) / tol)
    # column sums: at most rows / 4 + 4 float32 additions in one chain, the join in double
    chain = (rows / 4 + 8) * 2.0 ** -24
    ha = h + (np.abs(xd) + np.abs(md)[:, None]) * rd[:, None] * 2.0 ** -22
    assert dw.dtype == db.dtype == torch.float32
    assert (np.abs(f64(dw) - ew) <= (chain + 2.0 ** -20) * (np.abs(gd) * ha).sum(0) + 1e-30).all()
    assert (np.abs(f64(db) - eb) <= (chain + 2.0 ** -23) * np.abs(gd).sum(0) + 1e-30).all()


@pytest.mark.parametrize("t", ["f16", "bf16"])
def test_float32_parameters_with_two_byte_rows(gpu, t):
    t = TYPES[t]
    x = make((37, 1280), t, 5)
    w, b = make((1280,), torch.float32, 6, 1.0, 0.1), make((1280,), torch.float32, 7, 0.0, 0.1)
    _, mean, rstd = check_forward(x, w, b)
    check_forward(x, w, None)
    check_forward(x, None, b)
    check_forward(x, None, None)
    dx, dw, db = layer_norm_backward(x, x, mean, rstd)
    assert dw is None and db is None
    one = torch.ones_like(w)
    assert torch.equal(dx, layer_norm_backward(x, x, mean, rstd, one)[0])


def test_views_leading_axes_and_odd_alignment(gpu):
    base = make((5, 9, 1300), torch.bfloat16, 8)
    w, b = make((1279,), torch.bfloat16, 9, 1.0, 0.1), make((1279,), torch.bfloat16, 10, 0.0, 0.1)
    x = base[:, :, 1:1280]                   # rows of stride 1300 that start at odd elements
    y, mean, rstd = check_forward(x, w, b)
    assert torch.equal(y, layer_norm(x.contiguous(), w, b))
    dy = base[:, :, 3:1282]
    got = layer_norm_backward(dy, x, mean, rstd, w)
    want = layer_norm_backward(dy.contiguous(), x.contiguous(), mean, rstd, w)
    assert all(torch.equal(a, c) for a, c in zip(got, want))
    xt = base.transpose(0, 1)                # leading axes that do not collapse
    assert torch.equal(layer_norm(xt), layer_norm(xt.contiguous()))
    xs = base.transpose(1, 2)                # last axis not contiguous
    assert torch.equal(layer_norm(xs), layer_norm(xs.contiguous()))
    row = base[0, 0, :640].expand(4, 640)    # one row read four times
    assert torch.equal(layer_norm(row), layer_norm(row.contiguous()))


def test_rows_far_from_zero_and_constant_rows(gpu):
    x = make((8, 1024), torch.float32, 11, offset=1000.0, scale=0.5)
    check_forward(x, None, None)
    y, mean, rstd = layer_norm(torch.full((3, 640), 2.5, device="cuda"), eps=1e-5, return_stats=True)
    assert (y == 0).all() and (mean == 2.5).all() and torch.allclose(rstd, torch.full_like(rstd, 1e-5 ** -0.5))


def test_no_rows(gpu):
    x = torch.empty((0, 4, 64), device="cuda")
    y, mean, rstd = layer_norm(x, torch.ones(64, device="cuda"), return_stats=True)
    assert y.shape == x.shape and mean.shape == (0, 4)
    dx, dw, db = layer_norm_backward(x, x, mean, rstd, torch.ones(64, device="cuda"))
    assert dx.shape == x.shape and (dw == 0).all() and (db == 0).all()


def test_one_bad_row_stays_alone(gpu):
    x = make((6, 1280), torch.float32, 12)
    x[2, 5], x[4, 7] = float("nan"), float("inf")
    y = layer_norm(x)
    assert torch.isnan(y[2]).all() and torch.isnan(y[4]).all() and torch.isfinite(y[[0, 1, 3, 5]]).all()


def test_gradient_against_differences(gpu):
    """The directional derivative of sum(dy * y): central differences of the float64 oracle on the
    kernel's own inputs against the kernel's gradients (float32)."""
    x, dy = make((7, 300), torch.float32, 13), make((7, 300), torch.float32, 14, 0.0)
    w, b = make((300,), torch.float32, 15, 1.0, 0.1), make((300,), torch.float32, 16, 0.0, 0.1)
    _, mean, rstd = layer_norm(x, w, b, return_stats=True)
    dx, dw, db = map(f64, layer_norm_backward(dy, x, mean, rstd, w))
    rng = np.random.default_rng(0)
    ux, uw, ub = rng.standard_normal(x.shape), rng.standard_normal(300), rng.standard_normal(300)
    h = 1e-5
    loss = lambda s: (f64(dy) * o.layer_norm(f64(x) + s * ux, f64(w) + s * uw, f64(b) + s * ub)[0]).sum()
    want = (loss(h) - loss(-h)) / (2 * h)
    got = (dx * ux).sum() + (dw * uw).sum() + (db * ub).sum()
    scale = np.abs(dx * ux).sum() + np.abs(dw * uw).sum() + np.abs(db * ub).sum()
    assert abs(got - want) <= 1e-5 * scale   # 2 E from the kernel, h^2 from the difference


def test_two_calls_give_the_same_bits(gpu):
    x, dy = make((4099, 640), torch.float16, 17), make((4099, 640), torch.float16, 18)
    w = make((640,), torch.float16, 19)
    _, mean, rstd = layer_norm(x, w, return_stats=True)
    first = layer_norm_backward(dy, x, mean, rstd, w)
    for _ in range(3):
        assert all(torch.equal(a, c) for a, c in zip(first, layer_norm_backward(dy, x, mean, rstd, w)))


def test_rows_beyond_four_gigabytes(gpu):
    m, n = 2_200_000, 1024
    x = torch.zeros((m, n), dtype=torch.bfloat16, device="cuda")
    x[-5:] = make((5, n), torch.bfloat16, 20)
    w = make((n,), torch.bfloat16, 21, 1.0, 0.1)
    y, mean, rstd = layer_norm(x, w, return_stats=True)
    want = layer_norm(x[-5:].clone(), w, return_stats=True)
    assert all(torch.equal(a[-5:], c) for a, c in zip((y, mean, rstd), want)) and (y[:-5] == 0).all()
    dx, dw, db = layer_norm_backward(y, x, mean, rstd, w)
    ref = layer_norm_backward(y[-5:].clone(), x[-5:].clone(), mean[-5:], rstd[-5:], w)
    assert torch.equal(dx[-5:], ref[0]) and (dx[:-5] == 0).all()
    # five rows that are not zero, added in another order: 4 * 2^-24 of their magnitudes
    h = (f64(x[-5:]) - f64(mean[-5:])[:, None]) * f64(rstd[-5:])[:, None]
    assert (np.abs(f64(dw) - f64(ref[1])) <= 8 * 2.0 ** -24 * np.abs(f64(y[-5:]) * h).sum(0) + 1e-30).all()
    assert (np.abs(f64(db) - f64(ref[2])) <= 8 * 2.0 ** -24 * np.abs(f64(y[-5:])).sum(0) + 1e-30).all()
