"""GELU and its derivative far from zero, relative to their own size.

With an identity matrix as weight the value before the activation is x itself.  Tolerance: Phi(x) comes
from exp(-x^2 / 2) times a function fitted to 7.2e-7 of its value; the exponent's argument, up to
x^2 / 2 log2(e) = 120 at 12.9, is off by 3 roundings of 2^-24 of it, 120 ln 2 3 2^-24 = 1.5e-5, and the rest
is below 2e-6 (float32 takes the library's erfc of an argument rounded twice: 2 x^2 / 2 2 2^-24 = 2e-5).
So 2^-15 = 3.1e-5 of the value, besides the stored result's rounding."""
import numpy as np
import pytest
import torch

from mlx_audio_amd.frontends import linear, linear_backward
from oracle import transformer as o
from test_gpu_linear import TYPES, f64, tiny, u

pytestmark = pytest.mark.gpu
REL = 2.0 ** -15


def arguments(rows, t):
    x = np.linspace(-12.9, 6.0, rows * 64)
    return torch.from_numpy(x).to(t).view(rows, 64).cuda()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows", [16, 60, 700, 6000])
def test_gelu(gpu, t, rows):
    x = arguments(rows, TYPES[t])
    want = o.activate(f64(x), "gelu")
    err = np.abs(f64(linear(x, torch.eye(64, dtype=x.dtype, device="cuda"), activation="gelu")) - want)
    tol = (u(x.dtype) + REL) * np.abs(want) + tiny(x.dtype)
    assert (err <= tol).all(), (np.max(err / tol), f64(x).flat[np.argmax(err / tol)])


@pytest.mark.parametrize("t", TYPES)
def test_gelu_derivative(gpu, t):
    z = arguments(700, TYPES[t])
    eye = torch.eye(64, dtype=z.dtype, device="cuda")
    dx, dw, db = linear_backward(torch.ones_like(z), z, eye, activation="gelu", preactivation=z)
    zd = f64(z)
    want = o.derivative(zd, "gelu")
    # the two terms' errors where they cancel; the slope is rounded once, as dz, and dx is dz
    size = np.abs(want) + 2 * np.abs(zd) * np.exp(-0.5 * zd * zd) / np.sqrt(2 * np.pi)
    tol = u(z.dtype) * np.abs(want) * (1 + 1e-6) + (1 + u(z.dtype)) * REL * size + tiny(z.dtype)
    err = np.abs(f64(dx) - want)
    assert (err <= tol).all(), (np.max(err / tol), zd.flat[np.argmax(err / tol)])
    assert (np.abs(f64(db) - want.sum(0)) <= (REL + 700 * 2.0 ** -24) * size.sum(0)).all()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "relu"])
def test_slope_at_infinite_preactivations(gpu, t, act):
    """What the forward call keeps may be infinite (float16: beyond 65504) where its result is not: the slope
    there is the limit, 0 or 1."""
    t = TYPES[t]
    inf = float("inf")
    z = torch.tensor([[-inf, inf, -6e4, 6e4, float("nan")]], device="cuda").to(t)
    eye = torch.eye(5, dtype=t, device="cuda")
    db = linear_backward(torch.ones_like(z), z[:, :5], eye, activation=act, preactivation=z, input_grad=False,
                         weight_grad=False)[2]
    assert db[:4].tolist() == [0.0, 1.0, 0.0, 1.0] and torch.isnan(db[4])
    x = torch.full((70, 5), 300.0, dtype=t, device="cuda")
    w = torch.full((4, 5), -250.0, dtype=t, device="cuda")      # preactivation -375 000
    y, kept = linear(x, w, activation=act, return_preactivation=True)
    assert (y == 0).all() and (t != torch.float16 or torch.isinf(kept).all())
    dx, dw, db = linear_backward(torch.ones_like(y), x, w, activation=act, preactivation=kept)
    assert (dx == 0).all() and (dw == 0).all() and (db == 0).all()
