"""The linear layer on the GPU against the float64 oracle on the same (rounded) inputs.

Tolerances.  A product of K terms accumulated in float32 in any order is off by at most
K * 2^-23 * (|x| @ |w|.T) (2^-23 for a matrix instruction that truncates); GELU and its
approximation have slopes below 1.13 and 1.5e-7 |z| of their own (two-byte types), the stored
result adds u |y|, u = eps / 2 of its type.  Backward: dz is rounded once to the operands' type."""
import numpy as np
import pytest
import torch

from mlx_audio_amd.frontends import linear, linear_backward
from oracle import transformer as o

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def f64(t):
    return t.detach().cpu().double().numpy()


def u(t):
    return torch.finfo(t).eps / 2


def tiny(t):
    return torch.finfo(t).tiny * u(t)


def make(shape, t, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(t).cuda()


def check_forward(x, w, b, act, r):
    y, z = linear(x, w, b, activation=act, residual=r, return_preactivation=True)
    t = x.dtype
    xd, wd = f64(x).reshape(-1, x.shape[-1]), f64(w)
    n = w.shape[0]
    want, wz = o.linear(xd, wd, None if b is None else f64(b), act, None if r is None else f64(r).reshape(-1, n))
    acc = (xd.shape[1] + 4) * 2.0 ** -23 * (np.abs(xd) @ np.abs(wd).T + (0 if b is None else np.abs(f64(b))))
    assert y.dtype == z.dtype == t and y.shape == z.shape == x.shape[:-1] + (n,)
    ez = np.abs(f64(z).reshape(-1, n) - wz)
    assert (ez <= u(t) * np.abs(wz) * (1 + 1e-6) + acc + tiny(t)).all(), ez.max()
    ey = np.abs(f64(y).reshape(-1, n) - want)
    # 4e-7 |z|: the polynomial (two-byte) or a few float32 operations of the activation and the sum
    tol = u(t) * np.abs(want) * (1 + 1e-6) + 1.13 * acc + 4e-7 * (np.abs(wz) + np.abs(want)) + tiny(t)
    assert (ey <= tol).all(), np.max(ey / tol)
    assert torch.equal(y, linear(x, w, b, activation=act, residual=r))
    return z


def check_backward(dy, x, w, act, z):
    t = x.dtype
    n, k = w.shape
    dx, dw, db = linear_backward(dy, x, w, activation=act, preactivation=z)
    gd, xd, wd = f64(dy).reshape(-1, n), f64(x).reshape(-1, k), f64(w)
    zd = None if act is None else f64(z).reshape(-1, n)
    ex, ew, eb = o.linear_backward(gd, xd, wd, act, zd)
    dz = gd if act is None else gd * o.derivative(zd, act)
    # the derivative: 1e-6 of its own scale (at most |dy| (1 + |z|)), then one rounding
    ddz = (0 if act is None else 1e-6 * np.abs(gd) * (1 + np.abs(zd)))
    dza = np.abs(dz) + ddz
    edz = (0 if act is None else u(t)) * dza + ddz + tiny(t)
    assert dx.dtype == dw.dtype == t and db.dtype == torch.float32 and dx.shape == x.shape and dw.shape == w.shape
    for got, want, bound in ((dx.reshape(-1, k), ex, edz @ np.abs(wd) + (n + 4) * 2.0 ** -23 * (dza @ np.abs(wd))),
                             (dw, ew, edz.T @ np.abs(xd) + (len(xd) + 4) * 2.0 ** -23 * (dza.T @ np.abs(xd)))):
        err = np.abs(f64(got) - want)
        tol = u(t) * np.abs(want) * (1 + 1e-6) + (1 + u(t)) * bound + tiny(t)
        assert (err <= tol).all(), np.max(err / tol)
    eb_tol = (len(xd) / 4 + 8) * 2.0 ** -24 * dza.sum(0) + (0 if act is None else ddz.sum(0))
    assert (np.abs(f64(db) - eb) <= eb_tol + 1e-30).all()


SHAPES = [(1, 1, 1), (1, 64, 16), (2, 8, 5), (7, 777, 30), (8, 1280, 512), (16, 33, 130), (17, 96, 48), (40, 1280, 250),
          (64, 512, 384), (65, 64, 64), (65, 65, 65), (100, 20, 257), (130, 1280, 1280), (300, 384, 1030),
          (257, 2048, 96), (1, 5120, 1281), (1030, 40, 128), (70, 3, 1000), (66, 4000, 64)]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("m,k,n", SHAPES)
def test_shapes(gpu, t, m, k, n):
    t = TYPES[t]
    x, w = make((m, k), t, m + k), make((n, k), t, n + k, k ** -0.5)
    b, r, dy = make((n,), t, 1, 0.1), make((m, n), t, 2), make((m, n), t, 3)
    act = [None, "gelu", "gelu_tanh", "relu"][(m + n) % 4]
    z = check_forward(x, w, b, act, r)
    check_backward(dy, x, w, act, z)
    check_forward(x, w, None, None, None)
    check_backward(dy, x, w, None, None)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "relu"])
def test_activations(gpu, t, act):
    t = TYPES[t]
    x, w = make((90, 128), t, 4), make((200, 128), t, 5, 0.3)  # preactivations to +-10 and beyond
    z = check_forward(x, w, make((200,), torch.float32, 6), act, None)
    check_forward(x[:9], w, make((200,), torch.float32, 6), act, make((9, 200), t, 7))
    check_backward(make((90, 200), t, 8), x, w, act, z)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("m,k,n", [(4096, 96, 4096), (4100, 64, 4104), (2176, 72, 8200)])
def test_many_tiles(gpu, t, m, k, n):
    """Enough tiles for the largest of the compiled tiles, whole and with edges, all three products."""
    t = TYPES[t]
    x, w, dy = make((m, k), t, 9), make((n, k), t, 10, k ** -0.5), make((m, n), t, 11)
    b = make((n,), t, 12, 0.1)
    check_forward(x, w, b, "gelu", None)
    check_backward(dy, x, w, None, None)
    # the result of the input gradient as wide as the largest tile wants it
    xt, wt = make((m, n), t, 13), make((k, n), t, 14, n ** -0.5)
    check_backward(make((m, k), t, 15), xt, wt, None, None)


@pytest.mark.parametrize("t", TYPES)
def test_views(gpu, t):
    t = TYPES[t]
    base, wbase = make((3, 50, 300), t, 16), make((140, 290), t, 17, 0.06)
    for lo, hi in ((1, 258), (0, 256), (8, 264)):  # odd starts, aligned starts with a padded row
        x, w = base[:, :, lo:hi], wbase[:, lo:hi]
        dy = make((3, 50, 160), t, 18)[:, :, 2:142]
        r = make((3, 50, 150), t, 19)[:, :, 5:145]
        z = check_forward(x, w, None, "gelu", r)
        zv = torch.zeros((3, 50, 143), dtype=t, device="cuda")[:, :, 1:141]
        zv.copy_(z)
        got = linear_backward(dy, x, w, activation="gelu", preactivation=zv)
        want = linear_backward(dy.contiguous(), x.contiguous(), w.contiguous(), activation="gelu", preactivation=z)
        check_backward(dy, x, w, "gelu", zv)
        assert torch.equal(got[2], want[2])
    xt = base.transpose(0, 1)
    assert torch.equal(linear(xt, wbase[:, :280].repeat(1, 2)[:, :300]),
                       linear(xt.contiguous(), wbase[:, :280].repeat(1, 2)[:, :300].contiguous()))
    wt = make((64, 48), t, 20).t()   # weight with its other axis contiguous
    x = make((70, 64), t, 21)
    assert torch.equal(linear(x, wt), linear(x, wt.contiguous()))


def test_no_rows_and_parts(gpu):
    w = make((24, 16), torch.float16, 22)
    x, dy = torch.empty((0, 16), dtype=torch.float16, device="cuda"), torch.empty((0, 24), dtype=torch.float16, device="cuda")
    assert linear(x, w).shape == (0, 24)
    dx, dw, db = linear_backward(dy, x, w)
    assert dx.shape == (0, 16) and (dw == 0).all() and (db == 0).all()
    x, dy = make((80, 16), torch.float16, 23), make((80, 24), torch.float16, 24)
    full = linear_backward(dy, x, w)
    for i, name in enumerate(("input_grad", "weight_grad", "bias_grad")):
        part = linear_backward(dy, x, w, **{name: False})
        assert part[i] is None
        assert all(torch.equal(a, c) for j, (a, c) in enumerate(zip(part, full)) if j != i)


def test_bad_values_stay_in_their_rows(gpu):
    x, w = make((150, 128), torch.float32, 25), make((70, 128), torch.float32, 26, 0.1)
    want = linear(x, w)
    x[3, 4], x[149, 0] = float("nan"), float("inf")
    got = linear(x, w, activation="relu")
    good = [i for i in range(150) if i not in (3, 149)]
    assert torch.equal(got[good], torch.relu(want[good])) and torch.isnan(got[3]).all()
    z = torch.tensor([[float("nan"), 1e30, -1e30, 0.0]], device="cuda")
    for act in ("gelu", "gelu_tanh", "relu"):
        g = linear_backward(torch.ones_like(z), z, torch.eye(4, device="cuda"), activation=act, preactivation=z,
                            weight_grad=False)[2]
        assert torch.isnan(g[0]) and g[1] == 1.0 and g[2] == 0.0 and g[3] == (0.0 if act == "relu" else 0.5)


def test_gradient_against_differences(gpu):
    x, w, b = make((70, 48), torch.float32, 27), make((33, 48), torch.float32, 28, 0.2), make((33,), torch.float32, 29)
    dy = make((70, 33), torch.float32, 30)
    _, z = linear(x, w, b, activation="gelu", return_preactivation=True)
    dx, dw, db = map(f64, linear_backward(dy, x, w, activation="gelu", preactivation=z))
    rng = np.random.default_rng(1)
    ux, uw, ub = rng.standard_normal(x.shape), rng.standard_normal(w.shape), rng.standard_normal(33)
    h = 1e-5
    loss = lambda s: (f64(dy) * o.linear(f64(x) + s * ux, f64(w) + s * uw, f64(b) + s * ub, "gelu")[0]).sum()
    want = (loss(h) - loss(-h)) / (2 * h)
    got = (dx * ux).sum() + (dw * uw).sum() + (db * ub).sum()
    scale = np.abs(dx * ux).sum() + np.abs(dw * uw).sum() + np.abs(db * ub).sum()
    assert abs(got - want) <= 2e-5 * scale   # 74 * 2^-23 from the products, h^2 from the difference


def test_two_calls_give_the_same_bits(gpu):
    x, w = make((3000, 320), torch.bfloat16, 31), make((320, 320), torch.bfloat16, 32, 0.05)
    dy = make((3000, 320), torch.bfloat16, 33)
    z = linear(x, w)
    first = linear_backward(dy, x, w, activation="gelu", preactivation=z)
    for _ in range(3):
        assert all(torch.equal(a, c) for a, c in zip(first, linear_backward(dy, x, w, activation="gelu", preactivation=z)))


def test_rows_beyond_four_gigabytes(gpu):
    """Row offsets that pass 32 bits: the last rows against a call on a copy of them, bit for bit."""
    m, k, n = 2_200_000, 1024, 64
    x = torch.zeros((m, k), dtype=torch.bfloat16, device="cuda")
    x[-300:] = make((300, k), torch.bfloat16, 34)
    w = make((n, k), torch.bfloat16, 35, k ** -0.5)
    y = linear(x, w)
    want, _ = o.linear(f64(x[-300:]), f64(w))
    acc = (k + 4) * 2.0 ** -23 * (np.abs(f64(x[-300:])) @ np.abs(f64(w)).T)
    assert (np.abs(f64(y[-300:]) - want) <= u(torch.bfloat16) * np.abs(want) * (1 + 1e-6) + acc).all()
    assert (y[:-300] == 0).all()
    dx, dw, db = linear_backward(y, x, w)
    assert (dx[:-300] == 0).all() and torch.isfinite(dx[-300:].float()).all() and dx[-1].abs().sum() > 0
    ex, ew, eb = o.linear_backward(f64(y[-300:]), f64(x[-300:]), f64(w))
    dy = np.abs(f64(y[-300:]))
    tol = u(torch.bfloat16) * np.abs(ew) * (1 + 1e-6) + 304 * 2.0 ** -23 * (dy.T @ np.abs(f64(x[-300:]))) + 1e-30
    assert (np.abs(f64(dw) - ew) <= tol).all()
    tol = u(torch.bfloat16) * np.abs(ex) * (1 + 1e-6) + 68 * 2.0 ** -23 * (dy @ np.abs(f64(w))) + 1e-30
    assert (np.abs(f64(dx[-300:]) - ex) <= tol).all()
