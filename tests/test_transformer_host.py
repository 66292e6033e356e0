"""Refusals of the operators behind the encoder stem (no GPU needed: arguments are checked before any
device work), and the oracle against torch in float64."""
import ctypes

import numpy as np
import pytest
import torch

from mlx_audio_amd import _lib, frontends as f
from oracle import transformer as o

E = torch.empty


def test_layer_norm_refuses():
    x = E(4, 8)
    for bad in (dict(x=x.double()), dict(x=x.int()), dict(x=E(4, 0)), dict(x=E(()))):
        with pytest.raises(ValueError):
            f.layer_norm(**bad)
    with pytest.raises(ValueError, match=r"weight must have shape \(8,\)"):
        f.layer_norm(x, E(7))
    with pytest.raises(ValueError, match="bias must be float32 or torch.float16"):
        f.layer_norm(x.half(), None, E(8, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="expected one type"):
        f.layer_norm(x.half(), E(8), E(8).half())
    for eps in (-1e-5, float("nan")):
        with pytest.raises(ValueError, match="eps"):
            f.layer_norm(x, eps=eps)
    with pytest.raises(ValueError, match="dy must have x's shape"):
        f.layer_norm_backward(E(4, 7), x, E(4), E(4))
    with pytest.raises(ValueError, match="expected one type"):
        f.layer_norm_backward(x.half(), x, E(4), E(4))
    with pytest.raises(ValueError, match="mean must be float32"):
        f.layer_norm_backward(x, x, E(4).half(), E(4))
    with pytest.raises(ValueError, match="rstd must be float32"):
        f.layer_norm_backward(x, x, E(4), E(3))


def test_linear_refuses():
    x, w = E(4, 8), E(5, 8)
    with pytest.raises(ValueError, match="Unknown activation"):
        f.linear(x, w, activation="swish")
    with pytest.raises(ValueError, match="weight must be"):
        f.linear(x, E(8))
    with pytest.raises(ValueError, match="weight must be"):
        f.linear(E(4, 0), E(5, 0))
    with pytest.raises(ValueError, match="last axis of 8"):
        f.linear(E(4, 7), w)
    with pytest.raises(ValueError, match="expected one type"):
        f.linear(x.half(), w)
    with pytest.raises(ValueError, match="bias must have shape"):
        f.linear(x, w, E(4))
    with pytest.raises(ValueError, match="bias must be float32"):
        f.linear(x, w, E(5).half())
    with pytest.raises(ValueError, match="residual must have shape"):
        f.linear(x, w, residual=E(4, 8))
    with pytest.raises(ValueError, match="needs the preactivation"):
        f.linear_backward(E(4, 5), x, w, activation="gelu")
    with pytest.raises(ValueError, match="dy must have shape"):
        f.linear_backward(E(4, 8), x, w)
    with pytest.raises(ValueError, match="preactivation must have shape"):
        f.linear_backward(E(4, 5), x, w, activation="relu", preactivation=E(4, 4))


def test_attention_refuses():
    q, k = E(2, 3, 4, 16), E(2, 5, 2, 16)
    for bad in ((E(3, 4, 16), k, k), (q, k, E(2, 5, 2, 8)), (q, E(1, 5, 2, 16), E(1, 5, 2, 16)),
                (q, E(2, 5, 3, 16), E(2, 5, 3, 16)), (q, E(2, 5, 0, 16), E(2, 5, 0, 16)), (q.half(), k, k),
                (E(2, 3, 4, 0), E(2, 5, 2, 0), E(2, 5, 2, 0))):
        with pytest.raises(ValueError):
            f.attention(*bad)
    with pytest.raises(NotImplementedError, match="128"):
        f.attention(E(1, 2, 1, 129), E(1, 2, 1, 129), E(1, 2, 1, 129))
    for scale in (0.0, -1.0, float("inf"), float("nan")):
        with pytest.raises(ValueError, match="scale"):
            f.attention(q, k, k, scale=scale)
    for lengths in ([1], [1, 6], [-1, 2], [1.0, 2.0], [[1], [2]], [True, False]):
        with pytest.raises(ValueError, match="key_lengths"):
            f.attention(q, k, k, key_lengths=lengths)
    lse = E(2, 4, 3)
    with pytest.raises(ValueError, match="dout must have q's shape"):
        f.attention_backward(k, q, k, k, q, lse)
    with pytest.raises(ValueError, match="lse must be float32"):
        f.attention_backward(q, q, k, k, q, lse.transpose(1, 2))
    with pytest.raises(ValueError, match="expected one type"):
        f.attention_backward(q, q, k, k, q.half(), lse)


def test_a_gradient_is_never_lost_silently():
    x, w = E(4, 8), E(5, 8, requires_grad=True)
    with pytest.raises(RuntimeError, match="requires a gradient"):
        f.linear(x, w)
    with pytest.raises(RuntimeError, match="requires a gradient"):
        f.layer_norm(x.requires_grad_())
    if not torch.cuda.is_available():
        with torch.no_grad(), pytest.raises(RuntimeError, match="no CPU fallback"):
            f.linear(x, w)


@pytest.mark.skipif(torch.cuda.is_available(), reason="only meaningful on a machine without a GPU")
def test_no_cpu_fallback():
    x = E(4, 8)
    q = E(1, 2, 1, 8)
    for call in (lambda: f.layer_norm(x), lambda: f.layer_norm_backward(x, x, E(4), E(4)), lambda: f.linear(x, x),
                 lambda: f.linear_backward(E(4, 4), x, x), lambda: f.attention(q, q, q),
                 lambda: f.attention_backward(q, q, q, q, q, E(1, 1, 2))):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()


def test_c_entries_check_their_arguments():
    """Every call here ends in the argument checks, in front of any device work."""
    lib = _lib.lib()
    p = ctypes.c_void_p(256)

    def norm(rows=2, dim=8, stride=8, dtype=0, x=p, y=p, mean=None, rstd=None, eps=1e-5, w=None, pd=0):
        return lib.mia_layer_norm(x, rows, dim, stride, dtype, w, None, pd, eps, y, mean, rstd, None)

    for bad in (dict(rows=-1), dict(dim=0), dict(dtype=3), dict(x=None), dict(y=None), dict(mean=p), dict(eps=-1.0),
                dict(stride=-8), dict(w=p, pd=1), dict(rows=1 << 31)):
        assert norm(**bad) == _lib.MIA_ERR_INVALID, bad
    assert norm(rows=0) == _lib.MIA_OK
    assert lib.mia_layer_norm_backward(p, 8, p, 8, p, p, 2, 8, 0, p, 0, p, p, p, None, 0, None) == _lib.MIA_ERR_INVALID
    assert b"workspace" in lib.mia_last_error()

    def linear(rows=100, k=8, n=8, act=0, dtype=0, x=p, w=p, y=p, ws=None, need=0, bias=None, bd=0):
        return lib.mia_linear(x, k, w, k, bias, bd, None, 0, act, rows, k, n, dtype, y, None, ws, need, None)

    for bad in (dict(rows=-1), dict(k=0), dict(n=0), dict(act=4), dict(dtype=-1), dict(x=None), dict(w=None), dict(y=None),
                dict(bias=p, bd=2)):
        assert linear(**bad) == _lib.MIA_ERR_INVALID, bad
    assert linear(rows=0) == _lib.MIA_OK
    assert linear(rows=1 << 31) == _lib.MIA_ERR_UNSUPPORTED
    need = lib.mia_linear_workspace_bytes(100, 5120, 64, 2)
    assert need > 0 and linear(k=5120, n=64, dtype=2) == _lib.MIA_ERR_INVALID
    assert lib.mia_linear_backward(p, 8, p, 8, p, 8, None, 0, 1, 4, 8, 8, 0, p, p, p, p, 1 << 30, None) == _lib.MIA_ERR_INVALID

    def desc(**kw):
        d = dict(dtype=0, batch=1, queries=2, keys=3, heads=4, kv_heads=2, dim=16, causal=0, scale=0.25)
        d.update(kw)
        s = (ctypes.c_int64 * 3)(*d.pop("strides", (1, 1, 1)))
        return _lib.AttentionDesc(**d, stride_q=s, stride_k=s, stride_v=s)

    def attention(q=p, out=p, **kw):
        return lib.mia_attention(ctypes.byref(desc(**kw)), q, p, p, None, out, None, None, 0, None)

    for bad in (dict(dtype=5), dict(batch=-1), dict(heads=3), dict(kv_heads=0), dict(dim=0), dict(scale=0.0), dict(q=None),
                dict(out=None), dict(strides=(1, -1, 1)), dict(scale=float("inf"))):
        assert attention(**bad) == _lib.MIA_ERR_INVALID, bad
    for bad in (dict(dim=129), dict(batch=1 << 30, heads=64), dict(queries=1 << 31)):
        assert attention(**bad) == _lib.MIA_ERR_UNSUPPORTED, bad
    assert attention(batch=0) == _lib.MIA_OK and attention(queries=0) == _lib.MIA_OK
    assert attention(keys=100000) == _lib.MIA_ERR_INVALID   # split along the keys: needs a workspace


def test_workspace_sizes():
    lib = _lib.lib()
    assert lib.mia_layer_norm_backward_workspace_bytes(0, 8) == 0
    assert lib.mia_layer_norm_backward_workspace_bytes(3, 8) == 3 * 2 * 8 * 4
    assert lib.mia_linear_workspace_bytes(8, 1280, 5120, 2) == 0
    assert lib.mia_linear_workspace_bytes(0, 1280, 5120, 2) == 0
    assert lib.mia_linear_backward_workspace_bytes(0, 8, 8, 0, 1) == 0


def test_oracle_against_torch():
    g = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(s, generator=g, dtype=torch.float64, requires_grad=True)
    x, w, b = r(7, 12), r(12), r(12)
    y = torch.nn.functional.layer_norm(x, (12,), w, b, 1e-5)
    got = o.layer_norm(*(t.detach().numpy() for t in (x, w, b)))
    assert np.abs(got[0] - y.detach().numpy()).max() < 1e-12
    dy = r(7, 12).detach()
    y.backward(dy)
    grads = o.layer_norm_backward(dy.numpy(), x.detach().numpy(), got[1], got[2], w.detach().numpy())
    for a, t in zip(grads, (x, w, b)):
        assert np.abs(a - t.grad.numpy()).max() < 1e-11
    for act, fn in ((None, lambda z: z), ("gelu", torch.nn.functional.gelu), ("relu", torch.relu),
                    ("gelu_tanh", lambda z: torch.nn.functional.gelu(z, approximate="tanh"))):
        x, w, b = r(9, 6), r(5, 6), r(5)
        y = fn(torch.nn.functional.linear(x, w, b))
        want, z = o.linear(*(t.detach().numpy() for t in (x, w, b)), act)
        assert np.abs(want - y.detach().numpy()).max() < 1e-12
        dy = r(9, 5).detach()
        y.backward(dy)
        for a, t in zip(o.linear_backward(dy.numpy(), x.detach().numpy(), w.detach().numpy(), act, z), (x, w, b)):
            assert np.abs(a - t.grad.numpy()).max() < 1e-11
    q, k, v = r(2, 5, 4, 8), r(2, 7, 2, 8), r(2, 7, 2, 8)
    s = torch.einsum("bihd,bjhd->bhij", q, k.repeat_interleave(2, 2)) / 8 ** 0.5
    seen = torch.arange(7)[None, :] <= torch.arange(5)[:, None] + 2
    seen = seen & (torch.arange(7) < torch.tensor([7, 4])[:, None])[:, None, None]
    p = torch.softmax(s.masked_fill(~seen, float("-inf")), -1)
    out = torch.einsum("bhij,bjhd->bihd", p, v.repeat_interleave(2, 2))
    nq, nk, nv = (t.detach().numpy() for t in (q, k, v))
    got, lse = o.attention(nq, nk, nv, True, [7, 4])
    assert np.abs(got - out.detach().numpy()).max() < 1e-12
    assert np.abs(lse - torch.logsumexp(s.masked_fill(~seen, float("-inf")), -1).detach().numpy()).max() < 1e-12
    dout = r(2, 5, 4, 8).detach()
    out.backward(dout)
    for a, t in zip(o.attention_backward(dout.numpy(), nq, nk, nv, True, [7, 4]), (q, k, v)):
        assert np.abs(a - t.grad.numpy()).max() < 1e-11
