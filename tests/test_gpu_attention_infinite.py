"""Infinite values in attention: what the definition makes finite stays finite, at every head dimension.

Tolerances: the bounds of test_gpu_attention on the same call without the key in question, whose
probability is zero."""
import numpy as np
import pytest
import torch

from mlx_audio_amd.frontends import attention, attention_backward
from test_gpu_attention import TYPES, bounds, close, f64, make, u

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("dim", [8, 20, 24, 32, 40, 48, 64, 72, 80, 96, 104, 120, 128, 33])
@pytest.mark.parametrize("sq", [3, 70, 1100])
def test_a_key_of_minus_infinity_is_not_seen(gpu, t, dim, sq):
    """q k^T is -inf for one key: its probability is 0 and the result that of the other keys."""
    t = TYPES[t]
    B, H = (8, 8) if sq > 1000 else (1, 2)
    q, k, v = make((B, sq, H, dim), t, 1).abs(), make((B, 90, H, dim), t, 2), make((B, 90, H, dim), t, 3)
    k[:, 11, :, 0] = float("-inf")
    q[..., 0] += 0.5
    out, lse = attention(q, k, v, return_lse=True)
    out, lse, q, k, v = (x[:1, ..., :] if x is not lse else x[:1] for x in (out, lse, q, k, v))
    keep = [i for i in range(90) if i != 11]
    U = 0.0 if t == torch.float32 else u(t)
    want, wlse, e_out, e_lse, *_ = bounds(f64(q), f64(k[:, keep]), f64(v[:, keep]), np.zeros(q.shape), False, None,
                                          dim ** -0.5, U, u(t), 2.0 ** -25 if t == torch.float16 else 2.0 ** -125)
    close(out, want, e_out, t, "out")
    assert (np.abs(f64(lse) - wlse) <= e_lse + 1e-7).all()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("dim", [20, 48, 64, 80])
def test_infinite_values_stay_in_their_columns(gpu, t, dim):
    t = TYPES[t]
    q, k, v = make((2, 70, 2, dim), t, 4), make((2, 90, 2, dim), t, 5), make((2, 90, 2, dim), t, 6)
    want = attention(q, k, v)
    v[0, 5, 1, 2] = float("inf")
    out = attention(q, k, v)
    assert (out[0, :, 1, 2] == float("inf")).all()
    out[0, :, 1, 2] = want[0, :, 1, 2]
    assert torch.equal(out, want)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
@pytest.mark.parametrize("sq", [5, 300])
def test_gradients_behind_a_length_are_zero_whatever_dout_holds(gpu, t, bad, sq):
    t = TYPES[t]
    lengths = [1, 37, 64, 65, 150, 0]
    q, k, v = make((6, sq, 4, 64), t, 7), make((6, 150, 2, 64), t, 8), make((6, 150, 2, 64), t, 9)
    dout = make(q.shape, t, 10)
    out, lse = attention(q, k, v, key_lengths=lengths, return_lse=True)
    good = attention_backward(dout, q, k, v, out, lse, key_lengths=lengths)
    dout[:, sq // 2, 1, 3] = bad
    got = attention_backward(dout, q, k, v, out, lse, key_lengths=lengths)
    for b, n in enumerate(lengths):
        assert all((g[b, n:] == 0).all() for g in got[1:]), b
    # the query's own row of dq and its key head are spoilt, nothing else (float16: but for the scale)
    assert torch.equal(got[0][:, :, 2:], good[0][:, :, 2:]) if t != torch.float16 else torch.isfinite(got[0][:, :, 2:]).all()
    assert all(torch.isfinite(g[:, :, 1]).all() for g in got[1:])
