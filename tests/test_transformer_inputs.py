"""Inputs that the operators behind the encoder stem must take as they mean, or refuse (no GPU needed)."""
import ctypes

import pytest
import torch
from torch.autograd import forward_ad

from mlx_audio_amd import _lib, frontends as f
from mlx_audio_amd.frontends import transformer


@pytest.mark.parametrize("sizes", [(0, 5, 7), (1, 0, 7), (1, 5, 0), (0, 0, 0), (3, 1, 1), (2, 1500, 1500)])
def test_workspaces_of_attention_backward(sizes):
    """Sizes of zero too; float16 keeps its norms there beside what the other two-byte type keeps."""
    batch, queries, keys = sizes
    s = (ctypes.c_int64 * 3)(1, 1, 1)
    need = [_lib.lib().mia_attention_backward_workspace_bytes(ctypes.byref(
        _lib.AttentionDesc(t, batch, queries, keys, 4, 2, 16, 0, 0.25, s, s, s))) for t in (_lib.F16, _lib.BF16)]
    assert (need[0] > need[1]) == (batch > 0)


def calls(x):
    """Every operator with x as one of its arguments."""
    q = x.reshape(1, 2, 2, 8)
    plain, norm = torch.randn(4, 8), torch.randn(4)
    p = plain.reshape(1, 2, 2, 8)
    lse = torch.randn(1, 2, 2)
    return [lambda: f.layer_norm(x), lambda: f.layer_norm(plain, x.reshape(-1)[:8]), lambda: f.layer_norm_backward(x, plain, norm, norm),
            lambda: f.linear(x, plain), lambda: f.linear(plain, x), lambda: f.linear(plain, torch.randn(8, 8), residual=x),
            lambda: f.linear_backward(torch.randn(4, 4), x, plain), lambda: f.attention(q, p, p), lambda: f.attention(p, p, q),
            lambda: f.attention_backward(q, p, p, p, p, lse)]


def test_a_tangent_is_never_lost_silently():
    with forward_ad.dual_level():
        x = forward_ad.make_dual(torch.randn(4, 8), torch.randn(4, 8))
        for call in calls(x):
            with torch.no_grad(), pytest.raises(RuntimeError, match="carries a tangent"):
                call()
        if not torch.cuda.is_available():  # plain tensors inside a level, and a dual's primal, are taken
            for call in calls(torch.randn(4, 8)) + calls(forward_ad.unpack_dual(x).primal):
                with pytest.raises(RuntimeError, match="no CPU fallback"):
                    call()


def test_negated_views_are_taken_as_what_they_mean():
    """The imaginary part of a conjugate is a view of the stored values with the sign pending."""
    z = torch.randn(6, 1, dtype=torch.complex64)
    view = z.conj().imag
    assert view.is_neg() and view.stride(-1) != 0
    got = transformer._operands(x=view, weight=view[0])
    assert not any(t.is_neg() for t in got.values())
    assert torch.equal(got["x"], -z.imag) and torch.equal(got["weight"], -z.imag[0])
