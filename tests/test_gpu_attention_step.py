"""Attention with at most 64 queries loses nothing to the rounding of p in the forward pass and of ds in dq.

They go through the matrix units as their rounded value and the rest, itself rounded: with u = eps / 2 of the
type the rest is at most u p and its rounding at most u u p, or 2^-25 / 2^-126 of float16 / bfloat16 below
their normal range.  So the bounds of test_gpu_attention hold with u u in place of u; the second product
doubles the additions in float32: (Sk + 8) 2^-23 more."""
import pytest
import torch

from mlx_audio_amd.frontends import attention, attention_backward
from oracle import transformer as o
from test_gpu_attention import bounds, close, f64, make, u

pytestmark = pytest.mark.gpu
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
SHAPES = [  # batch, queries, keys, heads, key heads, dim
    (1, 1, 2, 16, 16, 64), (4, 1, 65, 8, 8, 64), (2, 1, 700, 8, 1, 128), (3, 1, 1500, 4, 4, 64), (2, 7, 65, 8, 4, 48),
    (2, 64, 64, 2, 2, 64), (1, 8, 300, 8, 1, 33), (2, 16, 20, 4, 2, 96)]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_result_is_rounded_once(gpu, t, causal, shape):
    B, Sq, Sk, H, Hk, D = shape
    t = TYPES[t]
    q, k, v = make((B, Sq, H, D), t, 11), make((B, Sk, Hk, D), t, 12), make((B, Sk, Hk, D), t, 13)
    got = attention(q, k, v, causal=causal)
    zero = f64(q) * 0.0
    want, _, error, *_ = bounds(f64(q), f64(k), f64(v), zero, causal, None, D ** -0.5, u(t) ** 2 + Sk * 2.0 ** -23, u(t),
                                2.0 ** -25 if t == torch.float16 else 2.0 ** -125)
    close(got, want, error, t, "out")


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("shape", SHAPES + [(1, 64, 2000, 16, 16, 64), (2, 64, 130, 4, 1, 127)])
def test_query_gradient_is_rounded_once(gpu, t, causal, shape):
    B, Sq, Sk, H, Hk, D = shape
    t = TYPES[t]
    q, k, v = make((B, Sq, H, D), t, 21), make((B, Sk, Hk, D), t, 22), make((B, Sk, Hk, D), t, 23)
    dout = make((B, Sq, H, D), t, 24)
    out, lse = attention(q, k, v, causal=causal, return_lse=True)
    got = attention_backward(dout, q, k, v, out, lse, causal=causal)[0]
    arrays = [f64(x) for x in (q, k, v, dout)]
    error = bounds(*arrays, causal, None, D ** -0.5, u(t) ** 2 + (Sk + 8) * 2.0 ** -23, u(t),
                   2.0 ** -25 if t == torch.float16 else 2.0 ** -125)[4]
    close(got, o.attention_backward(arrays[3], *arrays[:3], causal, None, D ** -0.5)[0], error, t, "dq")
