"""Attention on the GPU against the float64 oracle on the same (rounded) inputs.

Tolerances.  u = eps / 2 of the operands' type, U = u for two-byte types (p and ds are rounded once
to it before the products that read them), 0 for float32.  With S = scale |q| . |k| (products of
magnitudes) a score is off by at most ds_ = (D + 4) 2^-23 S, plus 4 2^-24 |s| from the exponent's
argument; p then by e = that (relative) + 2^-20 for the exponential and the running sum over at
most Sk / 4 additions per lane (Sk 2^-24 / 4).  out: |error| <= (U + 2 e + Sk 2^-23) sum p |v|, plus
u |out|.  Gradients: the same relative errors on the sums of magnitudes, with ds = p (dp - delta)
bounded by p (|dout| . |v| + |dout| . |out|) and out rounded to the type (u) in delta.

float16 below 2^-14 is a multiple of 2^-24, so a rounding there is off by up to 2^-25 whatever the
value: A = 2^-25 for each p and ds of a float16 product, A sum |v| (|dout|, |k|, |q|) over the terms of
the result.  (The first run lacked this term: probabilities of 1500 keys are around 2^-11 and many
below 2^-14.  The forward's p are relative to the row's largest, whose own p is 1, so dividing by
the sum only makes the term smaller.  The exponential instruction returns 0
below 2^-126, and so may the other types' rounding: A = 2^-125 for float32 and bfloat16, whose
exponents go no further - also missing in the first run, where scores of +-300 make such p.)"""
import numpy as np
import pytest
import torch

from mlx_audio_amd.frontends import attention, attention_backward
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


def bounds(q, k, v, dout, causal, lengths, scale, U, ut, A):
    """Bounds of the errors of (out, lse, dq, dk, dv) before the stored rounding."""
    B, Sq, H, D = q.shape
    Sk, group = k.shape[1], H // k.shape[2]
    out, lse = o.attention(q, k, v, causal, lengths, scale)
    e_out, e_lse = np.zeros(q.shape), np.zeros((B, H, Sq))
    e_dq, e_dk, e_dv = np.zeros(q.shape), np.zeros(k.shape), np.zeros(v.shape)
    for b in range(B):
        seen = o._visible(Sq, Sk, causal, Sk if lengths is None else lengths[b])
        for h in range(H):
            hk = h // group
            kk, vv = np.where(np.isfinite(k[b, :, hk]), k[b, :, hk], 0), np.where(np.isfinite(v[b, :, hk]), v[b, :, hk], 0)
            qq, do, oo = q[b, :, h], dout[b, :, h], out[b, :, h]
            s = scale * (qq @ kk.T)
            rows = np.isfinite(lse[b, h])
            p = np.where(seen & rows[:, None], np.exp(s - np.where(rows, lse[b, h], 0)[:, None]), 0.0)
            es = (D + 4) * 2.0 ** -23 * scale * (np.abs(qq) @ np.abs(kk).T) + 4 * 2.0 ** -24 * np.abs(s)
            e = np.where(seen, es, 0).max(1, keepdims=True) + es + 2.0 ** -20 + Sk * 2.0 ** -26
            e_lse[b, h] = np.where(rows, np.where(seen, es, 0).max(1) + 2.0 ** -20 + Sk * 2.0 ** -26
                                   + 4 * 2.0 ** -24 * np.abs(np.where(rows, lse[b, h], 0)), 0)
            e_out[b, :, h] = ((U + 2 * e + Sk * 2.0 ** -23) * p + A * (p > 0)) @ np.abs(vv)
            mag = np.abs(do) @ np.abs(vv).T + (np.abs(do) * np.abs(oo)).sum(1, keepdims=True)
            ds = p * np.abs(do @ vv.T - (do * oo).sum(1, keepdims=True))
            # dp - delta: D-term products and out's own error; then p's error; then ds rounded
            eds = p * ((D + 4) * 2.0 ** -23 * mag
                       + (np.abs(do) * (e_out[b, :, h] + ut * np.abs(oo))).sum(1, keepdims=True)) \
                + (2 * e + U) * ds + U * p * (D + 4) * 2.0 ** -23 * mag + A * (p > 0)
            n = 2.0 ** -23
            e_dq[b, :, h] = scale * (eds + (Sk + 4) * n * ds) @ np.abs(kk)
            e_dk[b, :, hk] += scale * (eds + (group * Sq + 4) * n * ds).T @ np.abs(qq)
            e_dv[b, :, hk] += (p * (U + 2 * e + (group * Sq + 4) * n) + A * (p > 0)).T @ np.abs(do)
    return out, lse, e_out, e_lse, e_dq, e_dk, e_dv


def close(got, want, err, t, what):
    d = np.abs(f64(got) - want)
    tol = u(t) * np.abs(want) * (1 + 1e-6) + (1 + u(t)) * err * (1 + 1e-3) + tiny(t)
    assert np.isfinite(f64(got)).all(), what
    assert (d <= tol).all(), (what, np.max(d / tol))


def check(q, k, v, causal=False, lengths=None, scale=None, backward=True, seed=99, device_lengths=None):
    t = q.dtype
    D = q.shape[3]
    kl = lengths if device_lengths is None else device_lengths
    out, lse = attention(q, k, v, causal=causal, key_lengths=kl, scale=scale, return_lse=True)
    assert out.shape == q.shape and out.dtype == t and out.is_contiguous()
    assert lse.shape == (q.shape[0], q.shape[2], q.shape[1]) and lse.dtype == torch.float32
    dout = make(q.shape, t, seed)
    s = D ** -0.5 if scale is None else scale
    qd, kd, vd, gd = f64(q), f64(k), f64(v), f64(dout)
    U = 0.0 if t == torch.float32 else u(t)
    want, wlse, e_out, e_lse, e_dq, e_dk, e_dv = bounds(qd, kd, vd, gd, causal, lengths, s, U, u(t),
                                                          2.0 ** -25 if t == torch.float16 else 2.0 ** -125)
    close(out, want, e_out, t, "out")
    gl = f64(lse)
    assert (np.isneginf(gl) == np.isneginf(wlse)).all()
    fin = np.isfinite(wlse)
    assert (np.abs(gl[fin] - wlse[fin]) <= e_lse[fin] + 1e-7).all()
    assert torch.equal(out, attention(q, k, v, causal=causal, key_lengths=kl, scale=scale))
    if not backward:
        return
    dq, dk, dv = attention_backward(dout, q, k, v, out, lse, causal=causal, key_lengths=kl, scale=scale)
    assert dq.shape == q.shape and dk.shape == k.shape == dv.shape and dq.dtype == dk.dtype == dv.dtype == t
    wq, wk, wv = o.attention_backward(gd, qd, kd, vd, causal, lengths, s)
    close(dq, wq, e_dq, t, "dq")
    close(dk, wk, e_dk, t, "dk")
    close(dv, wv, e_dv, t, "dv")


SHAPES = [  # batch, queries, keys, heads, key heads, dim
    (1, 1, 1, 1, 1, 1), (2, 1, 17, 2, 2, 64), (1, 3, 64, 4, 2, 8), (2, 16, 65, 2, 1, 32), (1, 63, 64, 1, 1, 64),
    (1, 64, 31, 2, 2, 48), (2, 65, 33, 3, 3, 64), (1, 100, 129, 4, 2, 80), (1, 130, 200, 2, 1, 128),
    (1, 37, 300, 6, 2, 72), (3, 1, 1500, 4, 4, 64), (2, 1, 700, 8, 1, 128), (1, 2, 900, 6, 3, 33),
    (1, 257, 70, 2, 2, 65), (1, 129, 129, 1, 1, 127), (2, 5, 520, 12, 4, 96)]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_shapes(gpu, t, causal, shape):
    B, Sq, Sk, H, Hk, D = shape
    t = TYPES[t]
    q, k, v = make((B, Sq, H, D), t, 1), make((B, Sk, Hk, D), t, 2), make((B, Sk, Hk, D), t, 3)
    check(q, k, v, causal)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("sq", [1, 70])
def test_padded_batch_with_bad_values_behind_the_lengths(gpu, t, causal, sq):
    t = TYPES[t]
    lengths = [0, 1, 63, 64, 65, 150]
    q, k, v = make((6, sq, 4, 64), t, 4), make((6, 150, 2, 64), t, 5), make((6, 150, 2, 64), t, 6)
    for b, n in enumerate(lengths):
        k[b, n:], v[b, n:] = float("nan"), float("inf")
    dev = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    for given in (lengths, dev, dev.long()):
        check(q, k, v, causal, lengths, device_lengths=given)
    out, lse = attention(q, k, v, causal=causal, key_lengths=dev, return_lse=True)
    assert (out[0] == 0).all() and torch.isneginf(lse[0]).all()
    # lengths on the device are not read by the host: values outside 0 .. Sk count as the nearest
    wild = torch.tensor([-5, 1, 63, 64, 65, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
    k2, v2 = torch.nan_to_num(k), torch.nan_to_num(v, posinf=0.0)
    assert torch.equal(attention(q, k2, v2, causal=causal, key_lengths=wild),
                       attention(q, k2, v2, causal=causal, key_lengths=dev))


@pytest.mark.parametrize("t", TYPES)
def test_views_and_alignment(gpu, t):
    t = TYPES[t]
    rows = make((2, 90, 3, 4, 64), t, 7)
    q, k, v = rows[:, :, 0], rows[:, :, 1], rows[:, :, 2]         # slices of one projection
    check(q, k, v)
    out, lse = attention(q, k, v, return_lse=True)
    dout = make((2, 4, 90, 64), t, 8).transpose(1, 2)             # heads in front of rows
    got = attention_backward(dout, q, k, v, out, lse)
    want = attention_backward(*(x.contiguous() for x in (dout, q, k, v)), out, lse)
    assert all(torch.equal(a, c) for a, c in zip(got, want))
    flat = make((2 * 90 * 4 * 70 + 1,), t, 9)[1:].view(2, 90, 4, 70)
    q2 = flat[..., 3:67]                                          # rows that start at odd elements
    assert torch.equal(attention(q2, q2, q2), attention(*(q2.contiguous() for _ in range(3))))
    check(q2, q2, q2)
    qt = make((2, 64, 4, 50), t, 10).permute(0, 3, 2, 1)          # dim not contiguous
    assert torch.equal(attention(qt, k[:, :50], v[:, :50]), attention(qt.contiguous(), k[:, :50], v[:, :50]))
    one = k[:1].expand(2, -1, -1, -1)                             # one item's keys for the whole batch
    assert torch.equal(attention(q, one, one), attention(q, one.contiguous(), one.contiguous()))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("dim", [32, 64, 96, 128])
def test_many_workgroups(gpu, t, dim):
    """Enough rows for the wider workgroups, forward and backward."""
    t = TYPES[t]
    q, k, v = make((16, 140, 16, dim), t, 11), make((16, 130, 16, dim), t, 12), make((16, 130, 16, dim), t, 13)
    lengths = [130 - 7 * i for i in range(16)]
    check(q, k, v, True, lengths)


def test_large_and_small_scores(gpu):
    for t in TYPES.values():
        q, k, v = make((1, 40, 2, 64), t, 14, 4.0), make((1, 80, 2, 64), t, 15, 4.0), make((1, 80, 2, 64), t, 16)
        check(q, k, v, scale=1.0)      # one key takes nearly all of a row
        check(q, k, v, scale=1e-4)     # nearly even
    q = torch.zeros((1, 5, 1, 64), device="cuda")
    v = make((1, 9, 1, 64), torch.float32, 17)
    out, lse = attention(q, v, v, return_lse=True)
    assert torch.allclose(lse, torch.full_like(lse, float(np.log(9.0))), atol=1e-6, rtol=0)


def test_empty_sizes(gpu):
    q, kv = make((2, 3, 2, 64), torch.float16, 18), torch.empty((2, 0, 2, 64), dtype=torch.float16, device="cuda")
    out, lse = attention(q, kv, kv, return_lse=True)
    assert (out == 0).all() and torch.isneginf(lse).all()
    dq, dk, dv = attention_backward(q, q, kv, kv, out, lse)
    assert (dq == 0).all() and dk.shape == kv.shape
    none = q[:, :0]
    out, lse = attention(none, q, q, return_lse=True)
    assert out.shape == (2, 0, 2, 64)
    dq, dk, dv = attention_backward(none, none, q, q, out, lse)
    assert (dk == 0).all() and (dv == 0).all() and dq.shape == none.shape
    assert attention(q[:0], q[:0], q[:0]).shape == (0, 3, 2, 64)


def test_gradient_against_differences(gpu):
    q, k, v = make((1, 20, 4, 24), torch.float32, 19), make((1, 30, 2, 24), torch.float32, 20), make((1, 30, 2, 24), torch.float32, 21)
    dout = make((1, 20, 4, 24), torch.float32, 22)
    out, lse = attention(q, k, v, causal=True, key_lengths=[25], return_lse=True)
    grads = [f64(x) for x in attention_backward(dout, q, k, v, out, lse, causal=True, key_lengths=[25])]
    rng = np.random.default_rng(2)
    dirs = [rng.standard_normal(g.shape) for g in grads]
    h = 1e-5
    loss = lambda s: (f64(dout) * o.attention(*(f64(x) + s * d for x, d in zip((q, k, v), dirs)), True, [25])[0]).sum()
    want = (loss(h) - loss(-h)) / (2 * h)
    terms = [g * d for g, d in zip(grads, dirs)]
    assert abs(sum(x.sum() for x in terms) - want) <= 3e-5 * sum(np.abs(x).sum() for x in terms)


def test_two_calls_give_the_same_bits(gpu):
    q, k = make((2, 300, 6, 64), torch.bfloat16, 23), make((2, 300, 2, 64), torch.bfloat16, 24)
    out, lse = attention(q, k, k, return_lse=True)
    first = attention_backward(out, q, k, k, out, lse)
    for _ in range(3):
        assert all(torch.equal(a, c) for a, c in zip(first, attention_backward(out, q, k, k, out, lse)))


@pytest.mark.parametrize("t", TYPES)
def test_many_items_and_split_keys_with_lengths(gpu, t):
    t = TYPES[t]
    lengths = [(17 * i) % 41 for i in range(70)]        # more items than a wave has lanes, lengths 0 ... 40
    q, k, v = make((70, 33, 1, 64), t, 25), make((70, 40, 1, 64), t, 26), make((70, 40, 1, 64), t, 27)
    check(q, k, v, False, lengths)
    q, k, v = make((3, 1, 4, 64), t, 28), make((3, 1500, 2, 64), t, 29), make((3, 1500, 2, 64), t, 30)
    for lengths in ([0, 700, 1500], [1, 256, 257]):
        for b, n in enumerate(lengths):
            k[b, n:], v[b, n:] = float("nan"), float("nan")
        check(q, k, v, False, lengths)
        check(q, k, v, True, lengths)
        k, v = torch.nan_to_num(k), torch.nan_to_num(v)


def test_a_cache_beyond_four_gigabytes(gpu):
    """Keys whose offsets pass 32 bits, in elements as well as bytes: the last head's keys and values
    against a compact copy of them, bit for bit."""
    Sk, Hk = 300_000, 64
    kv = torch.zeros((2, 1, Sk, Hk, 128), dtype=torch.bfloat16, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(31)
    kv[:, :, :, 63:] = torch.randn((2, 1, Sk, 1, 128), generator=g, device="cuda").to(torch.bfloat16)
    k, v = kv[0, :, :, 63:], kv[1, :, :, 63:]
    q = torch.randn((1, 2, 1, 128), generator=g, device="cuda").to(torch.bfloat16)
    for n in (Sk, Sk - 7):
        out, lse = attention(q, k, v, key_lengths=[n], return_lse=True)
        kc, vc = k.contiguous(), v.contiguous()
        want, wlse = attention(q, kc, vc, key_lengths=[n], return_lse=True)
        assert torch.equal(out, want) and torch.equal(lse, wlse)
        got = attention_backward(out, q, k, v, out, lse, key_lengths=[n])
        ref = attention_backward(out, q, kc, vc, out, lse, key_lengths=[n])
        assert all(torch.equal(a, c) for a, c in zip(got, ref))
