"""attention_backward of float16 over the range of magnitudes that gradients really have.

The oracle is the formula in float64 on the kernel's own inputs (out and lse among them).  A float16 result
carries its own rounding and, from the operands of the products, one more of the probabilities or of their
gradients, independent of it and of the same relative size: together sqrt(2) = 1.42 of a result rounded
once, in the root mean square over a tensor.  How values lie within their binades moves the size of a
rounding by a few per cent: 1.5.  Up to 64 queries dq carries both parts of ds, so the result's own rounding
is left: 1.05.  Nothing in this depends on the size of dout or v."""
import pytest
import torch

from mlx_audio_amd.frontends import attention, attention_backward
from test_gpu_attention import make

pytestmark = pytest.mark.gpu
HALF = torch.float16


def exact(dout, q, k, v, out, lse, causal=False, scale=None):
    dout, q, k, v, out, lse = (x.cpu().double() for x in (dout, q, k, v, out, lse))
    group = q.shape[2] // k.shape[2]
    scale = q.shape[3] ** -0.5 if scale is None else scale
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    for b in range(q.shape[0]):
        for h in range(q.shape[2]):
            kk, vv, qq, do = k[b, :, h // group], v[b, :, h // group], q[b, :, h], dout[b, :, h]
            s = scale * (qq @ kk.T)
            if causal:
                s.masked_fill_(torch.ones_like(s, dtype=torch.bool).triu(1 + len(kk) - len(qq)), float("-inf"))
            p = torch.exp(s - lse[b, h][:, None])
            ds = scale * p * (do @ vv.T - (do * out[b, :, h]).sum(1, keepdim=True))
            dq[b, :, h] = ds @ kk
            dk[b, :, h // group] += ds.T @ qq
            dv[b, :, h // group] += p.T @ do
    return dq, dk, dv


def against_one_rounding(got, want):
    """Root mean square error in units of that of a result rounded once."""
    once = (want.to(HALF).double() - want).square().mean().sqrt()
    return float((got.cpu().double() - want).square().mean().sqrt() / once)


SHAPES = [  # batch, queries, keys, heads, key heads, dim
    (1, 1500, 1500, 2, 2, 64), (2, 64, 1500, 4, 2, 64), (1, 300, 700, 4, 1, 80), (1, 1, 4000, 16, 16, 128),
    (1, 700, 333, 3, 3, 33), (16, 200, 200, 16, 16, 64)]


@pytest.mark.parametrize("size", [1e3, 1.0, 1e-2, 1e-3, 1e-4, 1e-5])
@pytest.mark.parametrize("shape", SHAPES)
def test_every_size_of_gradient(gpu, shape, size):
    B, Sq, Sk, H, Hk, D = shape
    q, k, v = make((B, Sq, H, D), HALF, 1), make((B, Sk, Hk, D), HALF, 2), make((B, Sk, Hk, D), HALF, 3)
    dout = make((B, Sq, H, D), HALF, 4, size)
    causal = Sq <= Sk and D == 80
    out, lse = attention(q, k, v, causal=causal, return_lse=True)
    got = attention_backward(dout, q, k, v, out, lse, causal=causal)
    want = exact(dout, q, k, v, out, lse, causal)
    ratios = [against_one_rounding(g, w) for g, w in zip(got, want)]
    assert ratios[0] <= (1.05 if Sq <= 64 else 1.5) and max(ratios[1:]) <= 1.5, ratios


@pytest.mark.parametrize("shape", SHAPES[:3])
def test_rows_of_different_sizes(gpu, shape):
    """Every query's dout of its own size: dq of the small ones is as exact as that of the large ones."""
    B, Sq, Sk, H, Hk, D = shape
    q, k, v = make((B, Sq, H, D), HALF, 5), make((B, Sk, Hk, D), HALF, 6), make((B, Sk, Hk, D), HALF, 7, 3.0)
    size = 10.0 ** -(torch.arange(Sq, device="cuda") % 5).float()
    dout = (make((B, Sq, H, D), torch.float32, 8) * size[None, :, None, None]).to(HALF)
    out, lse = attention(q, k, v, return_lse=True)
    got = attention_backward(dout, q, k, v, out, lse)
    want = exact(dout, q, k, v, out, lse)
    for i in range(5):
        assert against_one_rounding(got[0][:, i::5], want[0][:, i::5]) <= (1.05 if Sq <= 64 else 1.5), i
    assert max(against_one_rounding(g, w) for g, w in zip(got[1:], want[1:])) <= 1.5


@pytest.mark.parametrize("sq", [1, 20, 64, 65, 200, 1100])
def test_scores_whose_gradient_passes_the_largest_number(gpu, sq):
    """ds beyond 65504 while the gradients themselves are not: they are as exact as any; and where a gradient
    passes it as well, it is infinite."""
    B, Sk, H, D = 2, 150, 8, 64
    q, k = make((B, sq, H, D), HALF, 9, 1e-3), make((B, Sk, H, D), HALF, 10, 1e-3)
    v, dout = make((B, Sk, H, D), HALF, 11, 1000.0), make((B, sq, H, D), HALF, 12, 10000.0)
    out, lse = attention(q, k, v, return_lse=True)
    got = attention_backward(dout, q, k, v, out, lse)
    want = exact(dout, q, k, v, out, lse)
    # dv, sums of dout up to 4e4 itself, stays finite where the probabilities (1 / 150) keep it small
    ratios = [against_one_rounding(g, w) for g, w in zip(got, want)]
    assert ratios[0] <= (1.05 if sq <= 64 else 1.5) and max(ratios[1:]) <= 1.5, ratios
    large = make((B, Sk, H, D), HALF, 10, 1.0)
    out, lse = attention(q, large, v, return_lse=True)
    dq = attention_backward(dout, q, large, v, out, lse)[0].cpu()
    want = exact(dout, q, large, v, out, lse)[0]
    assert not torch.isnan(dq).any()
    beyond, within = want.abs() > 1.02 * 65504, want.abs() < 0.98 * 65504   # (in between either is right)
    assert beyond.any() and within.any()
    assert torch.equal(dq[beyond], want[beyond].sign().to(HALF) * float("inf")) and torch.isfinite(dq[within]).all()


def test_zero_gradients_and_zero_values(gpu):
    q, k = make((2, 70, 4, 64), HALF, 13), make((2, 90, 2, 64), HALF, 14)
    zero = torch.zeros_like(q)
    out, lse = attention(q, k, k, return_lse=True)
    assert all((g == 0).all() for g in attention_backward(zero, q, k, k, out, lse))
    none = torch.zeros_like(k)
    out, lse = attention(q, k, none, return_lse=True)
    dq, dk, dv = attention_backward(q, q, k, none, out, lse)
    assert (dq == 0).all() and (dk == 0).all()
    assert against_one_rounding(dv, exact(q, q, k, none, out, lse)[2]) <= 1.5


def test_captured_and_replayed(gpu):
    """The norms are worked out anew in every replay."""
    q, k, v, dout = (make((2, 130, 4, 64), HALF, 15 + i) for i in range(4))
    out, lse = attention(q, k, v, return_lse=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        attention_backward(dout, q, k, v, out, lse)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = attention_backward(dout, q, k, v, out, lse)
    for turn, size in enumerate((1.0, 1e-4, 1e3, 1e-2)):
        dout.copy_(make(dout.shape, HALF, 20 + turn, size))
        graph.replay()
        torch.cuda.synchronize()
        eager = attention_backward(dout, q, k, v, out, lse)
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(got, eager)), size


@pytest.mark.parametrize("dim", [40, 33])
def test_lengths_views_and_shared_heads(gpu, dim):
    """Values behind a length take no part in the scale; views read the same as their copies."""
    rows = make((3, 150, 6, dim + 3), HALF, 30)
    q, k, v = rows[:, :, :4, 1:dim + 1], rows[:, :, 4:5, 1:dim + 1], rows[:, :, 5:6, 1:dim + 1]
    dout = make((3, 150, 4, dim), HALF, 31, 1e-3)
    lengths = [150, 37, 0]
    out, lse = attention(q, k, v, key_lengths=lengths, return_lse=True)
    got = attention_backward(dout, q, k, v, out, lse, key_lengths=lengths)
    kc, vc = k.clone(), v.clone()
    for b, n in enumerate(lengths):
        kc[b, n:], vc[b, n:] = float("nan"), float("inf")
    again = attention_backward(dout, q.contiguous(), kc, vc, out, lse, key_lengths=lengths)
    assert all(torch.equal(a, c) for a, c in zip(got, again))
    want = exact(dout[:1], q[:1], k[:1], v[:1], out[:1], lse[:1])
    assert max(against_one_rounding(g[:1], w) for g, w in zip(got, want)) <= 1.5
    want = exact(dout[1:2], q[1:2], k[1:2, :37], v[1:2, :37], out[1:2], lse[1:2])
    assert max(against_one_rounding(g[1:2, :n], w) for g, w, n in zip(got, want, (150, 37, 37))) <= 1.5
    assert all((g[1, 37:] == 0).all() and (g[2] == 0).all() for g in got[1:]) and (got[0][2] == 0).all()


def test_no_items_queries_or_keys(gpu):
    for B, Sq, Sk in ((0, 5, 7), (2, 0, 7), (2, 5, 0), (0, 0, 0)):
        q, kv = make((B, Sq, 4, 40), HALF, 40), make((B, Sk, 2, 40), HALF, 41)
        out, lse = attention(q, kv, kv, return_lse=True)
        dq, dk, dv = attention_backward(q, q, kv, kv, out, lse)
        assert dq.shape == q.shape and dk.shape == dv.shape == kv.shape
        assert all((g == 0).all() for g in (dq, dk, dv))


def test_one_gradient_for_every_query(gpu):
    """dout expanded along items, queries and heads (the gradient of a sum), against its copy."""
    q, k, v = make((3, 70, 4, 64), HALF, 42), make((3, 90, 2, 64), HALF, 43), make((3, 90, 2, 64), HALF, 44)
    dout = make((64,), HALF, 45, 1e-3).expand(3, 70, 4, 64)
    out, lse = attention(q, k, v, return_lse=True)
    got, want = attention_backward(dout, q, k, v, out, lse), attention_backward(dout.contiguous(), q, k, v, out, lse)
    assert all(torch.equal(a, c) for a, c in zip(got, want))
    assert max(against_one_rounding(g, w) for g, w in zip(got, exact(dout, q, k, v, out, lse))) <= 1.5


def test_many_items_and_many_heads_on_one_key_head(gpu):
    q, k, v = make((300, 9, 8, 32), HALF, 46), make((300, 20, 1, 32), HALF, 47), make((300, 20, 1, 32), HALF, 48)
    dout = make(q.shape, HALF, 49, 1e-4)
    lengths = [(7 * i) % 21 for i in range(300)]
    out, lse = attention(q, k, v, key_lengths=lengths, return_lse=True)
    got = attention_backward(dout, q, k, v, out, lse, key_lengths=lengths)
    for b in (0, 1, 2, 150, 299):
        n = lengths[b]
        want = exact(dout[b:b + 1], q[b:b + 1], k[b:b + 1, :n], v[b:b + 1, :n], out[b:b + 1], lse[b:b + 1]) if n else None
        if n:
            alone = attention_backward(*(x[b:b + 1] for x in (dout, q)), k[b:b + 1, :n], v[b:b + 1, :n], out[b:b + 1], lse[b:b + 1])
            assert torch.equal(got[0][b], alone[0][0])
            assert max(against_one_rounding(g[b:b + 1, :m], w) for g, w, m in zip(got, want, (9, n, n))) <= 1.6  # (few values)
        assert (got[1][b, n:] == 0).all() and (got[2][b, n:] == 0).all()


def test_calls_at_once_on_two_streams(gpu):
    sets = []
    for i, size in enumerate((1.0, 1e-4)):
        q, k, v = make((4, 300, 8, 64), HALF, 50 + i), make((4, 300, 8, 64), HALF, 52 + i), make((4, 300, 8, 64), HALF, 54 + i)
        dout = make(q.shape, HALF, 56 + i, size)
        out, lse = attention(q, k, v, return_lse=True)
        sets.append((dout, q, k, v, out, lse))
    want = [attention_backward(*s) for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(attention_backward(*sets[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(a, c) for one in got[i] for a, c in zip(one, want[i]))
