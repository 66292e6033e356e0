"""The operators behind the encoder stem together, as a block of the encoder runs them: forward and
backward against the float64 oracle, captured into graphs, and on a stream of their own.

float32 tolerance: every product sums K <= 1024 terms in float32, at most K 2^-23 = 1.2e-4 of its sum of
magnitudes in the worst case and about sqrt(K) 2^-24 = 2e-6 for terms of random sign, as here; the
block chains seven of them and the backward pass as many again.  1e-4 of a result's largest magnitude
leaves that chain a factor of about seven, and is far below any mistake of layout or order."""
import numpy as np
import pytest
import torch

from mlx_audio_amd.frontends import (WhisperEncoderStem, attention, attention_backward, layer_norm, layer_norm_backward,
                                     linear, linear_backward, sinusoids)
from oracle import transformer as o, whisper_stem as ws

pytestmark = pytest.mark.gpu
N, H = 256, 4
D = N // H


def weights(seed, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s, scale=1.0: (torch.randn(s, generator=g) * scale).to(dtype).cuda()
    return {"ln1.w": 1 + r(N, scale=0.1), "ln1.b": r(N, scale=0.1), "qkv.w": r(3 * N, N, scale=N ** -0.5),
            "qkv.b": r(3 * N, scale=0.1), "out.w": r(N, N, scale=N ** -0.5), "out.b": r(N, scale=0.1),
            "ln2.w": 1 + r(N, scale=0.1), "ln2.b": r(N, scale=0.1), "up.w": r(4 * N, N, scale=N ** -0.5),
            "up.b": r(4 * N, scale=0.1), "down.w": r(N, 4 * N, scale=(4 * N) ** -0.5), "down.b": r(N, scale=0.1)}


def block(x, w, lengths):
    """(y, what the backward pass needs)"""
    B, S, _ = x.shape
    h1, m1, r1 = layer_norm(x, w["ln1.w"], w["ln1.b"], return_stats=True)
    qkv = linear(h1, w["qkv.w"], w["qkv.b"]).view(B, S, 3, H, D)
    q, k, v = qkv.unbind(2)
    a, lse = attention(q, k, v, key_lengths=lengths, return_lse=True)
    x1 = linear(a.view(B, S, N), w["out.w"], w["out.b"], residual=x)
    h2, m2, r2 = layer_norm(x1, w["ln2.w"], w["ln2.b"], return_stats=True)
    u, z = linear(h2, w["up.w"], w["up.b"], activation="gelu", return_preactivation=True)
    y = linear(u, w["down.w"], w["down.b"], residual=x1)
    return y, (x, h1, m1, r1, qkv, a, lse, x1, h2, m2, r2, u, z)


def block_backward(dy, kept, w, lengths):
    x, h1, m1, r1, qkv, a, lse, x1, h2, m2, r2, u, z = kept
    B, S, _ = x.shape
    g = {}
    du, g["down.w"], g["down.b"] = linear_backward(dy, u, w["down.w"])
    dh2, g["up.w"], g["up.b"] = linear_backward(du, h2, w["up.w"], activation="gelu", preactivation=z)
    dx1, g["ln2.w"], g["ln2.b"] = layer_norm_backward(dh2, x1, m2, r2, w["ln2.w"])
    dx1 = dx1 + dy
    da, g["out.w"], g["out.b"] = linear_backward(dx1, a.view(B, S, N), w["out.w"])
    q, k, v = qkv.unbind(2)
    dqkv = torch.stack(attention_backward(da.view(B, S, H, D), q, k, v, a, lse, key_lengths=lengths), 2)
    dh1, g["qkv.w"], g["qkv.b"] = linear_backward(dqkv.view(B, S, 3 * N), h1, w["qkv.w"])
    dx, g["ln1.w"], g["ln1.b"] = layer_norm_backward(dh1, x, m1, r1, w["ln1.w"])
    g["x"] = dx + dx1
    return g


def oracle_block(x, w, lengths):
    B, S, _ = x.shape
    h = o.layer_norm(x, w["ln1.w"], w["ln1.b"])[0]
    qkv = o.linear(h, w["qkv.w"], w["qkv.b"])[0].reshape(B, S, 3, H, D)
    a = o.attention(qkv[:, :, 0], qkv[:, :, 1], qkv[:, :, 2], False, lengths)[0].reshape(B, S, N)
    x1 = o.linear(a, w["out.w"], w["out.b"], None, x)[0]
    u = o.linear(o.layer_norm(x1, w["ln2.w"], w["ln2.b"])[0], w["up.w"], w["up.b"], "gelu")[0]
    return o.linear(u, w["down.w"], w["down.b"], None, x1)[0]


def f64(t):
    return t.detach().cpu().double().numpy()


def test_block_behind_the_stem(gpu):
    rng = np.random.default_rng(0)
    mel = rng.standard_normal((3, 80, 203)).astype(np.float32)
    w1, b1 = (rng.standard_normal((N, 3, 80)) / 16).astype(np.float32), (0.1 * rng.standard_normal(N)).astype(np.float32)
    w2, b2 = (rng.standard_normal((N, 3, N)) / 28).astype(np.float32), (0.1 * rng.standard_normal(N)).astype(np.float32)
    pos = sinusoids(102, N)
    x = WhisperEncoderStem(w1, b1, w2, b2, pos)(torch.from_numpy(mel).cuda())
    lengths = [102, 57, 0]
    w = weights(1)
    y, kept = block(x, w, lengths)
    wd = {n: f64(t) for n, t in w.items()}
    want = oracle_block(ws.encoder_stem(mel, w1, b1, w2, b2, pos.numpy(), dtype=np.float64), wd, lengths)
    assert np.abs(f64(y) - want).max() <= 1e-4 * np.abs(want).max()
    # gradients of sum(dy * y) along random directions of every weight and of x, by differences
    g = torch.Generator().manual_seed(2)
    dy = torch.randn(y.shape, generator=g).cuda()
    grads = block_backward(dy, kept, w, lengths)
    xd, dyd = f64(x), f64(dy)
    for name in ("x", *w):
        base = xd if name == "x" else wd[name]
        u = rng.standard_normal(base.shape)
        h = 1e-4 / np.abs(u).max()

        def loss(s):
            if name == "x":
                return (dyd * oracle_block(xd + s * u, wd, lengths)).sum()
            return (dyd * oracle_block(xd, {**wd, name: wd[name] + s * u}, lengths)).sum()

        diff = (loss(h) - loss(-h)) / (2 * h)
        terms = f64(grads[name]) * u
        # random directions cancel: the scale of the sum is the root of its terms' squares
        assert abs(terms.sum() - diff) <= 1e-4 * np.sqrt((terms ** 2).sum()) * np.sqrt(terms.size) ** 0.5, name


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16])
def test_captured_into_graphs(gpu, t):
    """Two graphs of a forward and backward pass, replayed in turn with new inputs and the program's own
    eager work between, against the eager results, bit for bit."""
    w = weights(3, t)
    g = torch.Generator().manual_seed(4)
    shapes = [(2, 130, N), (1, 300, N)]
    lengths = [torch.tensor([130, 77], dtype=torch.int32, device="cuda"), None]
    x = [torch.randn(s, generator=g).to(t).cuda() for s in shapes]
    dy = [torch.randn(s, generator=g).to(t).cuda() for s in shapes]

    def step(i):
        y, kept = block(x[i], w, lengths[i])
        return y, block_backward(dy[i], kept, w, lengths[i])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for i in range(2):
            step(i)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for i in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step(i))
        graphs.append(graph)
    for turn in range(4):
        for i in (0, 1) if turn % 2 else (1, 0):
            x[i].copy_(torch.randn(shapes[i], generator=g).to(t))
            if lengths[i] is not None:
                lengths[i].copy_(torch.tensor([130 - 40 * turn, 10 + turn], dtype=torch.int32))
            graphs[i].replay()
            torch.cuda.synchronize()
            y, grads = step(i)
            torch.cuda.synchronize()
            assert torch.equal(y, outs[i][0])
            for name in grads:
                assert torch.equal(grads[name], outs[i][1][name]), (turn, i, name)


def test_on_a_stream_of_its_own(gpu):
    w = weights(5)
    g = torch.Generator().manual_seed(6)
    x, dy = torch.randn((2, 90, N), generator=g).cuda(), torch.randn((2, 90, N), generator=g).cuda()
    y, kept = block(x, w, None)
    want = block_backward(dy, kept, w, None)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        late = torch.zeros_like(x)
        torch.cuda._sleep(20_000_000)   # the input arrives late on this stream; nothing may run ahead of it
        late.copy_(x)
        y2, kept2 = block(late, w, None)
        got = block_backward(dy, kept2, w, None)
    side.synchronize()
    assert torch.equal(y, y2) and all(torch.equal(got[n], want[n]) for n in want)


def test_memory_behind_the_outputs_is_left_alone(gpu):
    """Results of ragged sizes written into the front of a larger buffer through the C entry: nothing
    behind them changes."""
    from mlx_audio_amd import _lib

    lib = _lib.lib()
    for t, code in ((torch.float32, _lib.F32), (torch.bfloat16, _lib.BF16)):
        for m, k, n in ((5, 33, 19), (67, 40, 130), (130, 70, 65)):
            x, wt = torch.randn(m, k).to(t).cuda(), torch.randn(n, k).to(t).cuda()
            out = torch.full((m * n + 999,), 7.0, dtype=t, device="cuda")
            need = lib.mia_linear_workspace_bytes(m, k, n, code)
            wsp = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")
            _lib.check(lib.mia_linear(x.data_ptr(), k, wt.data_ptr(), k, None, code, None, 0, 0, m, k, n, code,
                                      out.data_ptr(), None, wsp.data_ptr(), need, torch.cuda.current_stream().cuda_stream))
            assert torch.equal(out[:m * n].view(m, n), linear(x, wt)) and (out[m * n:] == 7.0).all()
        for rows, dim in ((3, 77), (2, 9001)):
            x = torch.randn(rows, dim).to(t).cuda()
            out = torch.full((rows * dim + 999,), 7.0, dtype=t, device="cuda")
            _lib.check(lib.mia_layer_norm(x.data_ptr(), rows, dim, dim, code, None, None, code, 1e-5, out.data_ptr(),
                                          None, None, torch.cuda.current_stream().cuda_stream))
            assert torch.equal(out[:rows * dim].view(rows, dim), layer_norm(x)) and (out[rows * dim:] == 7.0).all()
