"""What is measured of the operators behind the encoder stem: layer normalisation, the linear
layer with its epilogue, and attention, each forward and backward.

The sizes are those of the Whisper encoder that `bench.py --workload whisper_stem` builds (1280
channels, 1500 frames a clip, 20 heads of 64, a hidden layer four times as wide) and generic ones
around them: single tokens, small batches, ragged and odd sizes.
"""

import math

import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "f16": 2, "bf16": 2}


# ---------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------
def _ln(name, direction, rows, dim, dtype):
    return {"name": name, "op": "layer_norm", "direction": direction, "rows": rows, "dim": dim, "dtype": dtype}


def _lin(name, direction, rows, k, n, dtype, activation="none", bias=True, residual=False):
    return {"name": name, "op": "linear", "direction": direction, "rows": rows, "k": k, "n": n, "dtype": dtype,
            "activation": activation, "bias": bias, "residual": residual}


def _att(name, direction, batch, sq, sk, heads, kv_heads, dim, dtype, causal=False, lengths=False, packed=False):
    return {"name": name, "op": "attention", "direction": direction, "batch": batch, "sq": sq, "sk": sk,
            "heads": heads, "kv_heads": kv_heads, "dim": dim, "dtype": dtype, "causal": causal,
            "lengths": lengths, "packed": packed}


def listed():
    return [
        # the norm in front of a decoding step's projections: eight tokens, latency only
        _ln("layer_norm_step", "forward", 8, 1280, "bf16"),
        # the norm in front of a block of the encoder, 64 clips of 30 s
        _ln("layer_norm_batch", "forward", 64 * 1500, 1280, "f16"),
        # its backward pass in a fine-tuning step of 32 clips, with the weight's and bias's gradients
        _ln("layer_norm_grad", "backward", 32 * 1500, 1280, "bf16"),
        # the hidden layer of one decoding step of eight sequences: reads the weights once
        _lin("linear_step", "forward", 8, 1280, 5120, "bf16", "gelu"),
        # the hidden layer of the encoder's block in training (keeps what its backward pass needs)
        _lin("linear_hidden", "forward", 16 * 1500, 1280, 5120, "bf16", "gelu"),
        # the layer back to the channels, added to the residual stream, for a float32 checkpoint
        _lin("linear_out_f32", "forward", 4 * 1500, 5120, 1280, "f32", "none", residual=True),
        # the backward pass of the hidden layer in the same training step
        _lin("linear_hidden_grad", "backward", 16 * 1500, 1280, 5120, "bf16", "gelu"),
        # a projection head of odd widths on a ragged batch, backward
        _lin("linear_odd_grad", "backward", 1111, 777, 1030, "f16", "relu"),
        # one new token of 16 sequences over the 1500 frames of the encoder's output
        _att("attention_step", "forward", 16, 1, 1500, 20, 20, 64, "f16"),
        # the encoder's self-attention over 16 clips of different lengths, views of one packed projection
        _att("attention_encoder", "forward", 16, 1500, 1500, 20, 20, 64, "bf16", lengths=True, packed=True),
        # its backward pass, eight clips
        _att("attention_encoder_grad", "backward", 8, 1500, 1500, 20, 20, 64, "bf16", lengths=True),
        # a causal layer with shared key heads, odd lengths and a head size between the common ones, float32
        _att("attention_causal_grad_f32", "backward", 3, 333, 333, 6, 2, 80, "f32", causal=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["layer_norm", "linear", "attention"])
    direction = rng.choice(["forward", "backward"])
    dtype = rng.choice(["bf16", "f16", "f32"])
    if op == "layer_norm":
        dim = rng.choice([384, 512, 768, 1024, 1280, _log_int(rng, 1, 10000)])
        rows = _log_int(rng, 1, min(96000, 123_000_000 // dim) if dtype != "f32" else min(48000, 61_000_000 // dim))
        case = _ln("", direction, rows, dim, dtype)
    elif op == "linear":
        k = rng.choice([384, 512, 768, 1280, _log_int(rng, 16, 5120)])
        n = rng.choice([384, 512, 1024, 1280, _log_int(rng, 16, 5120)])
        flops = 1.5e11 if direction == "backward" else 3e11
        if dtype == "f32":
            flops /= 4
        rows = _log_int(rng, 1, max(2, min(24000, int(flops / (2.0 * k * n)))))
        activation = rng.choice(["none", "gelu", "gelu_tanh", "relu"])
        case = _lin("", direction, rows, k, n, dtype, activation, bias=rng.random() < 0.8,
                    residual=rng.random() < 0.5)
    else:
        batch = _log_int(rng, 1, 16)
        kv_heads = rng.choice([1, 2, 4, 6, 8, 12])
        heads = kv_heads * rng.choice([1, 1, 2, 4])
        dim = rng.choice([64, 64, 128, 32, 48, 80, 96, rng.randint(8, 128)])
        sk = _log_int(rng, 1, 4096)
        self_attention = rng.random() < 0.6
        sq = sk if self_attention else rng.choice([1, 1, _log_int(rng, 1, 2048)])
        most = 1.0e8 if dtype == "f32" else 4.0e8   # query-key pairs over all heads
        while batch * heads * sq * sk > most and batch > 1:
            batch -= 1
        while batch * heads * sq * sk > most:
            sk = max(1, sk // 2)
            sq = min(sq, sk) if self_attention else max(1, sq // 2)
        case = _att("", direction, batch, sq, sk, heads, kv_heads, dim, dtype, causal=rng.random() < 0.4,
                    lengths=rng.random() < 0.4, packed=sq == sk and heads == kv_heads and rng.random() < 0.5)
    del case["name"]
    return case


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------
def _randn(gen, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32) * scale).to(dtype)


def _derivative(z, activation):
    """The activation's derivative at z, elementary operations in z's type."""
    if activation == "gelu":
        return 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)
    if activation == "gelu_tanh":
        c, a = math.sqrt(2.0 / math.pi), 0.044715
        t = torch.tanh(c * (z + a * z * z * z))
        return 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * c * (1.0 + 3.0 * a * z * z)
    if activation == "relu":
        return (z > 0).to(z.dtype)
    return torch.ones_like(z)


def _activate(z, activation):
    if activation == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
    if activation == "gelu_tanh":
        return 0.5 * z * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (z + 0.044715 * z * z * z)))
    if activation == "relu":
        return torch.clamp(z, min=0.0)
    return z


def _visible(case, lengths, b0=0, b1=None):
    """Which keys each query sees: [batch or 1, 1, sq or 1, sk] truth values, or None for all."""
    seen = None
    j = torch.arange(case["sk"], device="cuda")
    if case["causal"]:
        i = torch.arange(case["sq"], device="cuda")
        seen = (j[None, :] <= i[:, None] + (case["sk"] - case["sq"]))[None, None]
    if lengths is not None:
        inside = (j[None, :] < lengths[b0:b1, None])[:, None, None, :]
        seen = inside if seen is None else seen & inside
    return seen


def _per_head(x, group=1):
    """[batch, s, heads, dim] -> [batch, heads * group, s, dim] in 32 bits, contiguous."""
    x = x.to(torch.float32).transpose(1, 2).contiguous()
    return x if group == 1 else x.repeat_interleave(group, dim=1)


def _plain_attention(case, q, k, v, lengths):
    """(out, lse) in 32 bits: out [batch, sq, heads, dim], lse [batch, heads, sq]."""
    group = case["heads"] // case["kv_heads"]
    s = torch.matmul(_per_head(q), _per_head(k, group).transpose(-1, -2).contiguous())
    s = s * (1.0 / math.sqrt(case["dim"]))
    seen = _visible(case, lengths)
    if seen is not None:
        s = s.masked_fill(~seen, float("-inf"))
    top = s.amax(dim=-1, keepdim=True)
    top = torch.where(top == float("-inf"), torch.zeros_like(top), top)
    p = torch.exp(s - top)
    total = p.sum(dim=-1, keepdim=True)
    lse = (torch.log(total) + top)[..., 0]
    p = p / torch.where(total == 0, torch.ones_like(total), total)
    return torch.matmul(p, _per_head(v, group)).transpose(1, 2).contiguous(), lse


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    t = _TYPES[case["dtype"]]
    state = {"case": case}
    if case["op"] == "layer_norm":
        rows, dim = case["rows"], case["dim"]
        # residual-stream rows: each with its own offset and scale, a few strong channels
        x = torch.randn((rows, dim), generator=gen, device="cuda")
        x = x * (0.5 + torch.rand((rows, 1), generator=gen, device="cuda")) + 0.3 * torch.randn((rows, 1), generator=gen,
                                                                                             device="cuda")
        strong = torch.rand((dim,), generator=gen, device="cuda") < 0.005
        x = x * (1.0 + 9.0 * strong.to(torch.float32))
        state["x"] = x.to(t)
        state["weight"] = (1.0 + _randn(gen, dim, scale=0.1)).to(t)
        state["bias"] = _randn(gen, dim, dtype=t, scale=0.1)
        if case["direction"] == "backward":
            x32 = state["x"].to(torch.float32)
            mean = x32.mean(dim=-1)
            x32 = x32 - mean[:, None]
            state["mean"], state["rstd"] = mean, torch.rsqrt((x32 * x32).mean(dim=-1) + 1e-5)
            state["dy"] = _randn(gen, rows, dim, dtype=t)
        return state
    if case["op"] == "linear":
        rows, k, n = case["rows"], case["k"], case["n"]
        state["x"] = _randn(gen, rows, k, dtype=t)
        state["weight"] = _randn(gen, n, k, dtype=t, scale=1.0 / math.sqrt(k))
        state["bias"] = _randn(gen, n, dtype=t, scale=0.1) if case["bias"] else None
        if case["direction"] == "forward":
            state["residual"] = _randn(gen, rows, n, dtype=t) if case["residual"] else None
        else:
            state["dy"] = _randn(gen, rows, n, dtype=t)
            # what the forward pass kept: x W^T + b has unit spread
            state["preactivation"] = _randn(gen, rows, n, dtype=t) if case["activation"] != "none" else None
        return state
    b, sq, sk, h, hk, d = (case[n] for n in ("batch", "sq", "sk", "heads", "kv_heads", "dim"))
    if case["packed"]:  # views of one projection's output, heads of q, k and v side by side in each row
        rows = _randn(gen, b, sq, 3, h, d, dtype=t)
        state["q"], state["k"], state["v"] = rows[:, :, 0], rows[:, :, 1], rows[:, :, 2]
    else:
        state["q"], state["k"] = _randn(gen, b, sq, h, d, dtype=t), _randn(gen, b, sk, hk, d, dtype=t)
        state["v"] = _randn(gen, b, sk, hk, d, dtype=t)
    state["lengths"] = None
    if case["lengths"]:  # clips between a quarter and the whole of the padded length
        lengths = torch.randint(max(1, sk // 4), sk + 1, (b,), generator=gen, device="cuda", dtype=torch.int32)
        lengths[0] = sk
        state["lengths"] = lengths
    if case["direction"] == "backward":
        state["dout"] = _randn(gen, b, sq, h, d, dtype=t)
        out, state["lse"] = _plain_attention(case, state["q"], state["k"], state["v"], state["lengths"])
        state["out"] = out.to(t)
    return state


# ---------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------
def _run_own(s):
    from mlx_audio_amd import frontends as f

    case = s["case"]
    forward = case["direction"] == "forward"
    if case["op"] == "layer_norm":
        if forward:
            return f.layer_norm(s["x"], s["weight"], s["bias"], return_stats=True)
        return f.layer_norm_backward(s["dy"], s["x"], s["mean"], s["rstd"], s["weight"])
    if case["op"] == "linear":
        act = None if case["activation"] == "none" else case["activation"]
        if forward:
            return f.linear(s["x"], s["weight"], s["bias"], activation=act, residual=s["residual"],
                            return_preactivation=act is not None and case["rows"] > 64)
        dx, dweight, dbias = f.linear_backward(s["dy"], s["x"], s["weight"], activation=act,
                                               preactivation=s["preactivation"], bias_grad=case["bias"])
        return [dx, dweight, dbias] if case["bias"] else [dx, dweight]
    if forward:
        return f.attention(s["q"], s["k"], s["v"], causal=case["causal"], key_lengths=s["lengths"], return_lse=True)
    return f.attention_backward(s["dout"], s["q"], s["k"], s["v"], s["out"], s["lse"], causal=case["causal"],
                                key_lengths=s["lengths"])


def _run_plain(s):
    case = s["case"]
    t = _TYPES[case["dtype"]]
    forward = case["direction"] == "forward"
    if case["op"] == "layer_norm":
        x, w = s["x"].to(torch.float32), s["weight"].to(torch.float32)
        if forward:
            mean = x.mean(dim=-1)
            c = x - mean[:, None]
            rstd = torch.rsqrt((c * c).mean(dim=-1) + 1e-5)
            return (c * rstd[:, None] * w + s["bias"].to(torch.float32)).to(t), mean, rstd
        dy = s["dy"].to(torch.float32)
        xhat = (x - s["mean"][:, None]) * s["rstd"][:, None]
        g = dy * w
        dx = s["rstd"][:, None] * (g - g.mean(dim=-1, keepdim=True) - xhat * (g * xhat).mean(dim=-1, keepdim=True))
        # the sums over all rows are long ones
        return dx.to(t), (dy * xhat).sum(dim=0, dtype=torch.float64).float(), dy.sum(dim=0, dtype=torch.float64).float()
    if case["op"] == "linear":
        x, w = s["x"].to(torch.float32), s["weight"].to(torch.float32)
        if forward:
            z = torch.matmul(x, w.t())
            if s["bias"] is not None:
                z = z + s["bias"].to(torch.float32)
            y = _activate(z, case["activation"])
            if s["residual"] is not None:
                y = y + s["residual"].to(torch.float32)
            if case["activation"] != "none" and case["rows"] > 64:
                return y.to(t), z.to(t)
            return y.to(t)
        dz = s["dy"].to(torch.float32)
        if s["preactivation"] is not None:
            dz = dz * _derivative(s["preactivation"].to(torch.float32), case["activation"])
        out = [torch.matmul(dz, w).to(t), torch.matmul(dz.t(), x).to(t)]
        return out + [dz.sum(dim=0, dtype=torch.float64).float()] if case["bias"] else out
    if forward:
        out, lse = _plain_attention(case, s["q"], s["k"], s["v"], s["lengths"])
        return out.to(t), lse
    group = case["heads"] // case["kv_heads"]
    q, k, v = _per_head(s["q"]), _per_head(s["k"], group), _per_head(s["v"], group)
    dout, out = _per_head(s["dout"]), _per_head(s["out"])
    scale = 1.0 / math.sqrt(case["dim"])
    sc = torch.matmul(q, k.transpose(-1, -2).contiguous()) * scale
    seen = _visible(case, s["lengths"])
    if seen is not None:
        sc = sc.masked_fill(~seen, float("-inf"))
    lse = s["lse"][..., None]
    p = torch.exp(sc - torch.where(lse == float("-inf"), torch.zeros_like(lse), lse))
    dv = torch.matmul(p.transpose(-1, -2).contiguous(), dout)
    ds = p * (torch.matmul(dout, v.transpose(-1, -2).contiguous()) - (dout * out).sum(dim=-1, keepdim=True)) * scale
    dq = torch.matmul(ds, k)
    dk = torch.matmul(ds.transpose(-1, -2).contiguous(), q)
    if group > 1:
        dk = dk.unflatten(1, (case["kv_heads"], group)).sum(dim=2)
        dv = dv.unflatten(1, (case["kv_heads"], group)).sum(dim=2)
    return tuple(g.transpose(1, 2).contiguous().to(t) for g in (dq, dk, dv))


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------
def work(case):
    e = _SIZE[case["dtype"]]
    forward = case["direction"] == "forward"
    if case["op"] == "layer_norm":
        rows, dim = case["rows"], case["dim"]
        if forward:
            return {"bytes": 2 * rows * dim * e + 2 * dim * e + 8 * rows, "flops": 8 * rows * dim}
        return {"bytes": 3 * rows * dim * e + dim * e + 8 * rows + 8 * dim, "flops": 14 * rows * dim}
    if case["op"] == "linear":
        m, k, n = case["rows"], case["k"], case["n"]
        act = case["activation"] != "none"
        if forward:
            outs = 1 + (1 if act and m > 64 else 0) + (1 if case["residual"] else 0)
            return {"bytes": e * (m * k + n * k + outs * m * n + (n if case["bias"] else 0)), "flops": 2 * m * n * k}
        return {"bytes": e * (2 * m * k + 2 * n * k + (2 if act else 1) * m * n) + (4 * n if case["bias"] else 0),
                "flops": 4 * m * n * k}
    b, sq, sk, h, hk, d = (case[n] for n in ("batch", "sq", "sk", "heads", "kv_heads", "dim"))
    if case["lengths"]:
        # lengths are spread evenly over a quarter to the whole; the first is whole
        share = (1.0 + (b - 1) * 0.625) / b
    else:
        share = 1.0
    pairs = b * h * share * sq * sk
    if case["causal"]:
        full = max(0, sk - sq) * sq + min(sq, sk) * (min(sq, sk) + 1) / 2
        pairs = pairs * full / (sq * sk)
    qs, ks = b * sq * h * d * e, int(share * b * sk * hk * d * e)
    if forward:
        return {"bytes": 2 * qs + 2 * ks + 4 * b * h * sq, "flops": int(4 * d * pairs)}
    return {"bytes": 4 * qs + 2 * ks + 2 * b * sk * hk * d * e + 4 * b * h * sq, "flops": int(10 * d * pairs)}


# ---------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------
def _exact_layer_norm(case, s):
    x, w = s["x"].double(), s["weight"].double()
    n = case["dim"]
    if case["direction"] == "forward":
        mean = x.sum(-1) / n
        var = torch.square(x - mean.unsqueeze(-1)).sum(-1) / n
        rstd = 1.0 / torch.sqrt(var + 1e-5)
        return (x - mean.unsqueeze(-1)) * rstd.unsqueeze(-1) * w + s["bias"].double(), mean, rstd
    dy, rstd = s["dy"].double(), s["rstd"].double().unsqueeze(-1)
    h = (x - s["mean"].double().unsqueeze(-1)) * rstd
    g = dy * w
    dx = (g - g.sum(-1, keepdim=True) / n - h * ((g * h).sum(-1, keepdim=True) / n)) * rstd
    return dx, torch.einsum("rd,rd->d", dy, h), dy.sum(0)


def _exact_linear(case, s):
    x, w = s["x"].double(), s["weight"].double()
    act = case["activation"]
    half = math.sqrt(0.5)
    if case["direction"] == "forward":
        z = x @ w.T
        if s["bias"] is not None:
            z += s["bias"].double()
        if act == "gelu":
            y = z * 0.5 * torch.special.erfc(-z * half)
        elif act == "gelu_tanh":
            y = z * torch.sigmoid(2.0 * math.sqrt(2.0 / math.pi) * (z + 0.044715 * z.pow(3)))
        elif act == "relu":
            y = torch.where(z > 0, z, torch.zeros_like(z))
        else:
            y = z.clone()
        if s["residual"] is not None:
            y += s["residual"].double()
        return (y, z) if act != "none" and case["rows"] > 64 else y
    dz = s["dy"].double()
    if act != "none":
        z = s["preactivation"].double()
        if act == "gelu":
            slope = 0.5 * torch.special.erfc(-z * half) + z * torch.exp(-z.pow(2) / 2) * math.sqrt(0.5 / math.pi)
        elif act == "gelu_tanh":
            c = 2.0 * math.sqrt(2.0 / math.pi)
            sg = torch.sigmoid(c * (z + 0.044715 * z.pow(3)))
            slope = sg + z * sg * (1.0 - sg) * c * (1.0 + 3 * 0.044715 * z.pow(2))
        else:
            slope = (z > 0).double()
        dz = dz * slope
    out = [dz @ w, dz.T @ x]
    return out + [dz.sum(0)] if case["bias"] else out


def _exact_attention(case, s):
    b, sq, sk, h, hk, d = (case[n] for n in ("batch", "sq", "sk", "heads", "kv_heads", "dim"))
    group = h // hk
    ninf = float("-inf")
    forward = case["direction"] == "forward"
    q, k, v = s["q"], s["k"], s["v"]
    if forward:
        out = torch.zeros((b, sq, h, d), dtype=torch.float64, device=q.device)
        lse = torch.full((b, h, sq), ninf, dtype=torch.float64, device=q.device)
    else:
        dq = torch.zeros((b, sq, h, d), dtype=torch.float64, device=q.device)
        dk = torch.zeros((b, sk, hk, d), dtype=torch.float64, device=q.device)
        dv = torch.zeros((b, sk, hk, d), dtype=torch.float64, device=q.device)
    lens = [sk] * b if s["lengths"] is None else s["lengths"].tolist()
    for bi in range(b):
        n = lens[bi]
        if n == 0:
            continue
        hidden = None
        if case["causal"]:  # query i stands at position i + sk - sq
            hidden = torch.ones((sq, sk), dtype=torch.bool, device=q.device).triu(1 + sk - sq)[:, :n]
        for hi in range(h):
            qh, kh, vh = q[bi, :, hi].double(), k[bi, :n, hi // group].double(), v[bi, :n, hi // group].double()
            sc = qh @ kh.T / math.sqrt(d)
            if hidden is not None:
                sc[hidden] = ninf
            if forward:
                row = torch.logsumexp(sc, -1)
                empty = row == ninf
                p = torch.exp(sc - row.masked_fill(empty, 0.0).unsqueeze(-1))
                out[bi, :, hi] = p @ vh
                lse[bi, hi] = row
                continue
            row = s["lse"][bi, hi].double()
            p = torch.exp(sc - row.masked_fill(row == ninf, 0.0).unsqueeze(-1))
            do = s["dout"][bi, :, hi].double()
            delta = (do * s["out"][bi, :, hi].double()).sum(-1, keepdim=True)
            ds = p * (do @ vh.T - delta) / math.sqrt(d)
            dq[bi, :, hi] = ds @ kh
            dk[bi, :n, hi // group] += ds.T @ qh
            dv[bi, :n, hi // group] += p.T @ do
    return (out, lse) if forward else (dq, dk, dv)


def exact(case, seed):
    s = prepare(case, seed)
    return {"layer_norm": _exact_layer_norm, "linear": _exact_linear, "attention": _exact_attention}[case["op"]](case, s)
