"""The operators of the transformer blocks behind the encoder stem: layer normalisation, the linear
layer with bias, activation and residual in its epilogue, and attention, each with its backward
pass (the blocks `AudioEncoder.__call__` runs after the stem, models/whisper/layers/).

Element types are float32, float16 and bfloat16; every sum, statistic and intermediate value is
float32, and results are rounded once.  Tensors may be views: rows (the last axis) must be
contiguous and the leading axes of `layer_norm` / `linear` inputs collapse to rows of one stride,
anything else is copied first.  Host arrays (lists of key_lengths among them) are moved to the GPU by
a copy that waits.  With operands on the device nothing synchronises: work is enqueued on the current
stream and can be captured into a graph.

These functions record no autograd graph: the gradients come from the `*_backward` functions.
Inputs that require a gradient are refused while gradients are enabled (wrap the calls in
`torch.no_grad()`), and so are inputs that carry a tangent of forward-mode differentiation: neither
is lost silently.
"""

from __future__ import annotations

import ctypes
import math

import numpy as np
import torch
from torch.autograd import forward_ad

from .. import _lib
from .._runtime import require_gpu

_DTYPES = {torch.float32: _lib.F32, torch.float16: _lib.F16, torch.bfloat16: _lib.BF16}
_INTEGERS = (torch.uint8, torch.int8, torch.int16, torch.int32, torch.int64)
_ACTIVATIONS = {None: _lib.ACT_NONE, "gelu": _lib.ACT_GELU, "gelu_tanh": _lib.ACT_GELU_TANH, "relu": _lib.ACT_RELU}


def _operands(**given) -> dict:
    """The given arrays as tensors of a supported type that need no gradient, without the absent ones."""
    out = {}
    duals = getattr(forward_ad, "_current_level", 0) >= 0  # (inside a level; asking each tensor takes a microsecond)
    for name, x in given.items():
        if x is None:
            continue
        if not isinstance(x, torch.Tensor):
            x = torch.as_tensor(np.asarray(x))
        if x.dtype not in _DTYPES:
            raise ValueError(f"{name} must be float32, float16 or bfloat16, got {x.dtype}")
        if x.requires_grad and torch.is_grad_enabled():
            raise RuntimeError(f"{name} requires a gradient, which this function does not record: call the "
                               "*_backward function for it, under torch.no_grad()")
        if duals and forward_ad.unpack_dual(x).tangent is not None:
            raise RuntimeError(f"{name} carries a tangent, which this function does not propagate: pass "
                               "torch.autograd.forward_ad.unpack_dual(x).primal")
        if x.is_neg():  # (a view with its sign pending, as of a conjugate's imaginary part)
            x = x.resolve_neg()
        out[name] = x
    return out


def _same_type(ops: dict, names) -> torch.dtype:
    dtype = ops[names[0]].dtype
    for n in names:
        if n in ops and ops[n].dtype != dtype:
            raise ValueError("expected one type, got " + ", ".join(f"{n} {ops[n].dtype}" for n in names if n in ops))
    return dtype


def _to_device(ops: dict) -> torch.device:
    """Moves host tensors to the device of the others (the current one if all are host tensors)."""
    device, host = None, []
    for name, x in ops.items():
        if x.device.type != "cuda":
            host.append(name)
        elif device is None:
            device = x.device
        elif x.device != device:
            raise ValueError(f"tensors on different devices: {device}, {x.device}")
    if device is None:
        require_gpu()
        device = torch.device("cuda", torch.cuda.current_device())
    for name in host:
        ops[name] = ops[name].to(device)
    return device


def _call(fn, device: torch.device, *args) -> None:
    """Enqueues on the device's current stream (the last argument of every entry point)."""
    index = device.index
    if index == torch.cuda.current_device():
        _lib.check(fn(*args, torch._C._cuda_getCurrentRawStream(index)))
    else:
        with torch.cuda.device(index):
            _lib.check(fn(*args, torch._C._cuda_getCurrentRawStream(index)))


def _rows(x: torch.Tensor):
    """x as (tensor, rows, row stride): last axis contiguous, leading axes collapsed."""
    dim = x.shape[-1]
    if dim > 1 and x.stride(-1) != 1:
        x = x.contiguous()
    if x.dim() != 2:
        x = x.reshape(-1, dim) if x.numel() else x.new_empty((math.prod(x.shape[:-1]), dim))
    rows = x.shape[0]
    return x, rows, (x.stride(0) if rows > 1 else dim)


def _ptr(x):
    return None if x is None else x.data_ptr()


def _check_vector(x, name: str, n: int, dtype: torch.dtype) -> None:
    if x is None:
        return
    if x.shape != (n,):
        raise ValueError(f"{name} must have shape ({n},), got {tuple(x.shape)}")
    if x.dtype not in (dtype, torch.float32):
        raise ValueError(f"{name} must be float32 or {dtype}, got {x.dtype}")


def _check_norm(x, weight, bias) -> None:
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"x must have a last axis of at least one element, got shape {tuple(x.shape)}")
    _check_vector(weight, "weight", x.shape[-1], x.dtype)
    _check_vector(bias, "bias", x.shape[-1], x.dtype)
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise ValueError(f"expected one type, got weight {weight.dtype}, bias {bias.dtype}")


def layer_norm(x, weight=None, bias=None, eps: float = 1e-5, return_stats: bool = False):
    """Layer normalisation over the last axis: (x - mean) / sqrt(variance + eps) * weight + bias.

    x [..., D] -> y [..., D] of x's type; weight and bias [D], float32 or x's type, either may be
    None.  With return_stats also the rows' mean and 1 / sqrt(variance + eps), float32 [...], which
    `layer_norm_backward` takes.  One launch that reads x once.
    """
    ops = _operands(x=x, weight=weight, bias=bias)
    _check_norm(ops["x"], ops.get("weight"), ops.get("bias"))
    if not eps >= 0.0:
        raise ValueError(f"eps must not be negative (got {eps})")
    device = _to_device(ops)
    x, w, b = ops["x"], ops.get("weight"), ops.get("bias")
    w = None if w is None else w.contiguous()
    b = None if b is None else b.contiguous()
    flat, rows, stride = _rows(x)
    y = torch.empty_like(x, memory_format=torch.contiguous_format)
    mean = rstd = None
    if return_stats:
        mean = flat.new_empty(x.shape[:-1], dtype=torch.float32)
        rstd = torch.empty_like(mean)
    params = w if w is not None else b if b is not None else flat
    _call(_lib.lib().mia_layer_norm, device, flat.data_ptr(), rows, x.shape[-1], stride, _DTYPES[x.dtype], _ptr(w),
          _ptr(b), _DTYPES[params.dtype], float(eps), y.data_ptr(), _ptr(mean) if rows else None,
          _ptr(rstd) if rows else None)
    return (y, mean, rstd) if return_stats else y


def layer_norm_backward(dy, x, mean, rstd, weight=None):
    """Gradients of `layer_norm` from the statistics its forward call returned.

    dy and x [..., D] of one type -> (dx of that type, dweight, dbias): the vectors are sums over
    all rows and stay in float32; without a weight they are None (a bias alone has the gradient
    dy summed over its rows).  The sums have a fixed order: two calls give the same bits.
    """
    ops = _operands(dy=dy, x=x, mean=mean, rstd=rstd, weight=weight)
    dy, x, weight = ops["dy"], ops["x"], ops.get("weight")
    _check_norm(x, weight, None)
    _same_type(ops, ("dy", "x"))
    if dy.shape != x.shape:
        raise ValueError(f"dy must have x's shape {tuple(x.shape)}, got {tuple(dy.shape)}")
    for name in ("mean", "rstd"):
        if ops[name].dtype != torch.float32 or ops[name].shape != x.shape[:-1]:
            raise ValueError(f"{name} must be float32 of shape {tuple(x.shape[:-1])}, "
                             f"got {ops[name].dtype} {tuple(ops[name].shape)}")
    device = _to_device(ops)
    flat, rows, stride = _rows(ops["x"])
    gflat, _, gstride = _rows(ops["dy"])
    mean, rstd = ops["mean"].contiguous(), ops["rstd"].contiguous()
    w = None if weight is None else ops["weight"].contiguous()
    dim = x.shape[-1]
    dx = flat.new_empty(x.shape)
    dw = db = ws = None
    lib = _lib.lib()
    need = 0
    if w is not None:
        dw = flat.new_empty((dim,), dtype=torch.float32)
        db = torch.empty_like(dw)
        need = lib.mia_layer_norm_backward_workspace_bytes(rows, dim)
        ws = flat.new_empty((need,), dtype=torch.uint8)
    _call(lib.mia_layer_norm_backward, device, gflat.data_ptr(), gstride, flat.data_ptr(), stride, mean.data_ptr(),
          rstd.data_ptr(), rows, dim, _DTYPES[x.dtype], _ptr(w), _DTYPES[(flat if w is None else w).dtype],
          dx.data_ptr(), _ptr(dw), _ptr(db), _ptr(ws), need)
    return dx, dw, db


def _check_linear(x, weight, activation) -> None:
    if activation not in _ACTIVATIONS:
        raise ValueError(f"Unknown activation: {activation!r}. Supported: None, 'gelu', 'gelu_tanh', 'relu'")
    if weight.dim() != 2 or min(weight.shape) < 1:
        raise ValueError(f"weight must be (out, in) with at least one element each, got {tuple(weight.shape)}")
    if x.dim() < 1 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"x must have a last axis of {weight.shape[1]} elements, got shape {tuple(x.shape)}")


def linear(x, weight, bias=None, activation=None, residual=None, return_preactivation: bool = False):
    """The linear layer with its epilogue: activation(x @ weight.T + bias) + residual.

    x [..., in], weight [out, in], residual [..., out] of one type; bias [out] of that type or
    float32.  activation: None, "gelu" (erf), "gelu_tanh" or "relu".  Returns y [..., out] of x's
    type; with return_preactivation also x @ weight.T + bias, which `linear_backward` takes.
    Products of two-byte types accumulate in float32 on the matrix cores; float32 runs on the
    float32 matrix instruction.
    """
    ops = _operands(x=x, weight=weight, bias=bias, residual=residual)
    x, weight, bias, residual = ops["x"], ops["weight"], ops.get("bias"), ops.get("residual")
    _check_linear(x, weight, activation)
    dtype = _same_type(ops, ("x", "weight", "residual"))
    n, k = weight.shape
    _check_vector(bias, "bias", n, dtype)
    shape = x.shape[:-1] + (n,)
    if residual is not None and residual.shape != shape:
        raise ValueError(f"residual must have shape {tuple(shape)}, got {tuple(residual.shape)}")
    device = _to_device(ops)
    flat, rows, stride = _rows(ops["x"])
    w, _, wstride = _rows(ops["weight"])
    b = None if bias is None else ops["bias"].contiguous()
    r, rstride = None, 0
    if residual is not None:
        r, _, rstride = _rows(ops["residual"])
    y = flat.new_empty(shape)
    z = torch.empty_like(y) if return_preactivation else None
    lib = _lib.lib()
    need = lib.mia_linear_workspace_bytes(rows, k, n, _DTYPES[dtype])
    ws = flat.new_empty((need,), dtype=torch.uint8) if need else None
    _call(lib.mia_linear, device, flat.data_ptr(), stride, w.data_ptr(), wstride, _ptr(b),
          _DTYPES[(flat if b is None else b).dtype], _ptr(r), rstride, _ACTIVATIONS[activation], rows, k, n,
          _DTYPES[dtype], y.data_ptr(), _ptr(z), _ptr(ws), need)
    return (y, z) if return_preactivation else y


def linear_backward(dy, x, weight, activation=None, preactivation=None, input_grad: bool = True,
                    weight_grad: bool = True, bias_grad: bool = True):
    """Gradients of `linear`: with dz = dy * activation'(preactivation),
    (dx = dz @ weight, dweight = dz.T @ x, dbias = dz summed over its rows).

    dy [..., out], x [..., in], weight [out, in] and preactivation [..., out] (what the forward call
    returned; needed for an activation) of one type.  dx and dweight have that type, dbias is
    float32; a gradient not asked for is None.  The residual's gradient is dy itself.  For the two
    products dz is rounded to the operands' type: in float16 to multiples of 2^-24 at the finest, as
    dy itself is, so a dy below 1e-4 wants a scaled loss.
    """
    ops = _operands(dy=dy, x=x, weight=weight, preactivation=preactivation)
    dy, x, weight, z = ops["dy"], ops["x"], ops["weight"], ops.get("preactivation")
    _check_linear(x, weight, activation)
    dtype = _same_type(ops, ("dy", "x", "weight", "preactivation"))
    n, k = weight.shape
    shape = x.shape[:-1] + (n,)
    if dy.shape != shape:
        raise ValueError(f"dy must have shape {tuple(shape)}, got {tuple(dy.shape)}")
    if activation is not None:
        if z is None:
            raise ValueError("the backward pass of an activation needs the preactivation")
        if z.shape != shape:
            raise ValueError(f"preactivation must have shape {tuple(shape)}, got {tuple(z.shape)}")
    device = _to_device(ops)
    flat, rows, stride = _rows(ops["x"])
    w, _, wstride = _rows(ops["weight"])
    g, _, gstride = _rows(ops["dy"])
    zf, zstride = None, 0
    if activation is not None:
        zf, _, zstride = _rows(ops["preactivation"])
    dx = flat.new_empty(x.shape) if input_grad else None
    dw = flat.new_empty((n, k)) if weight_grad else None
    db = flat.new_empty((n,), dtype=torch.float32) if bias_grad else None
    lib = _lib.lib()
    act = _ACTIVATIONS[activation]
    need = lib.mia_linear_backward_workspace_bytes(rows, k, n, _DTYPES[dtype], act)
    ws = flat.new_empty((need,), dtype=torch.uint8) if need else None
    _call(lib.mia_linear_backward, device, g.data_ptr(), gstride, flat.data_ptr(), stride, w.data_ptr(), wstride,
          _ptr(zf), zstride, act, rows, k, n, _DTYPES[dtype], _ptr(dx) if rows else None, _ptr(dw), _ptr(db), _ptr(ws),
          need)
    return dx, dw, db


def _check_attention(q, k, v, scale) -> float:
    for name, x in (("q", q), ("k", k), ("v", v)):
        if x.dim() != 4:
            raise ValueError(f"{name} must be [batch, length, heads, dim], got shape {tuple(x.shape)}")
    B, _, H, D = q.shape
    if k.shape != v.shape:
        raise ValueError(f"k and v must have one shape, got {tuple(k.shape)} and {tuple(v.shape)}")
    if k.shape[0] != B or k.shape[3] != D:
        raise ValueError(f"q {tuple(q.shape)} and k {tuple(k.shape)} must agree in batch and dim")
    if H < 1 or k.shape[2] < 1 or H % k.shape[2]:
        raise ValueError(f"the number of query heads ({H}) must be a multiple of the number of key heads ({k.shape[2]})")
    if D < 1:
        raise ValueError("dim must be positive")
    if D > 128:
        raise NotImplementedError(f"head dimensions beyond 128 are not supported (got {D})")
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    if not 0.0 < scale < 2.3e38:  # (what float32 exponents to base 2 can be taken with)
        raise ValueError(f"scale must be positive and finite (got {scale})")
    return scale


def _check_lengths(lengths, batch: int, keys: int):
    """key_lengths as an int32 tensor (host or device); host values are checked."""
    if not isinstance(lengths, torch.Tensor):
        lengths = torch.as_tensor(np.asarray(lengths))
    if lengths.shape != (batch,) or lengths.dtype not in _INTEGERS:
        raise ValueError(f"key_lengths must be {batch} integers, got {lengths.dtype} {tuple(lengths.shape)}")
    if not lengths.is_cuda and batch and not 0 <= int(lengths.min()) <= int(lengths.max()) <= keys:
        raise ValueError(f"key_lengths must lie in 0 .. {keys}")
    if lengths.dtype != torch.int32:
        lengths = lengths.to(torch.int64).clamp(0, keys).to(torch.int32)  # (keys need not fit the given type)
    return lengths.contiguous()


def _heads(x: torch.Tensor) -> torch.Tensor:
    return x if x.shape[-1] == 1 or x.stride(-1) == 1 else x.contiguous()


def _strides(x: torch.Tensor):
    # (an axis of one element may have any stride)
    return (ctypes.c_int64 * 3)(*(st if n > 1 else 0 for n, st in zip(x.shape, x.stride()[:3])))


def _attention_desc(q, k, v, causal, scale) -> _lib.AttentionDesc:
    return _lib.AttentionDesc(_DTYPES[q.dtype], q.shape[0], q.shape[1], k.shape[1], q.shape[2], k.shape[2], q.shape[3],
                              int(bool(causal)), scale, _strides(q), _strides(k), _strides(v))


def attention(q, k, v, causal: bool = False, key_lengths=None, scale=None, return_lse: bool = False):
    """softmax(scale q k^T) v for every batch item and head.

    q [B, Sq, H, D], k and v [B, Sk, Hk, D] of one type, D <= 128, H a multiple of Hk (query head h
    uses key head h // (H // Hk)); any strides with D contiguous, so heads may be slices of one
    projection's rows.  scale defaults to 1 / sqrt(D).  key_lengths [B]: keys at and behind an item's
    length are neither seen nor read (padding may hold anything); values are brought into 0 .. Sk.
    causal: query i sees keys j <= i + Sk - Sq.  A query that sees no key gets zeros.  A value that
    is not finite in a key or value row which some query of a causal call sees may reach other
    queries.

    Returns out [B, Sq, H, D], contiguous; with return_lse also the logarithm of each row's sum of
    exponentials, float32 [B, H, Sq] (-inf where no key is seen), which `attention_backward` takes.
    Few queries over many keys (a decoding step) are split along the keys and joined.  The
    probabilities of two-byte types are rounded to that type for the product with v (relative eps / 2;
    float16 at least 2^-25 of a row's largest), except with at most 64 queries: those go in as the
    rounded value and the rest, itself rounded (eps / 2 squared, and the same 2^-25).
    """
    ops = _operands(q=q, k=k, v=v)
    _same_type(ops, ("q", "k", "v"))
    scale = _check_attention(ops["q"], ops["k"], ops["v"], scale)
    B, Sq, H, D = ops["q"].shape
    if key_lengths is not None:
        ops["key_lengths"] = _check_lengths(key_lengths, B, ops["k"].shape[1])
    device = _to_device(ops)
    q, k, v = (_heads(ops[n]) for n in ("q", "k", "v"))
    lengths = ops.get("key_lengths")
    out = q.new_empty((B, Sq, H, D))
    lse = q.new_empty((B, H, Sq), dtype=torch.float32) if return_lse else None
    desc = _attention_desc(q, k, v, causal, scale)
    lib = _lib.lib()
    need = lib.mia_attention_workspace_bytes(ctypes.byref(desc))
    ws = q.new_empty((need,), dtype=torch.uint8) if need else None
    _call(lib.mia_attention, device, ctypes.byref(desc), q.data_ptr(), k.data_ptr(), v.data_ptr(), _ptr(lengths),
          out.data_ptr(), _ptr(lse), _ptr(ws), need)
    return (out, lse) if return_lse else out


def attention_backward(dout, q, k, v, out, lse, causal: bool = False, key_lengths=None, scale=None):
    """Gradients (dq, dk, dv) of `attention` from its results `out` and `lse`.

    dout and out [B, Sq, H, D], lse float32 [B, H, Sq]; the other arguments as in the forward call.
    The probabilities are recomputed, nothing of size Sq x Sk is kept.  dk and dv are summed over the
    query heads that share a key head, and zero behind a length.  For the products the
    probabilities and their gradients are rounded to the operands' type (in dq with at most 64
    queries: carried in two parts); in float16 both are taken times powers of two first, worked out
    from the largest norms of v and dout, so that they neither overflow nor lose bits by being small.
    """
    ops = _operands(dout=dout, q=q, k=k, v=v, out=out, lse=lse)
    _same_type(ops, ("dout", "q", "k", "v", "out"))
    scale = _check_attention(ops["q"], ops["k"], ops["v"], scale)
    B, Sq, H, D = ops["q"].shape
    for name in ("dout", "out"):
        if ops[name].shape != ops["q"].shape:
            raise ValueError(f"{name} must have q's shape {tuple(ops['q'].shape)}, got {tuple(ops[name].shape)}")
    if ops["lse"].dtype != torch.float32 or ops["lse"].shape != (B, H, Sq):
        raise ValueError(f"lse must be float32 of shape {(B, H, Sq)}, got {ops['lse'].dtype} {tuple(ops['lse'].shape)}")
    if key_lengths is not None:
        ops["key_lengths"] = _check_lengths(key_lengths, B, ops["k"].shape[1])
    device = _to_device(ops)
    dout, q, k, v, out = (_heads(ops[n]) for n in ("dout", "q", "k", "v", "out"))
    lse, lengths = ops["lse"].contiguous(), ops.get("key_lengths")
    dq, dk, dv = q.new_empty((B, Sq, H, D)), k.new_empty(k.shape), k.new_empty(k.shape)
    desc = _attention_desc(q, k, v, causal, scale)
    lib = _lib.lib()
    need = lib.mia_attention_backward_workspace_bytes(ctypes.byref(desc))
    ws = q.new_empty((need,), dtype=torch.uint8) if need else None
    _call(lib.mia_attention_backward, device, ctypes.byref(desc), dout.data_ptr(), _strides(dout), q.data_ptr(),
          k.data_ptr(), v.data_ptr(), out.data_ptr(), _strides(out), lse.data_ptr(), _ptr(lengths), dq.data_ptr(),
          dk.data_ptr(), dv.data_ptr(), _ptr(ws), need)
    return dq, dk, dv
