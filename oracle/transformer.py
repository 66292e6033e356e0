"""Plain definitions of the operators behind the encoder stem, in float64: layer normalisation, the
linear layer with its epilogue, and attention, with their gradients (test infrastructure)."""
import numpy as np
from scipy.special import erfc


def layer_norm(x, w=None, b=None, eps=1e-5):
    mean = x.mean(-1)
    c = x - mean[..., None]
    rstd = 1.0 / np.sqrt((c * c).mean(-1) + eps)
    y = c * rstd[..., None]
    if w is not None:
        y = y * w
    if b is not None:
        y = y + b
    return y, mean, rstd


def layer_norm_backward(dy, x, mean, rstd, w=None):
    h = (x - mean[..., None]) * rstd[..., None]
    g = dy if w is None else dy * w
    dx = rstd[..., None] * (g - g.mean(-1, keepdims=True) - h * (g * h).mean(-1, keepdims=True))
    axes = tuple(range(x.ndim - 1))
    return dx, (dy * h).sum(axes), dy.sum(axes)


def activate(z, activation):
    if activation == "gelu":
        return 0.5 * z * erfc(-z / np.sqrt(2.0))
    if activation == "gelu_tanh":
        return 0.5 * z * (1.0 + np.tanh(np.sqrt(2.0 / np.pi) * (z + 0.044715 * z ** 3)))
    if activation == "relu":
        return np.where(z < 0, 0.0, z)
    return z


def derivative(z, activation):
    if activation == "gelu":
        return 0.5 * erfc(-z / np.sqrt(2.0)) + z * np.exp(-0.5 * z * z) / np.sqrt(2.0 * np.pi)
    if activation == "gelu_tanh":
        c = np.sqrt(2.0 / np.pi)
        t = np.tanh(c * (z + 0.044715 * z ** 3))
        return 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * c * (1.0 + 3 * 0.044715 * z * z)
    if activation == "relu":
        return np.where(z > 0, 1.0, 0.0)
    return np.ones_like(z)


def linear(x, w, b=None, activation=None, residual=None):
    z = x @ w.T
    if b is not None:
        z = z + b
    y = activate(z, activation)
    return (y if residual is None else y + residual), z


def linear_backward(dy, x, w, activation=None, z=None):
    dz = dy if activation is None else dy * derivative(z, activation)
    n, k = w.shape
    return dz @ w, dz.reshape(-1, n).T @ x.reshape(-1, k), dz.reshape(-1, n).sum(0)


def _visible(sq, sk, causal, length):
    seen = np.ones((sq, sk), bool)
    if causal:
        seen &= np.arange(sk)[None, :] <= np.arange(sq)[:, None] + (sk - sq)
    return seen & (np.arange(sk)[None, :] < length)


def attention(q, k, v, causal=False, lengths=None, scale=None):
    """q [B, Sq, H, D], k and v [B, Sk, Hk, D] -> (out [B, Sq, H, D], lse [B, H, Sq])."""
    B, Sq, H, D = q.shape
    Sk, group = k.shape[1], H // k.shape[2]
    scale = 1.0 / np.sqrt(D) if scale is None else scale
    out, lse = np.zeros(q.shape), np.full((B, H, Sq), -np.inf)
    for b in range(B):
        seen = _visible(Sq, Sk, causal, Sk if lengths is None else lengths[b])
        rows, cols = np.nonzero(seen.any(1))[0], np.nonzero(seen.any(0))[0]
        if not len(rows):
            continue
        s_seen = seen[np.ix_(rows, cols)]
        for h in range(H):
            s = scale * (q[b, rows, h] @ k[b, cols, h // group].T)
            s = np.where(s_seen, s, -np.inf)
            top = s.max(1, keepdims=True)
            p = np.exp(s - top)
            total = p.sum(1, keepdims=True)
            out[b, rows, h] = (p / total) @ v[b, cols, h // group]
            lse[b, h, rows] = (top + np.log(total))[:, 0]
    return out, lse


def attention_backward(dout, q, k, v, causal=False, lengths=None, scale=None):
    """Gradients of attention with respect to q, k and v."""
    B, Sq, H, D = q.shape
    Sk, group = k.shape[1], H // k.shape[2]
    scale = 1.0 / np.sqrt(D) if scale is None else scale
    out, lse = attention(q, k, v, causal, lengths, scale)
    dq, dk, dv = np.zeros(q.shape), np.zeros(k.shape), np.zeros(v.shape)
    for b in range(B):
        seen = _visible(Sq, Sk, causal, Sk if lengths is None else lengths[b])
        rows, cols = np.nonzero(seen.any(1))[0], np.nonzero(seen.any(0))[0]
        if not len(rows):
            continue
        s_seen = seen[np.ix_(rows, cols)]
        for h in range(H):
            hk = h // group
            qq, kk, vv, do = q[b, rows, h], k[b, cols, hk], v[b, cols, hk], dout[b, rows, h]
            p = np.where(s_seen, np.exp(np.where(s_seen, scale * (qq @ kk.T), -np.inf) - lse[b, h, rows][:, None]), 0.0)
            dv[b, cols, hk] += p.T @ do
            ds = p * (do @ vv.T - (do * out[b, rows, h]).sum(1, keepdims=True)) * scale
            dq[b, rows, h] += ds @ kk
            dk[b, cols, hk] += ds.T @ qq
    return dq, dk, dv
