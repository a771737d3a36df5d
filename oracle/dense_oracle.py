"""The dense operators (include/opus_dense.h) in numpy, 64 bits, from their formulas.  Test infrastructure only."""
import math

import numpy as np

_ERFC = np.frompyfunc(math.erfc, 1, 1)


def philox(counter, key, rounds=10):
    """Philox 4x32 of Salmon, Moraes, Dror, Shaw (SC'11): counter [..., 4] and key [2] of 32-bit values -> [..., 4]."""
    c = [np.asarray(counter[..., i], dtype=np.uint64) for i in range(4)]
    k = [int(key[0]), int(key[1])]
    low, by = np.uint64(0xFFFFFFFF), np.uint64(32)
    for _ in range(rounds):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> by) ^ c[1] ^ np.uint64(k[0]), b & low, (a >> by) ^ c[3] ^ np.uint64(k[1]), a & low]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return np.stack(c, -1).astype(np.uint32)


def keep(rows, cols, p, seed, offset=0, first_row=0):
    """[rows, cols]: 65536 / (65536 - round(65536 p)) where an element is kept, 0 where it is dropped."""
    k = int(round(p * 65536))
    if k == 0:
        return np.ones((rows, cols))
    units = -(-cols // 8)
    ctr = np.zeros((rows, units, 4), dtype=np.uint64)
    row = np.arange(first_row, first_row + rows, dtype=np.uint64)[:, None]
    ctr[..., 0] = np.arange(units, dtype=np.uint64)
    ctr[..., 1] = row & np.uint64(0xFFFFFFFF)
    ctr[..., 2] = row >> np.uint64(32)
    ctr[..., 3] = offset
    seed %= 2 ** 64
    words = philox(ctr, (seed & 0xFFFFFFFF, seed >> 32))
    bits = np.stack([words & 0xFFFF, words >> 16], -1).reshape(rows, units * 8)[:, :cols]
    return (bits >= k) * (65536.0 / (65536 - k) if k < 65536 else 0.0)


def act(z, name):
    """(value, derivative) of an activation."""
    if name == "none":
        return z, np.ones_like(z)
    if name == "relu":
        return np.maximum(z, 0), (z > 0).astype(np.float64)
    if name == "silu":
        s = 1 / (1 + np.exp(-z))
        return z * s, s * (1 + z * (1 - s))
    if name == "gelu":
        cdf = 0.5 * _ERFC(-z / math.sqrt(2)).astype(np.float64)
        return z * cdf, cdf + z * np.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    c = math.sqrt(2 / math.pi)
    t = np.tanh(c * (z + 0.044715 * z ** 3))
    return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)


def linear(x, w, bias=None, name="none", residual=None, kept=1.0):
    """-> (y, z)"""
    z = x @ w.T + (0.0 if bias is None else bias)
    return act(z, name)[0] * kept + (0.0 if residual is None else residual), z


def linear_backward(dy, x, w, z, name="none", kept=1.0):
    """-> (dx, dw, dbias, dz)"""
    dz = dy * kept * act(z, name)[1]
    return dz @ w, dz.T @ x, dz.sum(0), dz


def _norm(r, kind, eps):
    c = r - r.mean(-1, keepdims=True) if kind == "layer" else r
    rstd = 1 / np.sqrt((c * c).mean(-1, keepdims=True) + eps)
    return c * rstd, rstd


def _norm_backward(g, hat, rstd, kind):
    d = g - hat * (g * hat).mean(-1, keepdims=True)
    if kind == "layer":
        d = d - g.mean(-1, keepdims=True)
    return d * rstd


def residual_norm(x, block, weight=None, bias=None, kind="layer", eps=1e-5, post_weight=None, post_bias=None, gate=None,
                  scale=1.0, kept=1.0, dy=None, dstream=None):
    """[rows, width] each (gate too, already one row for each of x's) -> dict of y, stream and, for a dy or dstream,
    the gradients (dgate one row for each of x's)."""
    one = lambda v, d: np.full(x.shape[-1], d) if v is None else v           # noqa: E731
    w, b = one(weight, 1.0), one(bias, 0.0)
    g = np.ones_like(x) if gate is None else gate
    u = block
    if post_weight is not None:
        hhat, hrstd = _norm(block, kind, eps)
        u = hhat * post_weight + one(post_bias, 0.0)
    u = u * kept
    r = scale * x + g * u
    hat, rstd = _norm(r, kind, eps)
    out = {"y": hat * w + b, "stream": r}
    if dy is None and dstream is None:
        return out
    dy = np.zeros_like(x) if dy is None else dy
    dr = _norm_backward(dy * w, hat, rstd, kind) + (0.0 if dstream is None else dstream)
    out.update(dx=scale * dr, dweight=(dy * hat).sum(0), dbias=dy.sum(0), dgate=dr * u)
    du = dr * g * kept
    if post_weight is None:
        out["dblock"] = du
    else:
        out.update(dblock=_norm_backward(du * post_weight, hhat, hrstd, kind), dpost_weight=(du * hhat).sum(0),
                   dpost_bias=du.sum(0))
    return out
