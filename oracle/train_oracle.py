"""CPU restatement of a training step's operators around its attention (test
infrastructure only): LayerNorm, embedding, cross-entropy and their gradients in
float64, and AdamW with moments in 32 bits (float32 arithmetic, product by product,
bit by bit) or in 8. include/skv.h states the formulas and the formats.
"""
from __future__ import annotations

import numpy as np

BLOCK = 128


def f64(x):
    return np.asarray(x, np.float64)


def layernorm(x, gamma, beta, eps=1e-5):
    """(y, mean, rstd)."""
    x = f64(x)
    mean = x.mean(-1)
    c = x - mean[:, None]
    rstd = 1 / np.sqrt((c * c).mean(-1) + eps)
    return c * rstd[:, None] * f64(gamma) + f64(beta), mean, rstd


def layernorm_backward(dy, x, gamma, mean, rstd, residual=None):
    """(dx, dgamma, dbeta)."""
    dy, x, gamma, mean, rstd = map(f64, (dy, x, gamma, mean, rstd))
    xh = (x - mean[:, None]) * rstd[:, None]
    g = dy * gamma
    dx = rstd[:, None] * (g - g.mean(-1, keepdims=True) - xh * (g * xh).mean(-1, keepdims=True))
    if residual is not None:
        dx = dx + f64(residual)
    return dx, (dy * xh).sum(0), dy.sum(0)


def embedding(tokens, table, scale=1.0, pos_table=None):
    tokens, table = np.asarray(tokens), f64(table)
    real = (tokens >= 0) & (tokens < len(table))
    out = np.where(real[:, None], scale * table[np.where(real, tokens, 0)], 0.0)
    if pos_table is not None:
        out = out + f64(pos_table)[np.arange(len(tokens)) % len(pos_table)]
    return out


def embedding_backward(dout, tokens, vocab, scale=1.0):
    tokens = np.asarray(tokens)
    real = (tokens >= 0) & (tokens < vocab)
    grad = np.zeros((vocab, np.shape(dout)[1]))
    np.add.at(grad, tokens[real], f64(dout)[real])
    return grad * scale


def cross_entropy(x, targets, grad_scale=1.0):
    """(loss, row losses, dx)."""
    x, targets = f64(x), np.asarray(targets)
    rows, vocab = x.shape
    real = (targets >= 0) & (targets < vocab)
    at = np.where(real, targets, 0)
    with np.errstate(invalid="ignore"):
        top = x.max(-1, keepdims=True)
        e = np.exp(x - top)
        total = e.sum(-1, keepdims=True)
        # the difference first: 1e30 + log(vocab) is 1e30 in 64 bits too
        row = (top[:, 0] - x[np.arange(rows), at]) + np.log(total)[:, 0]
        p = e / total
    p[np.arange(rows), at] -= 1
    count = max(1, int(real.sum()))
    row = np.where(real, row, 0.0)
    return row.sum() / count, row, np.where(real[:, None], p, 0.0) * grad_scale / count


# ---- AdamW -----------------------------------------------------------------

def moments(m, v, g, beta1, beta2):
    """The new moments in float32, every product and sum rounded."""
    f = np.float32
    m, v, g = (np.asarray(t, f) for t in (m, v, g))
    with np.errstate(over="ignore", invalid="ignore"):
        m = f(beta1) * m + f(1 - beta1) * g
        v = f(beta2) * v + f(1 - beta2) * (g * g)
    return m, v


def stepped(p, m, v, t, lr, beta1, beta2, eps, weight_decay):
    """The new weights in float64 from the new moments."""
    p, m, v = map(f64, (p, m, v))
    denom = np.sqrt(v / (1 - beta2 ** t)) + eps
    with np.errstate(divide="ignore", invalid="ignore"):
        return p * (1 - lr * weight_decay) - lr / (1 - beta1 ** t) * m / denom


def hashed(seed, t, n):
    """The 32 random bits of every place of a state."""
    low = 0xffffffff
    w = (seed * 0x9E3779B9 + t * 0x6A09E667) & low
    w = ((w ^ (w >> 15)) * 0xBB67AE85) & low
    key = w ^ (w >> 16)
    u = (np.arange(n, dtype=np.uint64) * np.uint64(0x9E3779B9) + np.uint64(key)) & np.uint64(low)
    u = ((u ^ (u >> np.uint64(15))) * np.uint64(0x6A09E667)) & np.uint64(low)
    return (u ^ (u >> np.uint64(16))).astype(np.uint32)


def grid(unsigned):
    """The magnitudes of y in code order: 127 of m, 256 of v."""
    i = np.arange(256 if unsigned else 127)
    e, f = i >> 3, i & 7
    low = -32 if unsigned else -9
    return np.where(e == 0, np.ldexp(f, low), np.ldexp(8.0 + f, e - 1 + low))


def store(x, bits, unsigned):
    """(codes, scale bytes) of float32 moments x, of whole blocks, with 16 random bits each:
    y's neighbours on the grid, and of 2^20 steps between them as many as its fixed-point
    distance from the lower one."""
    g = f64(np.asarray(x, np.float32)).reshape(-1, BLOCK)
    amax = np.abs(g).max(-1)
    bad = ~np.isfinite(amax)
    k = np.frexp(np.where(bad | (amax == 0), 1.0, amax))[1] - 1
    k = np.clip(np.where(amax == 0, -90, k), -90, 126)
    with np.errstate(invalid="ignore"):
        y = np.abs(np.ldexp(g, (-k if unsigned else 7 - k)[:, None]))
    y = np.where(bad[:, None], 0.0, y)
    gr = grid(unsigned)
    # the 20 bits behind the third mantissa bit; where y lies among the subnormals, those of
    # y + the smallest normal number, to which the sum is rounded in float32
    normal = gr[8]
    y32 = np.where(y < normal, f64((y + normal).astype(np.float32)) - normal, y)
    top = len(gr) - 1
    code = np.minimum(np.searchsorted(gr, y32, "right") - 1, top)
    step = np.where(code < 8, gr[1], np.ldexp(1.0, (code >> 3) - 1 + (-32 if unsigned else -9)))
    part = np.round((y32 - gr[code]) / step * 2 ** 20).astype(np.int64)
    r = np.asarray(bits, np.int64).reshape(g.shape) * 16 + 8
    code = np.minimum(code + (part + r >= 2 ** 20), top)
    if unsigned:
        code = np.where((g > 0) & (code == 0), 1, code)
    else:
        code = code + 128 * np.signbit(g)
    code = np.where(bad[:, None], 0, code).astype(np.uint8)
    return code.reshape(-1), np.where(bad, 255, k + 127).astype(np.uint8)


def values(code, byte, unsigned):
    """Codes back, in float64."""
    c = np.asarray(code).reshape(-1, BLOCK).astype(np.int64)
    k = np.asarray(byte).astype(np.int64) - 127
    gr = grid(unsigned)
    if unsigned:
        y = gr[c]
    else:
        y = np.append(gr, np.nan)[c & 127] * np.where(c >= 128, -1.0, 1.0)
    scale = np.where(np.asarray(byte) == 255, np.nan, np.ldexp(1.0, k if unsigned else k - 7))
    return (y * scale[:, None]).reshape(-1)
