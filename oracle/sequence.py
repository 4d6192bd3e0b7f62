"""Plain 64-bit forms of the sequence operators (gated scan, its gradients, AdamW) in numpy: test infrastructure, step by step from the formulas in include/apx.h."""
import numpy as np


def sigmoid(z):
    e = np.exp(-np.abs(z))
    return np.where(z >= 0, 1 / (1 + e), e / (1 + e))


def gated_scan(f, x, o=None, h0=None, reset=None, lens=None):
    """f, x, o [T, B, H] f64 -> y [T, B, H], states [T, B, H], what entered each step [T, B, H], h_last [B, H]"""
    T, B, H = f.shape
    h = np.zeros((B, H)) if h0 is None else h0.astype(np.float64).copy()
    y, hs, prev = np.zeros((T, B, H)), np.zeros((T, B, H)), np.zeros((T, B, H))
    for t in range(T):
        live = np.ones(B, bool) if lens is None else t < lens
        p = h if reset is None else np.where((reset[t] != 0)[:, None], 0.0, h)
        prev[t] = p
        with np.errstate(invalid="ignore"):      # (padding may hold anything)
            new = sigmoid(f[t]) * p + sigmoid(-f[t]) * x[t]
            out = new if o is None else new * sigmoid(o[t])
        h = np.where(live[:, None], new, h)
        y[t] = np.where(live[:, None], out, 0.0)
        hs[t] = h
    return y, hs, prev, h


def gated_scan_grad(f, x, dy, o=None, h0=None, reset=None, lens=None, dh_last=None):
    """df, dx, do, dh0 of sum(dy y) + sum(dh_last h_last), and the largest |g| on the way"""
    T, B, H = f.shape
    _, hs, prev, _ = gated_scan(f, x, o, h0, reset, lens)
    c = np.zeros((B, H)) if dh_last is None else dh_last.astype(np.float64).copy()
    df, dx, do = np.zeros((T, B, H)), np.zeros((T, B, H)), np.zeros((T, B, H))
    top = 0.0
    for t in range(T - 1, -1, -1):
        live = (np.ones(B, bool) if lens is None else t < lens)[:, None]
        with np.errstate(invalid="ignore"):
            a, n = sigmoid(f[t]), sigmoid(-f[t])
            s = 1.0 if o is None else sigmoid(o[t])
            g = dy[t] * s + c
            df[t] = np.where(live, g * (prev[t] - x[t]) * a * n, 0.0)
            dx[t] = np.where(live, g * n, 0.0)
            if o is not None:
                do[t] = np.where(live, dy[t] * hs[t] * s * sigmoid(-o[t]), 0.0)
            back = a * g if reset is None else np.where((reset[t] != 0)[:, None], 0.0, a * g)
        c = np.where(live, back, c)
        top = max(top, float(np.abs(np.where(live, g, 0.0)).max()) if g.size else 0.0)
    return df, dx, (None if o is None else do), c, top


# ------------------------------------------------------------------------------------------------ AdamW
BLOCK = 256
M_OFFSET, V_OFFSET = 904, 776


def layout(sizes):
    at, off = [], 0
    for n in sizes:
        at.append(off); off += -(-n // BLOCK) * BLOCK
    return at, off


def adamw(p, g, m, v, t, lr, beta1, beta2, eps, wd, factor):
    """one tensor's step on its moments (f64, any shape); t = the step's number from 1; factor = what the gradient is multiplied by.  Returns the new (p, m, v)."""
    g = g * factor
    m, v = beta1 * m + (1 - beta1) * g, beta2 * v + (1 - beta2) * g * g
    u = m / (1 - beta1 ** t) / (np.sqrt(v / (1 - beta2 ** t)) + eps)
    return p * (1 - lr * wd) - lr * u, m, v


def clip_factor(grads, scale, max_norm):
    n = abs(scale) * np.sqrt(sum(float((g.astype(np.float64) ** 2).sum()) for g in grads))
    return n, (scale if not max_norm else scale * min(1.0, max_norm / (n + 1e-6)))


def moments_f32(g, m, v, beta1, beta2, factor):
    """the moments in f32, every product and sum rounded by itself"""
    f = np.float32
    g = g.astype(f) * f(factor)
    return m * f(beta1) + g * f(1 - beta1), v * f(beta2) + (g * g) * f(1 - beta2)


def _mix(x):
    x = x.astype(np.uint64) & np.uint64(0xffffffff)
    x ^= x >> np.uint64(16)
    x = x * np.uint64(0x6A09E667) & np.uint64(0xffffffff)
    x ^= x >> np.uint64(15)
    x = x * np.uint64(0xBB67AE85) & np.uint64(0xffffffff)
    return x ^ (x >> np.uint64(16))


def noise(seed, t, at):
    one = lambda k: int(_mix(np.array([k & 0xffffffff], np.uint64))[0])
    key = np.uint64(one(one(seed) ^ one((seed >> 32) + 0x3C6EF373) ^ one(t + 0x54FF53A5)))
    at = at.astype(np.uint64)
    return _mix((at & np.uint64(0xffffffff)) ^ key ^ ((at >> np.uint64(32)) * np.uint64(0x3C6EF373) & np.uint64(0xffffffff)))


def values(offset, signed):
    """what the 256 codes stand for, in units of their block's scale"""
    c = np.arange(256)
    mag = c & 127 if signed else c
    v = np.where(mag == 0, 0.0, ((mag + offset).astype(np.uint32) << 20).view(np.float32).astype(np.float64))
    return np.where(signed & (c > 127), -v, v)


def decode(codes, scale, offset, signed):
    return (values(offset, signed)[codes].reshape(-1, BLOCK) * scale.astype(np.float64)[:, None]).reshape(-1)


def encode(w, bits, offset, signed):
    """codes and scales of f32 values [blocks of 256] with 16 random bits each (numpy f32 throughout)"""
    q = np.abs(w).astype(np.float32).reshape(-1, BLOCK)
    e = np.maximum((q.max(1).view(np.uint32) >> 23).astype(np.int64), 33)      # a scale of 2^-94 at least
    scale, inv = (e << 23).astype(np.uint32).view(np.float32), ((254 - e) << 23).astype(np.uint32).view(np.float32)
    q = (q * inv[:, None]).reshape(-1)
    least = np.float32(values(offset, signed)[1])
    r = bits.astype(np.uint32) << 4
    c = ((q.view(np.uint32) + r) >> 20).astype(np.int64) - offset
    small = ((r.astype(np.float32) * np.float32(least / (1 << 20))) < q) if signed else q > 0
    c = np.where(q < least, small.astype(np.int64), c)
    if signed:
        c = c + np.where((w < 0) & (c > 0), 128, 0)
    return c.astype(np.uint8), scale
