"""Plain restatements in numpy, 64 bits, of the rotated append, the adapters per
request and the rules on logits, with the errors that the kernels may make."""
import numpy as np

E32 = 2.0 ** -24      # half a step of FP32, relative


def half_step(y):
    """Largest error of one rounding to FP16: 2^-11 of the value, 2^-25 below the normal range."""
    return np.maximum(2.0 ** -11 * np.abs(y), 2.0 ** -25)


def rope_table(positions, d, theta):
    i = np.arange(d // 2, dtype=np.float64)
    a = np.arange(positions, dtype=np.float64)[:, None] * np.float64(theta) ** (-2 * i / d)
    return np.stack((np.cos(a), np.sin(a)), 1).astype(np.float32)      # [p][2][d / 2]


def rotated(x, w, eps, cs):
    """Rows x [..., d] at a position with cs [2][d / 2]; w: norm weights or None.
    -> (64-bit result, error of doing the same in FP32).

    In FP32 the norm factor is off by at most (d + 8) e relative (the sum of d squares,
    a division, a square root), two products add 2 e, each product with a
    cosine or sine and their sum 2 e: (d / 2 + 12) e of |a cos| + |b sin|."""
    x = x.astype(np.float64)
    d = x.shape[-1]
    with np.errstate(invalid="ignore", over="ignore"):
        if w is not None:
            x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w.astype(np.float64)
        a, b = x[..., :d // 2], x[..., d // 2:]
        c, s = cs[0].astype(np.float64), cs[1].astype(np.float64)
        y = np.concatenate((a * c - b * s, b * c + a * s), -1)
        size = np.concatenate((np.abs(a * c) + np.abs(b * s), np.abs(b * c) + np.abs(a * s)), -1)
    return y, (d / 2 + 12) * E32 * size


def lora(x, A, B, scale, base):
    """x [n][K], A [r][K], B [N][r], base [n][N] -> (64-bit result, the largest error of the kernel).

    e = 2^-24.  h_j = sum_k A_jk x_k in FP32: (K + 2) e sum |A x|.  h_j as two FP16 parts of 11
    bits each behind a power of two that lifts the row's largest to 2^14 or more: 2^-22 |h_j|
    and 2^-39 of the largest.  The sum over 2 r products: (2 r + 2) e sum |B h|.  The
    products with the scale and the sum with base: 3 e; the rounding to FP16 half a step."""
    x, A, B, base = (t.astype(np.float64) for t in (x, A, B, base))
    h = x @ A.T
    dh = (A.shape[1] + 2) * E32 * (np.abs(x) @ np.abs(A).T) + 2.0 ** -22 * np.abs(h) + 2.0 ** -39 * np.abs(h).max(-1, keepdims=True)
    d = h @ B.T
    y = base + scale * d
    ad = np.abs(h) @ np.abs(B).T
    err = abs(scale) * (dh @ np.abs(B).T + (2 * A.shape[0] + 2) * E32 * ad) + 3 * E32 * (np.abs(base) + abs(scale) * ad)
    return y, err + half_step(np.abs(y) + err)


def rules(x, hist=(), rep=1.0, freq=0.0, pres=0.0, bias=(), mask=None):
    """One row of logits: FP32 operations, each rounded by itself. -> (FP32 row, best token)"""
    x = np.asarray(x).astype(np.float32)
    V = len(x)
    rep, freq, pres = (np.float32(v) for v in (rep, freq, pres))
    hist = np.asarray(hist, np.int64)
    hist = hist[(hist >= 0) & (hist < V)]
    with np.errstate(all="ignore"):
        t, n = np.unique(hist, return_counts=True)
        l = x[t]
        l = np.where(l > 0, l / rep, l * rep)
        x[t] = (l - freq * n.astype(np.float32)) - pres
        for k, v in bias:
            if 0 <= k < V:
                x[k] = x[k] + np.float32(v)
    if mask is not None:
        x = np.where(mask, x, np.float32(-np.inf))
    y = np.where(np.isnan(x), -np.inf, x)
    return x, int(np.argmax(y)) if V and y.max() > -np.inf else 0
