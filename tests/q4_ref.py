"""The 4-bit cache and its operators restated in numpy: the format in fp32 as it is defined, everything else in 64 bits."""
import numpy as np

BLOCK = 32
F = np.float32


def bf16(x):
    """fp32 values rounded to bf16, half to even (finite ones)."""
    u = np.asarray(x, dtype=F).view(np.uint32).astype(np.uint64)
    return ((u + 0x7FFF + ((u >> 16) & 1)) & 0xFFFF0000).astype(np.uint32).view(F)


def stored(x):
    """What the cache gives back for rows of fp32 values."""
    x = np.where(np.isnan(x), F(0), x.astype(F))
    b = x.reshape(x.shape[:-1] + (x.shape[-1] // BLOCK, BLOCK))
    most = np.abs(b).max(-1)
    with np.errstate(over="ignore", invalid="ignore"):
        s = np.where(np.isinf(most), F(np.inf), bf16(np.where(np.isinf(most), F(0), most) * F(1.0 / 7.0)))
        s = np.clip(s, F(2.0 ** -17), F(2.0 ** 13)).astype(F)
        code = np.clip(np.rint((b / s[..., None]).astype(F)), -7, 7)
    s = np.where(most > 0, s, F(0))
    return (code.astype(F) * s[..., None]).astype(F).reshape(x.shape)


def rotate32(x, c, s):
    """Interleaved pairs in fp32, every product and sum rounded."""
    y = np.empty_like(x)
    y[..., ::2] = x[..., ::2] * c - x[..., 1::2] * s
    y[..., 1::2] = x[..., ::2] * s + x[..., 1::2] * c
    return y


def rotate64(x, c, s):
    x, c, s = x.astype(np.float64), c.astype(np.float64), s.astype(np.float64)
    y = np.empty_like(x)
    y[..., ::2] = x[..., ::2] * c - x[..., 1::2] * s
    y[..., 1::2] = x[..., ::2] * s + x[..., 1::2] * c
    return y


def attend(K, V, qkv, starts, lens, pos, cos, sin, H, window=0, acc=None):
    """K, V [B][G][maxSeq][hd]: values in the cache, changed in place.  Returns out rows (NaN where none is written), the accumulated
    weights (NaN where none is written) and bounds of both errors.

    The bounds.  Operands carry 22 bits or more and sums are fp32, so a score is off by at most 2^-21 of A, the largest sum of its terms' magnitudes;
    a weight then by 2·2^-21·A + 2^-20 of itself (exponential, denominator and the sums over rows), an output by that times the largest value."""
    B, G, S, hd = K.shape
    R = H // G
    M = qkv.shape[0]
    out = np.full((M, H * hd), np.nan)
    tol = np.zeros((M, 1))
    weights = np.full((B, G, S), np.nan)
    wtol = np.zeros((B, G, S))
    for b in range(B):
        first, n, p0 = int(starts[b]), int(lens[b]), int(pos[b])
        T = int(starts[b + 1]) - first
        if n < 0 or n >= S or p0 < 0 or p0 >= cos.shape[0]:
            continue
        T = max(0, min(T, S - n, cos.shape[0] - p0))
        x = qkv[first:first + T].reshape(T, H + 2 * G, hd)
        c, s = cos[p0:p0 + T, None], sin[p0:p0 + T, None]
        q = rotate64(x[:, :H], c, s)
        K[b, :, n:n + T] = stored(rotate32(x[:, H:H + G], c, s)).transpose(1, 0, 2)
        V[b, :, n:n + T] = stored(x[:, H + G:]).transpose(1, 0, 2)
        if acc is not None:
            weights[b, :, :n + T] = 0.0
            weights[b, :, :n] = acc[b, :, :n]
            wtol[b, :, :n] = 2.0 ** -23 * np.abs(acc[b, :, :n])
        if T == 0:
            continue
        seen = np.arange(n + T)[None] <= n + np.arange(T)[:, None]
        for h in range(H):
            g = h // R
            k, v = K[b, g, :n + T].astype(np.float64), V[b, g, :n + T].astype(np.float64)
            sc = np.where(seen, q[:, h] @ k.T / np.sqrt(hd), -np.inf)
            A = (np.abs(q[:, h]) @ np.abs(k).T / np.sqrt(hd)).max(1)
            p = np.exp(sc - sc.max(1, keepdims=True))
            p /= p.sum(1, keepdims=True)
            out[first:first + T, h * hd:(h + 1) * hd] = p @ v
            rel = 2 * 2.0 ** -21 * A + 2.0 ** -20
            tol[first:first + T, 0] = np.maximum(tol[first:first + T, 0], rel * np.abs(v).max() + 1e-12)
            if acc is not None:
                w = min(window, T)
                weights[b, g, :n + T] += p[T - w:].sum(0)
                wtol[b, g, :n + T] += (p[T - w:] * (rel[T - w:, None] + 2.0 ** -21)).sum(0) + 1e-12
    return out, tol, weights, wtol


def evict(w, n, budget, recent):
    """Rows that stay of one head, in order."""
    stay = min(n, budget)
    recent = min(recent, stay)
    old = n - recent
    key = np.where(np.isnan(w[:old]), -np.inf, w[:old].astype(np.float64))
    nan_last = np.isnan(w[:old])
    order = np.lexsort((np.arange(old), nan_last, -key))[:stay - recent]
    return np.concatenate((np.sort(order), np.arange(old, n))).astype(int)
