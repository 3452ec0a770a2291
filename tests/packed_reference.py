"""8-bit floating point with block scales and causal attention over packed sequences, restated in numpy at 64 bits."""

import numpy as np

BLOCK = 128


def _e4m3_values():
    b = np.arange(256)
    e, m = b >> 3 & 15, b & 7
    v = np.where(e == 0, m * 2.0 ** -9, (8.0 + m) * 2.0 ** (e - 10.0))
    v = np.where(b & 127 == 127, np.nan, v)
    return np.where(b >= 128, -v, v)


E4M3 = _e4m3_values()
_POSITIVE = E4M3[:127]  # 0 .. 448, ascending


def encode(x):
    """e4m3 codes of x (|x| <= 448), to nearest, ties to the even code; what is not finite is 0x7f."""
    x = np.asarray(x, np.float64)
    a = np.abs(np.where(np.isfinite(x), x, 0.0))
    hi = np.clip(np.searchsorted(_POSITIVE, a), 0, 126)
    lo = np.maximum(hi - 1, 0)
    up, down = _POSITIVE[hi] - a, a - _POSITIVE[lo]
    code = np.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    code = code | np.where(np.signbit(x), 128, 0)
    return np.where(np.isfinite(x), code, 0x7f).astype(np.uint8)


def exponent(amax):
    """The smallest e >= -100 with amax <= 448 * 2^e."""
    e = np.full(np.shape(amax), -100)
    for i, a in np.ndenumerate(np.asarray(amax, np.float64)):
        while a > np.ldexp(448.0, e[i]):
            e[i] += max(1, int(np.frexp(a)[1]) - 9 - e[i])
    return e


def blocks(k):
    return -(-k // BLOCK)


def normed(x, w, add_one, eps):
    """Rows normed in 64 bits and rounded to fp32."""
    x = np.asarray(x, np.float64)
    with np.errstate(invalid="ignore", over="ignore"):
        y = x / np.sqrt((x * x).mean(1, keepdims=True) + eps) * (1.0 + w.astype(np.float64) if add_one else w)
        return y.astype(np.float32).astype(np.float64)


def quant(x, rows_each):
    """Codes [rows, whole blocks] and exponents [rows / rows_each up, blocks] of x [rows, k]."""
    rows, k = x.shape
    wide = np.zeros((rows, blocks(k) * BLOCK))
    wide[:, :k] = x
    a = np.abs(np.where(np.isfinite(wide), wide, 0.0)).reshape(rows, -1, BLOCK).max(2)
    groups = -(-rows // rows_each)
    amax = np.stack([a[g * rows_each:(g + 1) * rows_each].max(0) for g in range(groups)])
    e = exponent(amax)
    of = np.repeat(np.repeat(e, rows_each, 0)[:rows], BLOCK, 1)
    return encode(wide / 2.0 ** of), e


def scale_bytes(e, lds, fill=255):
    """Exponents [rows, blocks] as [words][lds][4] bytes; blocks behind the last 127, rows behind the last `fill`."""
    rows, nb = e.shape
    words = -(-nb // 4)
    out = np.full((words, lds, 4), fill, np.uint8)
    padded = np.full((rows, words * 4), 127)
    padded[:, :nb] = e + 127
    out[:, :rows] = padded.reshape(rows, words, 4).transpose(1, 0, 2)
    return out


def values(codes, e, rows_each, k):
    rows = len(codes)
    of = np.repeat(np.repeat(e, rows_each, 0)[:rows], BLOCK, 1)
    return (E4M3[codes[:, :of.shape[1]]] * 2.0 ** of)[:, :k]


def swiglu(y):
    g = y.reshape(len(y), -1, 2, 16)
    gate, up = g[:, :, 0], g[:, :, 1]
    with np.errstate(over="ignore"):
        return (gate / (1.0 + np.exp(-gate)) * up).reshape(len(y), -1)


def attention(q, k, v, gate, scale, q0, k0, heads, kv_heads, half):
    """y [rows, heads * dim] and how far it may be off, of the rows that belong to a sequence (others NaN), q, k, v as
    [rows][heads][dim]. `half`: half a step of the result's type, and of the weights'."""
    rows, _, dim = q.shape
    group = heads // kv_heads
    u = 2.0 ** -24
    y, err = np.full((rows, heads, dim), np.nan), np.zeros((rows, heads, dim))
    for s in range(len(q0) - 1):
        a, b = min(q0[s], rows), min(q0[s + 1], rows)
        ka, kb = min(k0[s], len(k)), min(k0[s + 1], len(k))
        nq, nk = max(b - a, 0), max(kb - ka, 0)
        seen = np.maximum(0, nk - nq + np.arange(nq) + 1)
        hidden = np.arange(nk)[None] >= seen[:, None]
        for h in range(heads if nq else 0):
            kk, vv, qq = k[ka:kb, h // group], v[ka:kb, h // group], q[a:b, h]
            none = seen == 0
            with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
                sc = np.where(hidden, -np.inf, scale * (qq @ kk.T))
                top = np.where(none, 0.0, sc.max(1, initial=-np.inf))[:, None]
                p = np.where(hidden, 0.0, np.exp(sc - top))
                total = np.where(none, 1.0, p.sum(1))[:, None]
                # a hidden value counts for nothing, whatever it is
                bad = ~np.isfinite(vv)
                val = p @ np.where(bad, 0.0, vv)
                if bad.any():
                    val = np.where(~hidden @ bad, np.nan, val)
                size = p @ np.where(bad, 0.0, np.abs(vv)) / total
                # Scores: dim products and sums in fp32 (each addition off by at most 2 U of the terms' sum, whichever way it
                # rounds), the scale's two roundings and the difference from the reference point, up to 8 past it, rounded
                # once: 2 U |score| + 8 U. exp2's own error 2 U. The weight's rounding as an operand: half.
                ds = 2 * (dim + 4) * u * abs(scale) * (np.abs(qq) @ np.abs(kk).T) + 4 * u * np.abs(sc) + 16 * u
                # A score of -infinity weighs 0 exactly.
                pd = p * np.where(sc == -np.inf, 0.0, 2 * ds)
                y[a:b, h] = np.where(none[:, None], 0.0, val / total)
                # sums of `seen` weights and products, twice U each at most, in numerator and denominator; the division
                sums = ((4 * seen + 8) * u)[:, None]
                e = half * size + pd @ np.where(bad, 0.0, np.abs(vv)) / total + \
                    np.abs(y[a:b, h]) * (pd.sum(1)[:, None] / total) + sums * size
                err[a:b, h] = np.where(none[:, None], 0.0, e)
    if gate is not None:
        sees = np.zeros(rows, bool)
        for s in range(len(q0) - 1):
            a, b = min(q0[s], rows), min(q0[s + 1], rows)
            nk = max(min(k0[s + 1], len(k)) - min(k0[s], len(k)), 0)
            for i in range(max(b - a, 0)):
                sees[a + i] = nk - (b - a) + i + 1 > 0
        with np.errstate(over="ignore", invalid="ignore"):
            g = 1.0 / (1.0 + np.exp(-gate.reshape(rows, heads, dim).astype(np.float64)))
        g[~sees] = 1.0
        y, err = y * g, err * g + np.abs(y) * 16 * u  # exp's and the division's few roundings
    return y, err + half * np.abs(y) + half * err
