"""The 8-bit paged cache and the rotary embedding from their definitions, in 64 bits on the host: what the HIP kernels
are compared with. Nothing here reads the library."""

import numpy as np

PAGE, BLOCK = 64, 16
NONE = 0xFFFFFFFF
FLOOR = 2.0 ** -100


def e4m3_values():
    """The 256 numbers of OCP e4m3 (1 sign, 4 exponent bits of bias 7, 3 mantissa bits; 0x7f and 0xff are NaN)."""
    out = np.empty(256)
    for b in range(256):
        e, m = b >> 3 & 15, b & 7
        v = m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10)
        if b & 127 == 127:
            v = np.nan
        out[b] = -v if b >= 128 else v
    return out


E4M3 = e4m3_values()


def values(codes, fmt):
    """Code bytes as numbers, without their scale."""
    return E4M3[codes] if fmt == "e4m3" else codes.astype(np.float64) - 128.0


def scale_of(amax, fmt):
    if fmt == "int8":
        return max(float(np.float32(amax) * (np.float32(1.0) / np.float32(127.0))), FLOOR)
    if not amax > 0:
        return FLOOR
    e = int(np.floor(np.log2(amax / 448.0))) - 1
    while amax > 448.0 * 2.0 ** e:
        e += 1
    return max(2.0 ** e, FLOOR)


def encode(x, fmt):
    """Numbers already divided by their scale as code bytes, to the nearest, ties to even."""
    x = np.asarray(x, np.float64)
    if fmt == "int8":
        return (np.rint(x) + 128).astype(np.uint8)
    a = np.abs(x)
    e = np.maximum(np.floor(np.log2(np.maximum(a, 2.0 ** -300))), -6)
    e = np.where(a >= 2.0 ** (e + 1), e + 1, e)
    step = 2.0 ** (e - 3)
    q = np.rint(a / step) * step
    mag = np.searchsorted(E4M3[:127], q)
    assert (E4M3[mag] == q).all()
    return (mag + 128 * np.signbit(x)).astype(np.uint8)


def page_bytes(kv, dim):
    return -(-kv * (2 * PAGE * dim + 32) // 128) * 128


def rope(x, pos, freq, amp, rot, layout, norm_w=None, add_one=True, eps=1e-6):
    """x [rows, heads, D] normed and turned, in 64 bits."""
    x = np.asarray(x, np.float64)
    if norm_w is not None:
        w = norm_w.astype(np.float64) + (1.0 if add_one else 0.0)
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + np.float64(np.float32(eps))) * w
    angle = np.asarray(pos, np.float64)[:, None] * np.asarray(freq, np.float32).astype(np.float64)
    c, s = (f(angle)[:, None] * np.float64(np.float32(amp)) for f in (np.cos, np.sin))
    y = x.copy()
    if layout == "half":
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        y[..., :rot // 2], y[..., rot // 2:rot] = a * c - b * s, b * c + a * s
    else:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        y[..., 0:rot:2], y[..., 1:rot:2] = a * c - b * s, b * c + a * s
    return y


class Pool:
    """One layer's pages: bytes as the library lays them out, with views of the parts."""

    def __init__(self, data, kv, dim, fmt):
        self.kv, self.dim, self.fmt = kv, dim, fmt
        self.data = data  # uint8 [pages, page_bytes]
        n, kb = len(data), kv * PAGE * dim
        self.k = data[:, :kb].reshape(n, kv, PAGE, dim) if n else None
        self.v = data[:, kb:2 * kb].reshape(n, kv, dim, PAGE)
        self.s = data[:, 2 * kb:2 * kb + 32 * kv].copy().view(np.float32).reshape(n, kv, 2, 4)

    @classmethod
    def empty(cls, pages, kv, dim, fmt, fill=0):
        return cls(np.full((pages, page_bytes(kv, dim)), fill, np.uint8), kv, dim, fmt)

    def bytes(self):
        """The records again, from the (possibly changed) parts."""
        out, kb = self.data.copy(), self.kv * PAGE * self.dim
        n = len(out)
        out[:, :kb] = self.k.reshape(n, -1)
        out[:, kb:2 * kb] = self.v.reshape(n, -1)
        out[:, 2 * kb:2 * kb + 32 * self.kv] = np.ascontiguousarray(self.s).view(np.uint8).reshape(n, -1)
        return out

    def tokens(self, pages, n):
        """(K, V) [n, kv, D] of the sequence that holds `pages`."""
        sc = np.repeat(self.s[pages].astype(np.float64), BLOCK, axis=3)
        with np.errstate(invalid="ignore"):
            k = values(self.k[pages], self.fmt) * sc[:, :, 0, :, None]
            v = values(self.v[pages], self.fmt) * sc[:, :, 1, None, :]
        return (k.transpose(0, 2, 1, 3).reshape(-1, self.kv, self.dim)[:n],
                v.transpose(0, 3, 1, 2).reshape(-1, self.kv, self.dim)[:n])

    def append(self, table, row0, qpos, k, v):
        """k, v: float32 rows [rows, kv, D] as they are to be coded."""
        self.k, self.v = self.k.copy(), self.v.copy()
        rows = len(k)
        for s in range(len(row0) - 1):
            r0, r1 = min(row0[s], rows), min(row0[s + 1], rows)
            if r1 <= r0 or qpos[r0] == NONE:
                continue
            p, end = int(qpos[r0]), int(qpos[r0]) + (r1 - r0)
            r = r0
            while p < end:
                o = p % BLOCK
                m = min(BLOCK - o, end - p)
                page = p // PAGE
                if page < table.shape[1] and table[s, page] < len(self.data):
                    self._block(int(table[s, page]), p % PAGE // BLOCK, o, k[r:r + m], v[r:r + m])
                p, r = p + m, r + m

    def _block(self, page, b, kept, k, v):
        span = slice(b * BLOCK, (b + 1) * BLOCK)
        for h in range(self.kv):
            for which, x, codes in ((0, k[:, h], self.k[page, h, span]), (1, v[:, h], self.v[page, h, :, span].T)):
                old = float(self.s[page, h, which, b])
                x = x.astype(np.float32)
                end = kept + len(x)
                finite = np.isfinite(x).all()
                new = codes.copy()
                if not finite or (kept and np.isnan(old)):
                    sc = np.nan
                    new[kept:end] = 0 if self.fmt == "e4m3" else 128
                else:
                    sc = scale_of(float(np.abs(x).max()), self.fmt)
                    if kept:
                        sc = max(sc, old)
                        if sc != old:
                            ratio = np.float32(old) / np.float32(sc)
                            new[:kept] = encode((values(codes[:kept], self.fmt).astype(np.float32) * ratio), self.fmt)
                    new[kept:end] = encode(x / np.float32(sc), self.fmt)
                new[end:] = 0 if self.fmt == "e4m3" else 128
                codes[:] = new
                self.s[page, h, which, b] = sc

    def attention(self, table, row0, qpos, q, scale, gate=None):
        """q [rows, heads, D] float64 → y [rows, heads, D]; rows of no sequence are left NaN with `mine` False."""
        rows, heads, dim = q.shape
        y, mine = np.zeros(q.shape), np.zeros(rows, bool)
        group = heads // self.kv
        for s in range(len(row0) - 1):
            r0, r1 = min(row0[s], rows), min(row0[s + 1], rows)
            if r1 <= r0:
                continue
            mine[r0:r1] = True
            seen = np.where(qpos[r0:r1] == NONE, 0, qpos[r0:r1].astype(np.int64) + 1)
            n = int(seen.max())
            if n == 0:
                continue
            need = -(-n // PAGE)
            ids = [int(table[s, p]) if p < table.shape[1] else len(self.data) for p in range(need)]
            bad = np.array([i >= len(self.data) for i in ids])
            k, v = self.tokens([0 if b else i for i, b in zip(ids, bad)], n)
            k[np.repeat(bad, PAGE)[:n]] = np.nan
            for i, r in enumerate(range(r0, r1)):
                t = int(seen[i])
                if t == 0:
                    continue
                for h in range(heads):
                    kh, vh = k[:t, h // group], v[:t, h // group]
                    sc = kh @ q[r, h] * scale
                    w = np.exp(sc - sc.max())
                    y[r, h] = (w @ vh) / w.sum()
        if gate is not None:
            y = y / (1.0 + np.exp(-gate.astype(np.float64)))
        return y, mine
