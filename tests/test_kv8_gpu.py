"""The rotary embedding and the 8-bit paged cache on the GPU against their definitions in 64 bits
(kv8_reference.py): every format, head layout and direction at the sizes, masks, strides and contents where they can
go wrong, and a run of them together."""

import numpy as np
import pytest

import kv8_reference as ref
from decide_amd.hip import DeviceArray, Stream, check, rt
from decide_amd.kernels import Kernels, Kv8Batch, Kv8Cache, Pages, RopeSpec, rope_freqs
from gpu_util import full, sync, to_dev, to_host

pytestmark = pytest.mark.gpu

U = 2.0 ** -24  # half a step of fp32, relative
HALF_STEP = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8, "f32": U}
NUMPY = {"f16": np.float16, "bf16": np.uint16, "f32": np.float32}
NONE = ref.NONE


def u32(a):
    return to_dev(np.ascontiguousarray(a, dtype=np.uint32))


def to_type(x, dtype):
    """x (float) as device values of dtype, and what they are in float64 (bf16 values: float32 cut to 16 bits)."""
    if dtype == "bf16":
        b = (np.asarray(x, np.float32).view(np.uint32) >> 16).astype(np.uint16)
        return b, (b.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    v = np.asarray(x, NUMPY[dtype])
    return v, v.astype(np.float64)


def from_type(v, dtype):
    return (v.astype(np.uint32) << 16).view(np.float32).astype(np.float64) if dtype == "bf16" else v.astype(np.float64)


# ---- rope -----------------------------------------------------------------------------------------------------------
def rope_bound(x, freq, amp, rot, layout, norm_w, add_one, out):
    """How far an element may be off. fp32 arithmetic, in units of U relative to the turned pair's size |a| + |b|: the norm
    factor 8 (a tree of 10 additions, halved by the root, the root and the division), the weight 2, its product 1; cos and
    sin 2 plus the angle's rounding to fp32 (half turns up to 1: pi U = 4) and amp 1; the products and the sum 3:
    21. Then one rounding to the result's type."""
    y0 = ref.rope(x, np.zeros(len(x)), np.zeros(rot // 2), 1.0, rot, layout, norm_w, add_one)
    size = np.abs(y0)
    if layout == "half":
        s = size[..., :rot // 2] + size[..., rot // 2:rot]
        size[..., :rot // 2], size[..., rot // 2:rot] = s, s
    else:
        s = size[..., 0:rot:2] + size[..., 1:rot:2]
        size[..., 0:rot:2], size[..., 1:rot:2] = s, s
    return 21 * U * size * max(1.0, abs(amp))


@pytest.mark.parametrize("rows,heads,dim,rot,layout,src,dst,norm,far", [
    (1, 16, 256, 64, "half", "f32", "f16", True, 8192),
    (41, 16, 256, 64, "half", "f32", "f16", True, 8192),
    (7, 5, 128, 128, "interleaved", "f16", "f16", False, 1000000),
    (3, 1, 4, 2, "half", "f32", "f32", True, 100),
    (3, 3, 4, 4, "interleaved", "bf16", "f32", True, 100),
    (5, 7, 80, 36, "half", "f16", "bf16", True, 131072),        # pairs that start inside a lane's four elements
    (5, 7, 80, 38, "interleaved", "bf16", "bf16", False, 131072),
    (2, 33, 192, 192, "half", "f32", "f32", True, 4000000000),  # positions past 2^31
    (9, 2, 64, 6, "half", "bf16", "f16", False, 70000),
    (300, 4, 256, 256, "interleaved", "f32", "bf16", True, 2307),
])
def test_rope_matches_its_definition(gpu, kernels, stream, rows, heads, dim, rot, layout, src, dst, norm, far):
    rng = np.random.default_rng(rows * 1000 + dim)
    ldx, ldy = heads * dim + 12, heads * dim + 8
    raw, x = to_type(rng.standard_normal((rows, ldx)), src)
    pos = rng.integers(0, far, rows).astype(np.uint32)
    pos[0] = far - 1
    freq, amp = rope_freqs(rot, 1e4, "plain")
    freq, amp = np.array(freq, np.float32), 1.25
    w = rng.standard_normal(dim).astype(np.float32) * 0.2 if norm else None
    add_one = rows % 2 == 1
    fr, wd = to_dev(freq), to_dev(w) if norm else None
    spec = RopeSpec((fr, 0), dim, rot, layout, amp, (wd, 0) if norm else None, add_one)
    y = full((rows, ldy), NUMPY[dst], 7)
    xd = to_dev(raw)
    kernels.rope.rope(stream, (xd, 0), ldx, src, (y, 0), ldy, dst, (u32(pos), 0), rows, heads, spec)
    sync()
    got = to_host(y)
    head = x[:, :heads * dim].reshape(rows, heads, dim)
    want = ref.rope(head, pos, freq, amp, rot, layout, w, add_one)
    bound = rope_bound(head, freq, amp, rot, layout, w, add_one, dst)
    err = np.abs(from_type(got[:, :heads * dim], dst).reshape(want.shape) - want)
    assert (err <= bound + HALF_STEP[dst] * (np.abs(want) + bound) + 2.0 ** -25).all(), (err / (bound + 1e-30)).max()
    assert (got[:, heads * dim:] == 7).all()  # behind the heads
    # in place, where types and strides agree
    if src == dst:
        kernels.rope.rope(stream, (xd, 0), ldx, src, (xd, 0), ldx, src, (u32(pos), 0), rows, heads, spec)
        sync()
        assert np.array_equal(to_host(xd)[:, :heads * dim], got[:, :heads * dim])
        assert np.array_equal(to_host(xd)[:, heads * dim:], raw[:, heads * dim:])


def test_rope_of_no_rows_is_a_no_op(gpu, kernels, stream):
    y = full((2, 64), np.float32, 3.0)
    f = to_dev(np.ones(32, np.float32))
    kernels.rope.rope(stream, (y, 0), 64, "f32", (y, 0), 64, "f32", (u32([0]), 0), 0, 1, RopeSpec((f, 0), 64, 64))
    kernels.rope.rope(stream, (y, 0), 64, "f32", (y, 0), 64, "f32", (u32([0]), 0), 1, 0, RopeSpec((f, 0), 64, 64))
    sync()
    assert (to_host(y) == 3.0).all()


def test_rope_agrees_with_q_norm_rope(gpu, kernels, stream):
    """decide's own layout, at positions where an fp32 angle is exact to 2^-13: the two differ by that times the pair,
    and one fp16 step."""
    rng = np.random.default_rng(5)
    rows = 37
    x = rng.standard_normal((rows, 10240)).astype(np.float32)
    w = rng.standard_normal(256).astype(np.float32) * 0.1
    freq = np.array(rope_freqs(64, 1e7)[0], np.float32)
    pos = rng.integers(0, 2048, rows).astype(np.uint32)
    xd, wd, fd, pd = to_dev(x), to_dev(w), to_dev(freq), u32(pos)
    a, b = full((rows, 4096), np.float16, 0), full((rows, 4096), np.float16, 0)
    kernels.rope.q_norm_rope(stream, (xd, 0), (wd, 0), (fd, 0), (pd, 0), (a, 0), rows, 10240)
    kernels.rope.rope(stream, (xd, 0), 10240, "f32", (b, 0), 4096, "f16", (pd, 0), rows, 16,
                      RopeSpec((fd, 0), 256, 64, "half", 1.0, (wd, 0)))
    sync()
    a, b = to_host(a).astype(np.float64), to_host(b).astype(np.float64)
    assert (np.abs(a - b) <= 2.0 ** -13 * 8 + 2 * 2.0 ** -11 * np.abs(a) + 2.0 ** -24).all()


# ---- append ---------------------------------------------------------------------------------------------------------
class Setup:
    """A cache of `layers` layers whose pages hold `fill` bytes, and a batch over it."""

    def __init__(self, kv, dim, fmt, lens, counts, pages=None, layers=2, layer=1, fill=0xFF, seed=0, before=0, behind=3,
                 wide=None):
        rng = np.random.default_rng(seed)
        need = [-(-n // ref.PAGE) for n in lens]
        self.pages = pages or sum(need) + 4
        ids = rng.permutation(self.pages)
        wide = wide or max(need) + 1
        self.table = np.full((len(lens), wide), 0xFFFFFFF0, np.uint32)
        at = 0
        for s, n in enumerate(need):
            self.table[s, :n] = ids[at:at + min(n, wide)]
            at += n
        self.row0 = np.cumsum([before] + list(counts)).astype(np.uint32)
        self.rows = int(self.row0[-1]) + behind
        self.qpos = np.full(self.rows, 5, np.uint32)
        for s, (n, c) in enumerate(zip(lens, counts)):
            self.qpos[self.row0[s]:self.row0[s + 1]] = np.arange(n - c, n)
        self.kv, self.dim, self.fmt, self.layers, self.layer = kv, dim, fmt, layers, layer
        self.host = [ref.Pool.empty(self.pages, kv, dim, fmt, fill) for _ in range(layers)]
        self.rng = rng

    def fill(self, length_of, big=1.0):
        """Gives every sequence its first length_of[s] tokens, through the reference."""
        p = self.host[self.layer]
        k = (self.rng.standard_normal((sum(length_of), self.kv, self.dim)) * big).astype(np.float32)
        v = self.rng.standard_normal(k.shape).astype(np.float32)
        v *= np.exp(self.rng.standard_normal((len(v), 1, 1))).astype(np.float32)
        row0 = np.cumsum([0] + list(length_of))
        qpos = np.concatenate([np.arange(n) for n in length_of] + [np.zeros(0)]).astype(np.int64)
        p.append(self.table, row0, qpos, k, v)

    def device(self):
        self.pool = to_dev(np.stack([p.bytes() for p in self.host]))
        self.cache = Kv8Cache((self.pool, 0), self.pages, self.layers, self.kv, self.dim, self.fmt)
        self.batch = Kv8Batch((u32(self.table), 0), self.table.shape[1], (u32(self.row0), 0), (u32(self.qpos), 0),
                              len(self.row0) - 1, self.rows)
        return self


def same_pool(setup, host):
    got, want = to_host(setup.pool), np.stack([p.bytes() for p in host])
    bad = np.argwhere(got != want)
    assert len(bad) == 0, (len(bad), bad[:5], [(got[tuple(i)], want[tuple(i)]) for i in bad[:5]])


APPENDS = [
    # tokens after the call, rows of the call
    ([1], [1]), ([16], [16]), ([17], [1]), ([64], [64]), ([65], [1]), ([200], [137]), ([64, 63, 130], [1, 3, 66]),
    ([5, 90, 31, 64], [0, 33, 0, 15]), ([100 + 7 * i for i in range(70)], [1 + i % 4 for i in range(70)]),
]


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("kv,dim,dtype", [(4, 256, "f32"), (2, 128, "f16"), (3, 64, "bf16"), (1, 256, "bf16")])
@pytest.mark.parametrize("lens,counts", APPENDS)
def test_append_codes_rows_as_defined(gpu, kernels, stream, kv, dim, dtype, fmt, lens, counts):
    t = Setup(kv, dim, fmt, lens, counts, seed=len(lens) * 100 + dim, before=2)
    t.fill([n - c for n, c in zip(lens, counts)])
    t.device()
    wide = kv * dim
    raw, x = to_type(t.rng.standard_normal((t.rows, 2 * wide + 8)) * 3.0, dtype)
    d = to_dev(raw)
    kernels.kv8.append(stream, t.cache, t.layer, t.batch, (d, 0), 2 * wide + 8, (d, wide * raw.itemsize), 2 * wide + 8,
                       dtype)
    sync()
    k = x[:, :wide].reshape(-1, kv, dim).astype(np.float32)
    v = x[:, wide:2 * wide].reshape(-1, kv, dim).astype(np.float32)
    t.host[t.layer].append(t.table, t.row0, t.qpos, k, v)
    same_pool(t, t.host)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("kv,dim,dtype,turned", [(17, 64, "f32", True), (33, 64, "bf16", False), (16, 128, "f16", True),
                                                 (15, 256, "f32", False)])
def test_append_of_many_sequences_and_heads(gpu, kernels, stream, kv, dim, dtype, turned, fmt):
    """More blocks of tokens and heads than run at once: a workgroup takes several heads, the last one fewer."""
    lens, counts = [5 + 3 * i for i in range(70)], [1 + i % 4 for i in range(70)]
    t = Setup(kv, dim, fmt, lens, counts, seed=kv, layers=1, layer=0)
    t.fill([n - c for n, c in zip(lens, counts)])
    t.device()
    wide = kv * dim
    raw, x = to_type(t.rng.standard_normal((t.rows, 2 * wide)) * 3.0, dtype)
    freq, d = np.array(rope_freqs(dim, 1e4)[0], np.float32), to_dev(raw)
    fd = to_dev(freq)
    kernels.kv8.append(stream, t.cache, 0, t.batch, (d, 0), 2 * wide, (d, wide * raw.itemsize), 2 * wide, dtype,
                       RopeSpec((fd, 0), dim, dim) if turned else None)
    sync()
    k, v = (x[:, i * wide:(i + 1) * wide].reshape(-1, kv, dim) for i in (0, 1))
    if turned:
        pos = np.zeros(t.rows)
        pos[:t.row0[-1]] = t.qpos[:t.row0[-1]]
        k = ref.rope(k, pos, freq, 1.0, dim, "half")
    t.host[0].append(t.table, t.row0, t.qpos, k.astype(np.float32), v.astype(np.float32))
    same_pool(t, t.host)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("dim,rot,layout,norm", [(256, 64, "half", True), (128, 128, "interleaved", True),
                                                 (64, 30, "half", False), (64, 64, "half", True)])
def test_append_turns_keys_in_64_bits(gpu, kernels, stream, fmt, dim, rot, layout, norm):
    """A key is rounded to fp32 once and then coded: the codes are those of the 64-bit definition (the two sides' 64-bit
    sums differ by 2^-50, which moves an fp32 rounding in one of 10^8 values)."""
    kv, lens, counts = 2, [70, 4097, 33], [70, 30, 1]
    t = Setup(kv, dim, fmt, lens, counts, seed=dim + rot)
    t.fill([n - c for n, c in zip(lens, counts)])
    t.device()
    wide = kv * dim
    x = t.rng.standard_normal((t.rows, 2 * wide)).astype(np.float32)
    w = t.rng.standard_normal(dim).astype(np.float32) * 0.2 if norm else None
    freq, amp = rope_freqs(rot, 1e6, "parts", factor=4.0, trained_len=1024)
    freq, d = np.array(freq, np.float32), to_dev(x)
    wd, fd = to_dev(w) if norm else None, to_dev(freq)
    spec = RopeSpec((fd, 0), dim, rot, layout, amp, (wd, 0) if norm else None)
    kernels.kv8.append(stream, t.cache, t.layer, t.batch, (d, 0), 2 * wide, (d, 4 * wide), 2 * wide, "f32", spec)
    sync()
    pos = np.zeros(t.rows)
    pos[:t.row0[-1]] = t.qpos[:t.row0[-1]]
    k = ref.rope(x[:, :wide].reshape(-1, kv, dim), pos, freq, amp, rot, layout, w).astype(np.float32)
    t.host[t.layer].append(t.table, t.row0, t.qpos, k, x[:, wide:].reshape(-1, kv, dim))
    same_pool(t, t.host)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_append_token_by_token_over_growing_and_shrinking_values(gpu, kernels, stream, fmt):
    """33 single tokens whose size runs over many powers of two: each grown scale codes the block's earlier tokens again,
    exactly as the definition does."""
    kv, dim = 2, 64
    t = Setup(kv, dim, fmt, [33], [1], behind=0)
    t.device()
    host = t.host[t.layer]
    for i in range(33):
        size = 2.0 ** ((i * 7) % 23 - 11) if i != 20 else 0.0
        x = (t.rng.standard_normal((1, 2, kv, dim)) * size).astype(np.float32)
        d, q = to_dev(x), u32([i])
        b = Kv8Batch((u32(t.table), 0), t.table.shape[1], (u32([0, 1]), 0), (q, 0), 1, 1)
        kernels.kv8.append(stream, t.cache, t.layer, b, (d, 0), kv * dim, (d, 4 * kv * dim), kv * dim, "f32")
        sync()
        host.append(t.table, np.array([0, 1]), np.array([i]), x[:, 0], x[:, 1])
        same_pool(t, t.host)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_append_of_extreme_values(gpu, kernels, stream, fmt):
    """Zeros, the smallest and largest fp32 numbers, values next to a power of two, infinities and NaN: a block with a
    value that is not finite gets a NaN scale, its neighbours are untouched."""
    kv, dim = 1, 64
    t = Setup(kv, dim, fmt, [112], [112], behind=0)
    t.device()
    x = t.rng.standard_normal((112, 2, dim)).astype(np.float32)
    x[:16] = 0.0
    x[16:32] *= np.float32(1e-42)                                 # subnormal
    x[32:48] = np.float32(3.4028235e38) * np.sign(x[32:48])
    x[48:64, 0, 0], x[48:64, 1, 3] = 448.0, np.nextafter(np.float32(448.0), np.float32(500.0))
    x[70, 0, 5], x[71, 1, 6] = np.inf, np.nan
    x[80, 1, 1] = -np.inf
    d = to_dev(x)
    kernels.kv8.append(stream, t.cache, t.layer, t.batch, (d, 0), 2 * dim, (d, 4 * dim), 2 * dim, "f32")
    sync()
    t.host[t.layer].append(t.table, t.row0, t.qpos, x[:, :1], x[:, 1:])
    got, want = to_host(t.pool)[t.layer], t.host[t.layer].bytes()
    g, w = (ref.Pool(b, kv, dim, fmt) for b in (got, want))
    assert np.array_equal(np.isnan(g.s[t.table[0, :2]]), np.isnan(w.s[t.table[0, :2]]))
    assert np.isnan(g.s[t.table[0, 1], 0, :, :3]).sum() == 3  # tokens 112 .. are not this call's
    assert np.array_equal(np.nan_to_num(g.s, nan=-1.0), np.nan_to_num(w.s, nan=-1.0))
    assert np.array_equal(g.k, w.k) and np.array_equal(g.v, w.v)


def test_append_leaves_out_what_has_no_page(gpu, kernels, stream):
    """A page id that the pool does not have, a token past the table, a sequence without a position: not stored, and
    everything else is."""
    kv, dim, fmt = 2, 64, "e4m3"
    t = Setup(kv, dim, fmt, [130, 200, 70, 90], [130, 200, 70, 20], wide=3, layers=1, layer=0)
    t.fill([0, 0, 0, 70])
    t.table[0, 1] = t.pages          # the page behind the last
    t.table[2, 0] = 0xFFFFFFFF
    t.qpos[t.row0[3]] = NONE         # sequence 3's rows have no place
    t.device()                       # sequence 1's tokens 192.. lie past the table's 3 entries
    x = t.rng.standard_normal((t.rows, 2, kv, dim)).astype(np.float32)
    d = to_dev(x)
    kernels.kv8.append(stream, t.cache, 0, t.batch, (d, 0), 2 * kv * dim, (d, 4 * kv * dim), 2 * kv * dim, "f32")
    sync()
    t.host[0].append(t.table, t.row0, t.qpos, x[:, 0], x[:, 1])
    same_pool(t, t.host)


# ---- attention ------------------------------------------------------------------------------------------------------
def attention_bound(q, k, v, scale, p, want):
    """How far y may be off, for one row and head, p its weights in 64 bits. Scores: fp32 sums of D exact products, off by
    at most (D + 2) U sum|q k| scale, twice (numerator and denominator); exp2, the reference point and the running sums: 2^-20;
    a weight's rounding to fp16: 2^-11 of it, and 2^-24 of the largest |v| where it is subnormal (weights are at most 2^8
    and their sum is at least 1); y's rounding to fp16."""
    size = p @ np.abs(v)
    err = 2 * (q.shape[-1] + 2) * U * float(np.max(np.abs(k) @ np.abs(q))) * abs(scale)
    return (2.0 ** -11 + err + 2.0 ** -20) * size + len(p) * 2.0 ** -24 * np.abs(v).max() + 2.0 ** -11 * np.abs(want) + 2.0 ** -25


def run_attention(kernels, stream, t, heads, gate=True, scale=None, max_tokens=None, pad=8, q_size=1.0, q=None):
    """(y as float64 [rows, heads, D], what lies behind the heads, q, gate)."""
    dim, wide = t.dim, heads * t.dim
    rng = np.random.default_rng(heads)
    qs = (rng.standard_normal((t.rows, wide + 2 * pad)) * q_size).astype(np.float16) if q is None else q
    gs = rng.standard_normal((t.rows, wide + 4)).astype(np.float32) if gate else None
    y = full((t.rows, wide + pad), np.float16, 7)
    qd, gd = to_dev(qs), to_dev(gs) if gate else None
    most = max_tokens or int((t.qpos.astype(np.uint32) + np.uint32(1)).max())
    kernels.kv8.attention(stream, t.cache, t.layer, t.batch, (qd, 2 * pad), wide + 2 * pad, heads,
                          scale if scale is not None else dim ** -0.5, (y, 0), wide + pad, most,
                          (gd, 0) if gate else None, wide + 4)
    sync()
    got = to_host(y)
    q = qs[:, pad:pad + wide].astype(np.float64).reshape(t.rows, heads, dim)
    g = gs[:, :wide].reshape(t.rows, heads, dim) if gate else None
    return got[:, :wide].reshape(t.rows, heads, dim), got[:, wide:], q, g


def check_attention(kernels, stream, t, heads, gate=True, scale=None, only=None, nan=None, **kw):
    """`only`: the heads that are held to the reference (all of them, unless there are many rows). `nan`: rows and heads that
    are NaN, left to the caller."""
    got, behind, q, g = run_attention(kernels, stream, t, heads, gate, scale, **kw)
    scale = t.dim ** -0.5 if scale is None else scale
    assert (behind == 7).all()
    pool, group = t.host[t.layer], heads // t.kv
    mine = np.zeros(t.rows, bool)
    for s in range(len(t.row0) - 1):
        r0, r1 = (min(int(x), t.rows) for x in t.row0[s:s + 2])
        mine[r0:r1] = True
        seen = (t.qpos[r0:r1].astype(np.uint32) + np.uint32(1)).astype(np.int64)
        n = int(seen.max()) if len(seen) else 0
        if n == 0:
            assert (got[r0:r1] == 0).all()
            continue
        k, v = pool.tokens(t.table[s, :-(-n // ref.PAGE)], n)
        for i, r in enumerate(range(r0, r1)):
            m = int(seen[i])
            if m == 0:
                assert (got[r] == 0).all()
                continue
            for h in only or range(heads):
                if nan is not None and nan[r, h]:
                    continue
                kh, vh = k[:m, h // group], v[:m, h // group]
                sc = kh @ q[r, h] * scale
                p = np.exp(sc - sc.max())
                p /= p.sum()
                want = p @ vh
                bound = attention_bound(q[r, h], kh, vh, scale, p, want)
                if gate:
                    sg = 1.0 / (1.0 + np.exp(-g[r, h].astype(np.float64)))
                    want, bound = want * sg, bound * sg + 2.0 ** -20 * np.abs(want) + 2.0 ** -25
                err = np.abs(got[r, h].astype(np.float64) - want)
                assert (err <= bound).all(), (s, r, h, m, float((err / bound).max()))
    assert (got[~mine] == 7).all()  # rows of no sequence
    return got


LAYOUTS = [(4, 4, 256), (16, 4, 256), (8, 1, 128), (6, 2, 128), (5, 1, 64), (40, 2, 64), (3, 3, 64)]


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("heads,kv,dim", LAYOUTS)
def test_attention_of_single_tokens(gpu, kernels, stream, heads, kv, dim, fmt):
    """One row a sequence, at every edge of a block and a page; bytes behind the last token are NaN codes and scales."""
    lens = [1, 2, 15, 16, 17, 31, 48, 63, 64, 65, 127, 128, 129, 193, 300]
    t = Setup(kv, dim, fmt, lens, [1] * len(lens), seed=dim + heads, before=1)
    t.fill(lens)
    check_attention(kernels, stream, t.device(), heads)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("heads,kv,dim", LAYOUTS)
def test_attention_of_ragged_prompts(gpu, kernels, stream, heads, kv, dim, fmt):
    """Prompts and chunks of many lengths in one call, sequences without rows among them, rows that see nothing, rows in no
    order of positions."""
    lens, counts = [70, 5, 333, 64, 9, 150, 1], [70, 0, 21, 64, 9, 1, 1]
    t = Setup(kv, dim, fmt, lens, counts, seed=dim + heads + 1)
    t.fill(lens)
    r0, r1 = int(t.row0[2]), int(t.row0[3])
    t.qpos[r0:r1] = t.rng.permutation(t.qpos[r0:r1])
    t.qpos[r0 + 3] = 0
    t.qpos[2:t.row0[-1]:13] = NONE
    t.qpos[t.row0[4]:t.row0[5]] = NONE  # a sequence none of whose rows sees anything
    check_attention(kernels, stream, t.device(), heads, gate=heads % 2 == 0)


@pytest.mark.parametrize("fmt,heads,kv,dim,length,rows", [
    ("e4m3", 4, 1, 64, 40000, 1), ("int8", 8, 1, 128, 9000, 3), ("e4m3", 4, 1, 256, 5000, 9), ("int8", 1, 1, 64, 70000, 1)])
def test_attention_over_long_sequences(gpu, kernels, stream, fmt, heads, kv, dim, length, rows):
    """Few rows over many tokens: the pages are divided between workgroups and the pieces merged; a second, short sequence
    has one piece, a third none."""
    lens, counts = [length, 100, 64], [rows, 2, 1]
    t = Setup(kv, dim, fmt, lens, counts, seed=length)
    t.fill(lens)
    t.qpos[t.row0[2]] = NONE
    got = check_attention(kernels, stream, t.device(), heads)
    # a bound that is too low or too high moves the cuts, not the answer
    for most in (1, 64 * t.table.shape[1]):
        again = run_attention(kernels, stream, t, heads, max_tokens=most)[0]
        assert np.allclose(again.astype(np.float64), got.astype(np.float64), rtol=2.0 ** -9, atol=2.0 ** -9)


@pytest.mark.parametrize("gate", [True, False])
@pytest.mark.parametrize("fmt,heads,kv,dim,rows", [
    ("e4m3", 16, 4, 256, 520), ("int8", 32, 2, 256, 180), ("int8", 40, 8, 128, 120), ("e4m3", 96, 3, 128, 0),
    ("e4m3", 72, 8, 64, 500), ("int8", 64, 4, 64, 560)])
def test_attention_of_many_rows(gpu, kernels, stream, fmt, heads, kv, dim, rows, gate):
    """Enough rows to fill the device with tiles of 128: ragged sequences of every kind, one of them `rows` rows, groups of
    which 128 is no multiple among the layouts; a sequence that ends inside a page next to NaN codes and scales; NaN blocks
    and a bad page that some rows see; rows that see nothing, in no order of positions."""
    lens, counts = [rows + 70, 5, 333, 64, 9, 150, 1, 200], [rows, 0, 121, 64, 9, 1, 1, 60]
    t = Setup(kv, dim, fmt, lens, counts, seed=dim + heads, layers=1, layer=0)
    t.fill(lens)
    r0, r1 = int(t.row0[2]), int(t.row0[3])
    t.qpos[r0:r1] = t.rng.permutation(t.qpos[r0:r1])
    t.qpos[r0 + 3] = 0
    t.qpos[2:t.row0[-1]:13] = NONE
    t.qpos[t.row0[4]:t.row0[5]] = NONE
    only = [0, heads // kv // 2, heads // kv, heads - 1]
    got = check_attention(kernels, stream, t.device(), heads, gate=gate, only=only)
    again = run_attention(kernels, stream, t, heads, gate=gate)[0]
    assert np.array_equal(again, got)
    # sequence 7: V's scale of tokens 32 .. 47 of kv head 0 is NaN; a page of sequence 2 that is none
    t.host[0].s[t.table[7, 0], 0, 1, 2] = np.nan
    page, t.table[2, 4] = t.table[2, 4], t.pages
    want = np.zeros((t.rows, heads), bool)
    seen = (t.qpos + np.uint32(1)).astype(np.int64)
    for s, start, of in ((7, 32, heads // kv), (2, 256, heads)):
        r = slice(int(t.row0[s]), int(t.row0[s + 1]))
        want[r, :of] = (seen[r] > start)[:, None]
    t.device()
    t.table[2, 4] = page
    bad = check_attention(kernels, stream, t, heads, gate=gate, only=only, nan=want)
    nan = np.isnan(bad.astype(np.float64))
    assert np.array_equal(nan.all(-1), want) and np.array_equal(nan.any(-1), want)
    if fmt == "e4m3":  # scales are powers of two: which one weights are taken relative to moves no bit
        assert np.array_equal(bad[~want], got[~want])


@pytest.mark.parametrize("fmt,heads,kv,dim,lens,counts", [
    ("e4m3", 12, 2, 128, [5000, 700, 64], [250, 30, 1]), ("int8", 8, 1, 128, [9000], [70]),
    ("int8", 8, 1, 256, [4200, 900], [110, 40]), ("e4m3", 16, 4, 256, [7001, 4099], [130, 150])])
def test_attention_of_chunks_behind_long_sequences(gpu, kernels, stream, fmt, heads, kv, dim, lens, counts):
    """Some hundred rows over thousands of tokens: tiles of 128 in runs, their states merged; a sequence whose rows see
    nothing, rows in no order. Another stream's workspace, sized for more rows and tokens beforehand, gives the same bits."""
    t = Setup(kv, dim, fmt, lens, counts, seed=dim + heads, layers=1, layer=0)
    t.fill(lens)
    r0, r1 = int(t.row0[0]), int(t.row0[1])
    t.qpos[r0:r1] = t.rng.permutation(t.qpos[r0:r1])
    t.qpos[r0 + 1] = 20
    t.qpos[2:t.row0[-1]:13] = NONE
    t.qpos[t.row0[2] if len(lens) > 2 else t.rows:] = NONE
    got = check_attention(kernels, stream, t.device(), heads, only=[0, heads // kv - 1, heads - 1])
    s = Stream()
    kernels.kv8.attention_ws(s.handle, t.cache, 2 * t.rows, len(lens), heads, 2 * max(lens))
    again = run_attention(kernels, s.handle, t, heads)[0]
    s.synchronize()
    assert np.array_equal(again, got)
    s.destroy()


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("scale", [0.0, -0.125, 2.0])
def test_attention_scales_and_sharp_weights(gpu, kernels, stream, fmt, scale):
    """scale 0 (the mean), a negative one, and scores of many hundreds, whose largest comes late: the reference point moves."""
    lens, counts = [260, 130], [40, 130]
    t = Setup(2, 64, fmt, lens, counts, seed=9)
    t.fill(lens, big=4.0)
    check_attention(kernels, stream, t.device(), 4, scale=scale, q_size=3.0, gate=False)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_attention_where_pages_differ_in_scale_by_many_powers(gpu, kernels, stream, fmt):
    """Values of 2^-40, 1 and 2^12 in different pages, and a page of zeros: weights are taken relative to the largest scale,
    so the small pages' share is held to the largest value's precision."""
    t = Setup(1, 128, fmt, [320], [5], layers=1, layer=0, seed=4)
    k = t.rng.standard_normal((320, 1, 128)).astype(np.float32)
    v = t.rng.standard_normal((320, 1, 128)).astype(np.float32)
    v[:64] *= np.float32(2.0 ** -40)
    v[64:128] = 0.0
    v[256:] *= np.float32(2.0 ** 12)
    t.host[0].append(t.table, np.array([0, 320]), np.arange(320), k, v)
    check_attention(kernels, stream, t.device(), 2, gate=False)
    t.qpos[:5] = [10, 63, 100, 127, 200]  # rows that see the small pages only
    check_attention(kernels, stream, t.device(), 2, gate=False)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("which", [0, 1])
def test_attention_passes_on_blocks_that_are_not_finite(gpu, kernels, stream, fmt, which):
    """A NaN scale (K's or V's) reaches the rows that see a token of its block, and no other row."""
    t = Setup(2, 128, fmt, [200], [200], layers=1, layer=0, seed=6)
    t.fill([200])
    t.host[0].s[t.table[0, 1], 1, which, 2] = np.nan  # tokens 96 .. 111 of kv head 1
    got = run_attention(kernels, stream, t.device(), 4, gate=False)[0].astype(np.float64)
    nan = np.isnan(got[:200])
    assert nan[96:, 2:].all() and not nan[:96].any() and not nan[:, :2].any()


@pytest.mark.parametrize("rows", [1, 120])
def test_attention_makes_rows_that_see_a_bad_page_nan(gpu, kernels, stream, rows):
    t = Setup(1, 64, "e4m3", [200, 200], [rows, rows], layers=1, layer=0, seed=8, wide=4, fill=0)
    t.fill([200, 200])
    t.table[0, 2] = t.pages  # tokens 128 .. 191 of sequence 0
    t.qpos[t.row0[1]:t.row0[2]] += 60  # sequence 1 sees up to token 259: past its table's 4 entries
    got = run_attention(kernels, stream, t.device(), 2, gate=False)[0]
    nan = np.isnan(got.astype(np.float64))
    seen = t.qpos[:2 * rows] + 1
    assert np.array_equal(nan[:rows].all((1, 2)), seen[:rows] > 128) and np.array_equal(nan[:rows].any((1, 2)), seen[:rows] > 128)
    assert np.array_equal(nan[rows:2 * rows].all((1, 2)), seen[rows:] > 256)


@pytest.mark.parametrize("rows", [3, 700])
def test_attention_over_one_table_of_any_stated_length(gpu, kernels, stream, rows):
    """One sequence's table may be said to be as long as 32 bits count: only entries at the seen pages are read (and the few
    behind them that are there)."""
    t = Setup(2, 128, "e4m3", [rows + 30], [rows], layers=1, layer=0, seed=rows, wide=40)
    t.fill([rows + 30])
    t.device()
    t.batch = Kv8Batch((u32(t.table), 0), 0xFFFFFFFF, (u32(t.row0), 0), (u32(t.qpos), 0), 1, t.rows)
    check_attention(kernels, stream, t, 32, only=[0, 17])


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("garbage", [np.nan, np.inf, 3e38])
@pytest.mark.parametrize("rows", [8, 120, 500])
def test_attention_keeps_a_bad_page_from_rows_that_do_not_see_it(gpu, kernels, stream, rows, garbage, fmt):
    """Whatever the unused pages hold: NaN codes, scales that are not finite or huge."""
    t = Setup(4, 128, fmt, [1000], [rows], layers=1, layer=0, seed=rows, pages=40)
    t.table[0, :16] = np.arange(1, 17)  # page 0 is not used
    t.fill([1000])
    t.host[0].s[0] = garbage
    got = run_attention(kernels, stream, t.device(), 32)[0]
    first = 14 if rows > 8 else 15  # the bad page: rows before and behind its start, or its inside
    if rows == 8:
        t.qpos[:8] = np.arange(956, 964)
        got = run_attention(kernels, stream, t.device(), 32)[0]
    t.table[0, first] = 0xFFFFFFFF
    bad = run_attention(kernels, stream, t.device(), 32)[0].astype(np.float64)
    sees = t.qpos[:rows] >= 64 * first
    assert sees.any() and not sees.all()
    assert np.isnan(bad[:rows][sees]).all() and np.isfinite(bad[:rows][~sees]).all()
    good = got[:rows][~sees].astype(np.float64)
    assert (np.abs(bad[:rows][~sees] - good) <= 2.0 ** -8 * (np.abs(good) + 1)).all()


def test_attention_reads_pages_past_4_gib(gpu, kernels, stream):
    """Offsets that do not fit 32 bits: the pages used are the first and the last of a pool of 4.4 GB."""
    kv, dim, fmt = 8, 256, "int8"
    size = ref.page_bytes(kv, dim)
    pages = (9 << 29) // size
    t = Setup(kv, dim, fmt, [100], [3], pages=5, layers=1, layer=0, behind=0)
    t.fill([100])
    pool = DeviceArray((pages * size,), np.uint8)
    host = t.host[0].bytes()
    far = t.table[0, :2].copy()
    ids = np.array([pages - 1, 0], np.uint32)
    for page, at in zip(far, ids):
        check(rt().hipMemcpy(pool.ptr + int(at) * size, host[page].ctypes.data, size, 1))
    t.device()
    t.cache = Kv8Cache((pool, 0), pages, 1, kv, dim, fmt)
    table = np.zeros((1, 3), np.uint32)
    table[0, :2] = ids
    t.batch = Kv8Batch((u32(table), 0), 3, (u32(t.row0), 0), (u32(t.qpos), 0), 1, t.rows)
    check_attention(kernels, stream, t, 8)
    # and the append writes there
    x = t.rng.standard_normal((3, 2, kv, dim)).astype(np.float32)
    d = to_dev(x)
    kernels.kv8.append(stream, t.cache, 0, t.batch, (d, 0), 2 * kv * dim, (d, 4 * kv * dim), 2 * kv * dim, "f32")
    sync()
    t.host[0].append(t.table, t.row0, t.qpos, x[:, 0], x[:, 1])
    back = np.empty(size, np.uint8)
    for page, at in zip(far, ids):
        check(rt().hipMemcpy(back.ctypes.data, pool.ptr + int(at) * size, size, 2))
        assert np.array_equal(back, t.host[0].bytes()[page])


# ---- pages ----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kv,dim,layers,n", [(4, 256, 3, 5), (1, 64, 1, 1), (3, 64, 2, 7), (8, 128, 2, 20)])
def test_copy_pages(gpu, kernels, stream, kv, dim, layers, n):
    pages = 2 * n + 3
    rng = np.random.default_rng(n)
    host = rng.integers(0, 256, (layers, pages, ref.page_bytes(kv, dim))).astype(np.uint8)
    pool, order = to_dev(host), rng.permutation(pages).astype(np.uint32)
    src, dst = order[:n].copy(), order[n:2 * n].copy()
    if n > 4:
        src[3] = src[1]                # one page to two places: a fork
        src[0], dst[2] = pages, 0xFFFFFFFF  # left out
    cache = Kv8Cache((pool, 0), pages, layers, kv, dim)
    kernels.kv8.copy_pages(stream, cache, (u32(src), 0), (u32(dst), 0), n)
    kernels.kv8.copy_pages(stream, cache, (u32(src), 0), (u32(dst), 0), 0)
    sync()
    for a, b in zip(src, dst):
        if a < pages and b < pages:
            host[:, b] = host[:, a]
    assert np.array_equal(to_host(pool), host)


# ---- streams, graphs, together --------------------------------------------------------------------------------------
def test_attention_on_two_streams_at_once(gpu, kernels, stream):
    """Each stream has its own workspace: long sequences whose pieces overlap in time give the bits of the same calls one
    after another."""
    ts, want = [], []
    for i, (fmt, length) in enumerate((("e4m3", 30000), ("int8", 24000))):
        t = Setup(1, 64, fmt, [length], [2], layers=1, layer=0, seed=20 + i)
        t.fill([length])
        t.device()
        t.q = to_dev(t.rng.standard_normal((t.rows, 256)).astype(np.float16))
        t.y = full((t.rows, 256), np.float16, 0)
        kernels.kv8.attention(stream, t.cache, 0, t.batch, (t.q, 0), 256, 4, 0.125, (t.y, 0), 256, length)
        sync()
        want.append(to_host(t.y))
        t.y = full((t.rows, 256), np.float16, 0)
        ts.append(t)
    streams = [Stream(), Stream()]
    for _ in range(10):
        for t, s in zip(ts, streams):
            kernels.kv8.attention(s.handle, t.cache, 0, t.batch, (t.q, 0), 256, 4, 0.125, (t.y, 0), 256,
                                  int(t.qpos[1]) + 1)
    for t, s, w in zip(ts, streams, want):
        s.synchronize()
        assert np.array_equal(to_host(t.y), w)
        s.destroy()


def test_a_step_replays_from_a_graph(gpu):
    """rope, append, attention of a batch captured once; between replays the positions, rows and tables change and eager work
    runs: every replay is the eager result, byte for byte. A capture that would have to grow the workspace is refused."""
    import ctypes

    kernels = Kernels()  # no workspace from another test
    kv, dim, heads, fmt = 1, 64, 4, "e4m3"
    lens = [5000, 40]
    t = Setup(kv, dim, fmt, [n + 8 for n in lens], [1, 1], layers=1, layer=0, seed=31, behind=0)
    t.fill(lens)
    t.device()
    s = Stream()
    freq = to_dev(np.array(rope_freqs(32, 1e4)[0], np.float32))
    spec = RopeSpec((freq, 0), dim, 32)
    wide = heads * dim
    x = DeviceArray((2, wide + 2 * dim), np.float32)
    q, y = full((2, wide), np.float16, 0), full((2, wide), np.float16, 0)
    qpos = u32([0, 0])
    b = Kv8Batch((u32(t.table), 0), t.table.shape[1], (u32([0, 1, 2]), 0), (qpos, 0), 2, 2)

    def step():
        ld = wide + 2 * dim
        kernels.rope.rope(s.handle, (x, 0), ld, "f32", (q, 0), wide, "f16", (qpos, 0), 2, heads, spec)
        kernels.kv8.append(s.handle, t.cache, 0, b, (x, 4 * wide), ld, (x, 4 * (wide + dim)), ld, "f32", spec)
        kernels.kv8.attention(s.handle, t.cache, 0, b, (q, 0), wide, heads, 0.125, (y, 0), wide, 5008)

    def capture(body):
        g, ge = ctypes.c_void_p(), ctypes.c_void_p()
        check(rt().hipStreamBeginCapture(s.handle, 0), "begin")
        try:
            body()
        finally:
            check(rt().hipStreamEndCapture(s.handle, ctypes.byref(g)), "end")
        check(rt().hipGraphInstantiate(ctypes.byref(ge), g, None, None, 0), "instantiate")
        return g, ge

    kernels.kv8.attention_ws(s.handle, t.cache, 2, 2, heads, 5008)
    wider = Kv8Cache((t.pool, 0), 1, 1, 1, 256)
    none = Kv8Batch((u32(np.zeros((1, 100))), 0), 100, (u32([0, 0]), 0), (u32([0]), 0), 1, 1)
    more = full((1, 256), np.float16, 0)
    with pytest.raises(AssertionError, match="being captured"):
        capture(lambda: kernels.kv8.attention(s.handle, wider, 0, none, (more, 0), 256, 1, 0.125, (more, 0), 256, 6400))
    start = to_host(t.pool)
    rows = [np.random.default_rng(i).standard_normal((2, wide + 2 * dim)).astype(np.float32) for i in range(4)]

    def setup(i):
        x.copy_from(rows[i])
        qpos.copy_from(np.array([lens[0] + i, lens[1] + i], np.uint32))

    eager = []
    for i in range(4):
        setup(i)
        step()
        s.synchronize()
        eager.append((to_host(y), to_host(t.pool)))
    t.pool.copy_from(start)
    g, ge = capture(step)
    for i in range(4):
        setup(i)
        check(rt().hipGraphLaunch(ge, s.handle), "launch")
        s.synchronize()
        assert np.array_equal(to_host(y), eager[i][0]) and np.array_equal(to_host(t.pool), eager[i][1])
        kernels.kv8.attention(0, t.cache, 0, b, (q, 0), wide, heads, 0.125, (y, 0), wide, 5008)  # eager, another stream
        sync()
    check(rt().hipGraphExecDestroy(ge), "destroy")
    check(rt().hipGraphDestroy(g), "destroy")
    s.destroy()


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_a_prefix_its_forks_and_their_follow_ups(gpu, kernels, stream, fmt):
    """The run they are made for, in decide's attention layout over two layers: a prompt is appended and attended to, three
    sequences fork from it (one inside a page), each appends its own follow-up behind a page of its own, all are attended
    to in one call, the prompt is dropped and the pool compacted. What is stored is held to the rows that went in, and
    what comes out to attention in 64 bits over what is stored."""
    heads, kv, dim, rot, layers, pages = 16, 4, 256, 64, 2, 24
    rng = np.random.default_rng(12)
    p = Pages(pages, 4)
    pool = full((layers, pages, ref.page_bytes(kv, dim)), np.uint8, 0xFF)
    cache = Kv8Cache((pool, 0), pages, layers, kv, dim, fmt)
    freq = np.array(rope_freqs(rot, 1e7)[0], np.float32)
    fd, qw, kw = to_dev(freq), rng.standard_normal(dim).astype(np.float32) * 0.1, rng.standard_normal(dim).astype(np.float32) * 0.1
    qwd, kwd = to_dev(qw), to_dev(kw)
    qs, ks = (RopeSpec((fd, 0), dim, rot, "half", 1.0, (w, 0)) for w in (qwd, kwd))
    truth = [[(np.zeros((0, kv, dim)),) * 2 for _ in range(4)] for _ in range(layers)]  # K, V of each layer and sequence

    def ids():
        t = np.full((4, 8), 0xFFFFFFF0, np.uint32)
        for s in range(4):
            page = p.table(s)[1]
            t[s, :len(page)] = page
        return t

    def copy(pairs):
        if pairs:
            a, b = zip(*pairs)
            kernels.kv8.copy_pages(stream, cache, (u32(a), 0), (u32(b), 0), len(pairs))

    def step(counts, appends):
        """Appends counts[s] tokens to every sequence and attends to them, in each layer."""
        have = [p.table(s)[0] for s in range(4)]
        copy([c for c in (p.resize(s, have[s] + n) for s, n in enumerate(counts) if n) if c])
        rows, row0 = sum(counts), np.cumsum([0] + list(counts))
        qpos = np.concatenate([np.arange(h, h + n) for h, n in zip(have, counts)]).astype(np.uint32)
        held = (u32(ids()), u32(row0), u32(qpos))
        b = Kv8Batch((held[0], 0), 8, (held[1], 0), (held[2], 0), 4, rows)
        for layer in range(layers):
            x = rng.standard_normal((rows, 10240)).astype(np.float32)  # q | gate | k | v
            xd, qd, yd = to_dev(x), full((rows, 4096), np.float16, 0), full((rows, 4096), np.float16, 0)
            kernels.rope.rope(stream, (xd, 0), 10240, "f32", (qd, 0), 4096, "f16", (held[2], 0), rows, heads, qs)
            kernels.kv8.append(stream, cache, layer, b, (xd, 4 * 8192), 10240, (xd, 4 * 9216), 10240, "f32", ks)
            kernels.kv8.attention(stream, cache, layer, b, (qd, 0), 4096, heads, 1 / 16, (yd, 0), 4096, 400,
                                  (xd, 4 * 4096), 10240)
            sync()
            k = ref.rope(x[:, 8192:9216].reshape(rows, kv, dim), qpos, freq, 1.0, rot, "half", kw)
            v = x[:, 9216:].reshape(rows, kv, dim).astype(np.float64)
            q = to_host(qd).astype(np.float64).reshape(rows, heads, dim)
            gate = 1 / (1 + np.exp(-x[:, 4096:8192].astype(np.float64))).reshape(rows, heads, dim)
            got = to_host(yd).astype(np.float64).reshape(rows, heads, dim)
            held_pool = ref.Pool(to_host(pool)[layer], kv, dim, fmt)
            for s in range(4):
                r = slice(row0[s], row0[s + 1])
                old = truth[layer][s]
                truth[layer][s] = tuple(np.concatenate([o, n[r]]) for o, n in zip(old, (k, v)))
                n, pages_of = p.table(s)
                if n == 0:
                    continue
                stored = held_pool.tokens(pages_of, n)
                for have_, want in zip(stored, truth[layer][s]):
                    # Each append may code a block anew, each time half a step off. int8: a step is the block's largest
                    # value / 127, and scales only grow. e4m3: half a step is 2^-4 of the value, once (another power of
                    # two as scale moves no larger code), and 2^-10 of the scale, which is below 2^-5 here, for those near 0.
                    off = (appends * np.abs(want).max() / 254.0 if fmt == "int8"
                           else 2.0 ** -4 * np.abs(want) + appends * 2.0 ** -15)
                    assert (np.abs(have_ - want) <= off * (1 + 2.0 ** -20)).all()
                for i in range(row0[s], row0[s + 1]):
                    m = int(qpos[i]) + 1
                    for h in range(heads):
                        kk, vv = stored[0][:m, h // 4], stored[1][:m, h // 4]
                        sc = kk @ q[i, h] / 16
                        w = np.exp(sc - sc.max())
                        w /= w.sum()
                        want = w @ vv
                        bound = attention_bound(q[i, h], kk, vv, 1 / 16, w, want)
                        bound = bound * gate[i, h] + 2.0 ** -20 * np.abs(want) + 2.0 ** -25
                        assert (np.abs(got[i, h] - want * gate[i, h]) <= bound).all()

    step([107, 0, 0, 0], 1)
    for s, n in ((1, 107), (2, 64), (3, 100)):
        p.fork(0, s, n)
        for layer in range(layers):
            truth[layer][s] = tuple(a[:n] for a in truth[layer][0])
    step([1, 41, 30, 3], 2)
    step([0, 1, 1, 1], 3)
    before = [[ref.Pool(to_host(pool)[layer], kv, dim, fmt).tokens(p.table(s)[1], p.table(s)[0]) for s in (1, 2, 3)]
              for layer in range(layers)]
    p.resize(0, 0)
    for layer in range(layers):
        truth[layer][0] = (np.zeros((0, kv, dim)),) * 2
    moves = p.compact()
    copy(moves)
    sync()
    after = [[ref.Pool(to_host(pool)[layer], kv, dim, fmt).tokens(p.table(s)[1], p.table(s)[0]) for s in (1, 2, 3)]
             for layer in range(layers)]
    for a, b in zip(before, after):
        for x, y in zip(a, b):
            assert np.array_equal(x[0], y[0]) and np.array_equal(x[1], y[1])
    step([5, 1, 70, 1], 4)


def test_nothing_is_launched_for_no_rows(gpu, kernels, stream):
    t = Setup(1, 64, "e4m3", [10], [1], layers=1, layer=0).device()
    y = full((4, 64), np.float16, 7)
    for rows, seqs in ((0, 1), (4, 0)):
        b = Kv8Batch((u32(t.table), 0), t.table.shape[1], (u32(t.row0), 0), (u32(t.qpos), 0), seqs, rows)
        d = to_dev(np.zeros((4, 128), np.float32))
        before = to_host(t.pool)
        kernels.kv8.append(stream, t.cache, 0, b, (d, 0), 128, (d, 256), 128, "f32")
        kernels.kv8.attention(stream, t.cache, 0, b, (y, 0), 64, 1, 1.0, (y, 0), 64, 10)
        sync()
        assert np.array_equal(to_host(t.pool), before) and (to_host(y) == 7).all()


def test_nothing_new_is_loaded_after_warm_up(gpu, kernels, stream):
    kernels.gemm.warm_up(stream, max_m=64)
    n = kernels.gemm.fast_pipelines()
    t = Setup(1, 64, "e4m3", [5000], [1], layers=1, layer=0)
    t.fill([5000])
    t.device()
    check_attention(kernels, stream, t, 4)
    assert kernels.gemm.fast_pipelines() == n


# ---- V scales that differ by many powers within a sequence ----------------------------------------------------------
def uneven(layout, rows, small, ahead, power, far, seed):
    """(a cache layer of one sequence, its queries): `small` tokens of values near 2^-12, then a block whose
    values are 2^power times larger and whose keys lie 2^-far below in weight for every query (`far` 0: like the others).
    Rows stand before, at and behind the block's start in turn; `ahead`: the large block comes first."""
    fmt, heads, kv, dim = layout
    n = small + 16
    t = Setup(kv, dim, fmt, [n], [rows], layers=1, layer=0, seed=seed)
    k = t.rng.standard_normal((n, kv, dim)).astype(np.float32) * 0.25
    v = t.rng.standard_normal((n, kv, dim)).astype(np.float32) * np.float32(2.0 ** -12)
    big = slice(0, 16) if ahead else slice(small, n)
    v[big] *= np.float32(2.0 ** power)
    q = (t.rng.standard_normal((t.rows, heads * dim + 16)) * 0.25).astype(np.float16)
    if far:
        q[:, 8::dim] = 8.0
        k[:, :, 0] = 0.0
        k[big, :, 0] = -far * np.log(2.0) / (8.0 * dim ** -0.5)
    t.host[0].append(t.table, np.array([0, n]), np.arange(n), k, v)
    t.qpos[:rows] = (np.arange(rows) * 5 % 32 + n - 32 if not ahead else 16 + np.arange(rows) * 7 % (n - 16)).astype(np.uint32)
    return t, q


def uneven_bound(t, n, kh, vh, qv, p, want, fmt, g):
    """attention_bound, with the subnormal weights' share relative to the largest product of a block's weight and its scale:
    weights are held as weight x scale / (at least the largest such product / 2^8), so each is off by half of fp16's smallest
    step, 2^-25, times that product and its code."""
    sc = np.repeat(t.host[0].s[t.table[0, :-(-n // ref.PAGE)], g, 1].astype(np.float64).ravel(), ref.BLOCK)[:n]
    code = 448.0 if fmt == "e4m3" else 127.0
    size = p @ np.abs(vh)
    err = 2 * (len(qv) + 2) * U * float(np.max(np.abs(kh) @ np.abs(qv))) * t.dim ** -0.5
    return ((2.0 ** -11 + err + 2.0 ** -20) * size + n * 2.0 ** -25 * code * (p * sc).max() + 2.0 ** -11 * np.abs(want)
            + 2.0 ** -25)


def check_uneven(t, got, q, n, heads, fmt):
    """Some 40 of the rows, the first and the last head, over the sequence's n tokens."""
    k, v = t.host[0].tokens(t.table[0, :-(-n // ref.PAGE)], n)
    rows, worst = int(t.row0[1]), 0.0
    for r in range(0, rows, max(1, rows // 40)):
        m = int(t.qpos[r]) + 1
        for h in (0, heads - 1):
            g = h // (heads // t.kv)
            sc = k[:m, g] @ q[r, h] * t.dim ** -0.5
            p = np.exp(sc - sc.max())
            p /= p.sum()
            want = p @ v[:m, g]
            bound = uneven_bound(t, m, k[:m, g], v[:m, g], q[r, h], p, want, fmt, g)
            worst = max(worst, float((np.abs(got[r, h].astype(np.float64) - want) / bound).max()))
    assert worst <= 1.0, worst


UNEVEN = [("narrow", 5, 8, 2, 128), ("narrow", 9, 4, 1, 256), ("narrow", 40, 6, 3, 64), ("wide", 330, 32, 4, 128),
          ("wide", 260, 40, 4, 256), ("wide", 650, 64, 4, 64)]


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("power", [16, 20, 26])
@pytest.mark.parametrize("small", [16, 592, 4112])
@pytest.mark.parametrize("which,rows,heads,kv,dim", UNEVEN)
def test_attention_of_rows_before_and_behind_a_large_block(gpu, kernels, stream, which, rows, heads, kv, dim, small, power,
                                                           fmt):
    """Rows of one tile, some of which see a block of values 2^power larger than all before it: the others are held
    to their own tokens' values, whatever their neighbours see."""
    t, q = uneven((fmt, heads, kv, dim), rows, small, False, power, 0, small + power)
    got, _, qv, _ = run_attention(kernels, stream, t.device(), heads, gate=False, q=q)
    check_uneven(t, got, qv, small + 16, heads, fmt)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("ahead", [False, True])
@pytest.mark.parametrize("small", [32, 592, 4112])
@pytest.mark.parametrize("which,rows,heads,kv,dim", UNEVEN)
def test_attention_over_a_large_block_that_weighs_next_to_nothing(gpu, kernels, stream, which, rows, heads, kv, dim, small,
                                                                  ahead, fmt):
    """A block of values 2^26 larger that is seen with weights 2^-34 of the others': its share is 2^-8, and it takes nothing
    from theirs."""
    t, q = uneven((fmt, heads, kv, dim), rows, small, ahead, 26, 34.0, small)
    got, _, qv, _ = run_attention(kernels, stream, t.device(), heads, gate=False, q=q)
    check_uneven(t, got, qv, small + 16, heads, fmt)


@pytest.mark.parametrize("heads,kv,dim,rows", [(32, 32, 128, 400), (24, 24, 256, 432)])
def test_a_capture_after_the_sizing_call_of_many_kv_heads(gpu, heads, kv, dim, rows):
    """Many kv heads turn to tiles of 128 with fewer pairs a head: the sizing call holds what they take, and each replay has the
    bits of an eager call on a stream of its own."""
    import ctypes

    kernels = Kernels()  # no workspace from another test
    t = Setup(kv, dim, "int8", [4200], [rows], layers=1, layer=0, seed=kv, behind=0)
    t.fill([4200])
    t.device()
    s, other = Stream(), Stream()
    q, wide = to_dev(t.rng.standard_normal((rows, heads * dim)).astype(np.float16)), heads * dim
    want, y = full((rows, wide), np.float16, 0), full((rows, wide), np.float16, 0)

    def call(stream, to):
        kernels.kv8.attention(stream, t.cache, 0, t.batch, (q, 0), wide, heads, dim ** -0.5, (to, 0), wide, 4200)

    call(other.handle, want)
    other.synchronize()
    kernels.kv8.attention_ws(s.handle, t.cache, rows, 1, heads, 4200)
    g, ge = ctypes.c_void_p(), ctypes.c_void_p()
    check(rt().hipStreamBeginCapture(s.handle, 0), "begin")
    try:
        call(s.handle, y)
    finally:
        check(rt().hipStreamEndCapture(s.handle, ctypes.byref(g)), "end")
    check(rt().hipGraphInstantiate(ctypes.byref(ge), g, None, None, 0), "instantiate")
    for _ in range(3):
        y.copy_from(np.zeros((rows, wide), np.float16))
        check(rt().hipGraphLaunch(ge, s.handle), "launch")
        s.synchronize()
        assert np.array_equal(to_host(y), to_host(want)) and np.isfinite(to_host(y).astype(np.float32)).all()
        call(other.handle, want)
        other.synchronize()
    check(rt().hipGraphExecDestroy(ge), "destroy")
    check(rt().hipGraphDestroy(g), "destroy")
    s.destroy()
    other.destroy()


def test_calls_without_work_count_no_kernel(gpu, stream):
    """What dh_variants_loaded counts are launches: a call of no rows, heads, sequences or pairs is none."""
    kernels = Kernels()
    n = kernels.gemm.fast_pipelines()
    t = Setup(1, 64, "e4m3", [10], [1], layers=1, layer=0).device()
    x, f, ids = to_dev(np.zeros((4, 128), np.float32)), to_dev(np.ones(32, np.float32)), u32([0])
    spec = RopeSpec((f, 0), 64, 64)
    kernels.rope.rope(stream, (x, 0), 64, "f32", (x, 0), 64, "f32", (ids, 0), 0, 1, spec)
    kernels.rope.rope(stream, (x, 0), 64, "f32", (x, 0), 64, "f32", (ids, 0), 1, 0, spec)
    for rows, seqs in ((0, 1), (4, 0)):
        b = Kv8Batch((u32(t.table), 0), t.table.shape[1], (u32(t.row0), 0), (u32(t.qpos), 0), seqs, rows)
        kernels.kv8.append(stream, t.cache, 0, b, (x, 0), 128, (x, 256), 128, "f32")
        kernels.kv8.attention(stream, t.cache, 0, b, (x, 0), 64, 1, 1.0, (x, 0), 64, 10)
    kernels.kv8.copy_pages(stream, t.cache, (ids, 0), (ids, 0), 0)
    sync()
    assert kernels.gemm.fast_pipelines() == n


def test_warm_up_covers_every_operator_of_the_cache(gpu, stream):
    kernels = Kernels()
    kernels.gemm.warm_up(stream, max_m=64)
    n = kernels.gemm.fast_pipelines()
    for kv, heads, rows, length in ((4, 16, 520, 540), (1, 4, 1, 5000)):  # tiles of 128; of 16, in runs
        t = Setup(kv, 256, "int8", [length], [rows], layers=1, layer=0, seed=rows, behind=0)
        t.fill([length])
        t.device()
        x = to_dev(t.rng.standard_normal((t.rows, 2 * kv * 256)).astype(np.float16))
        f = to_dev(np.array(rope_freqs(64, 1e4)[0], np.float32))
        spec = RopeSpec((f, 0), 256, 64, "interleaved")
        q, y = full((t.rows, heads * 256), np.float16, 0.5), full((t.rows, heads * 256), np.float16, 0)
        pos = u32(t.qpos)
        kernels.rope.rope(stream, (q, 0), heads * 256, "f16", (y, 0), heads * 256, "f16", (pos, 0), t.rows, heads, spec)
        kernels.kv8.append(stream, t.cache, 0, t.batch, (x, 0), 512 * kv, (x, 512 * kv), 512 * kv, "f16", spec)
        kernels.kv8.attention(stream, t.cache, 0, t.batch, (q, 0), heads * 256, heads, 0.0625, (y, 0), heads * 256, length)
        kernels.kv8.copy_pages(stream, t.cache, (u32([0]), 0), (u32([1]), 0), 1)
        sync()
    assert kernels.gemm.fast_pipelines() == n


# (rows, heads, kv heads, head dims, tokens): tiles of 16, of 16 in runs, of 128, of 128 in runs
KINDS = [(5, 8, 2, 128, 100), (9, 4, 1, 256, 70), (40, 6, 3, 64, 90), (5, 8, 2, 128, 4000), (7, 12, 4, 256, 3000),
         (3, 2, 1, 64, 6000), (330, 32, 4, 128, 400), (260, 40, 4, 256, 300), (650, 64, 4, 64, 700),
         (120, 12, 2, 128, 5000), (130, 16, 4, 256, 4200)]


def raw_attention(kernels, stream, t, heads, q, gate=None, scale=None):
    wide = heads * t.dim
    y, qd, gd = full((t.rows, wide), np.float16, 7), to_dev(q), to_dev(gate) if gate is not None else None
    most = int((t.qpos.astype(np.uint32) + np.uint32(1)).max())
    kernels.kv8.attention(stream, t.cache, t.layer, t.batch, (qd, 0), wide, heads, t.dim ** -0.5 if scale is None else scale,
                          (y, 0), wide, most, (gd, 0) if gate is not None else None, wide)
    sync()
    return to_host(y).reshape(t.rows, heads, t.dim)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("rows,heads,kv,dim,n", KINDS)
def test_attention_of_padding_rows_is_zero_whatever_they_hold(gpu, kernels, stream, rows, heads, kv, dim, n, fmt):
    """Rows without a position, as a padded batch has them: their queries and gates are NaN, infinite or the type's lowest,
    their outputs zero, and the other rows keep the bits that they have beside clean ones."""
    t = Setup(kv, dim, fmt, [n], [rows], layers=1, layer=0, seed=n, behind=0)
    t.fill([n])
    t.qpos[1:rows:3] = NONE
    t.device()
    q = t.rng.standard_normal((rows, heads * dim)).astype(np.float16)
    gate = t.rng.standard_normal((rows, heads * dim)).astype(np.float32)
    clean = raw_attention(kernels, stream, t, heads, q, gate)
    for i, (a, b) in enumerate([(np.nan, np.nan), (np.inf, np.inf), (-np.inf, -np.inf), (-65504.0, -3.4e38)]):
        q[1 + 3 * i:rows:12], gate[1 + 3 * i:rows:12] = a, b
    got = raw_attention(kernels, stream, t, heads, q, gate)
    none = t.qpos == NONE
    assert (got[none] == 0).all() and (clean[none] == 0).all()
    assert np.isfinite(clean.astype(np.float32)).all() and np.array_equal(got[~none], clean[~none])


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("rows,heads,kv,dim,n", KINDS)
def test_attention_of_queries_that_are_not_finite_is_nan(gpu, kernels, stream, rows, heads, kv, dim, n, fmt):
    """An infinite or NaN element of a query makes its scores infinite, of either sign, or NaN; the softmax of any of them is
    NaN, also where every score is -infinity. The other rows and heads keep their bits."""
    t = Setup(kv, dim, fmt, [n], [rows], layers=1, layer=0, seed=n + 1, behind=0)
    k = t.rng.standard_normal((n, kv, dim)).astype(np.float32)
    k[:, :, 5] = np.abs(k[:, :, 5]) + 0.5  # a query that is -inf there has no other score than -inf
    t.host[0].append(t.table, np.array([0, n]), np.arange(n), k, t.rng.standard_normal(k.shape).astype(np.float32))
    t.device()
    q = t.rng.standard_normal((rows, heads, dim)).astype(np.float16)
    clean = raw_attention(kernels, stream, t, heads, q.reshape(rows, -1))
    bad = np.zeros((rows, heads), bool)
    for i, v in enumerate((-np.inf, np.inf, np.nan)):
        q[i::5, i % heads, 5] = v
        bad[i::5, i % heads] = True
    got = raw_attention(kernels, stream, t, heads, q.reshape(rows, -1))
    assert np.isnan(got[bad].astype(np.float32)).all()
    assert np.isfinite(clean.astype(np.float32)).all() and np.array_equal(got[~bad], clean[~bad])


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("rows,heads,kv,dim,n", [k for k in KINDS if k[4] < 1000] + [(16, 16, 4, 256, 1000), (700, 32, 4, 128, 1400)])
def test_the_bits_of_a_row_that_is_not_cut_are_its_own(gpu, kernels, stream, rows, heads, kv, dim, n, fmt):
    """Where no sequence is divided, a row's bits depend on its own query, position and pages: every other row moves (to the
    start, behind a large block, out of sight), and the rest keep theirs."""
    t = Setup(kv, dim, fmt, [n], [rows], layers=1, layer=0, seed=n + 2, behind=0)
    k, v = (t.rng.standard_normal((n, kv, dim)).astype(np.float32) for _ in range(2))
    v[n // 2:n // 2 + 9] *= np.float32(300.0)
    t.host[0].append(t.table, np.array([0, n]), np.arange(n), k, v)
    t.qpos[:] = t.rng.integers(0, n, rows)
    t.qpos[0::2] = np.sort(t.qpos[0::2])
    q = t.rng.standard_normal((rows, heads * dim)).astype(np.float16)
    first, stay = None, np.arange(rows) % 2 == 0
    for move in (None, 0, n - 1, NONE, 17):
        if move is not None:
            t.qpos[~stay] = move
        t.device()
        qq = q.copy()
        if move == 17:
            qq[~stay] = np.inf
        got = raw_attention(kernels, stream, t, heads, qq)
        first = got if first is None else first
        assert np.array_equal(got[stay], first[stay]), (move, np.argwhere((got != first).any((1, 2)) & stay).ravel()[:9])


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("rows,heads,kv,dim,n", KINDS)
def test_attention_over_a_zeroed_pool_is_zero(gpu, kernels, stream, rows, heads, kv, dim, n, fmt):
    """Scales of zero, as a pool has them that nothing was written to (a program's dry run): every value is zero, and so is
    every output; written tokens behind such blocks come out as if those held zeros."""
    t = Setup(kv, dim, fmt, [n], [rows], layers=1, layer=0, seed=n + 3, behind=0, fill=0)
    q = t.rng.standard_normal((rows, heads * dim)).astype(np.float16)
    gate = t.rng.standard_normal((rows, heads * dim)).astype(np.float32)
    got = raw_attention(kernels, stream, t.device(), heads, q, gate)
    assert (got == 0).all()
    t.fill([n])
    want = t.host[0].s.copy()
    pages = t.table[0, :2]
    t.host[0].s[pages] = 0.0
    zeros = raw_attention(kernels, stream, t.device(), heads, q, gate)
    t.host[0].s[pages] = want[pages]
    t.host[0].k, t.host[0].v = t.host[0].k.copy(), t.host[0].v.copy()
    t.host[0].k[pages] = t.host[0].v[pages] = 0 if fmt == "e4m3" else 128
    same = raw_attention(kernels, stream, t.device(), heads, q, gate)
    a, b = zeros.astype(np.float64), same.astype(np.float64)
    # weights are rounded to fp16 relative to different references: 2^-11 each of what is summed, at most the largest |v|
    _, v = t.host[0].tokens(t.table[0, :-(-n // ref.PAGE)], n)
    assert (np.abs(a - b) <= 2.0 ** -9 * np.abs(v).max()).all() and np.isfinite(a).all()
