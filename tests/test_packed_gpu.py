"""Causal attention over packed sequences on the GPU against its definition in 64 bits (packed_reference.py), and a run of
the 8-bit products around it, as a layer uses them."""

import ctypes

import numpy as np
import pytest

import packed_reference as ref
from decide_amd.hip import DeviceArray, Stream, check, rt
from decide_amd.kernels import Epilogue, Fp8Matrix, Kernels, PackedBatch, RopeSpec, rope_freqs
from gpu_util import full, sync, to_dev, to_host
from test_fp8_gpu import to_type, up

pytestmark = pytest.mark.gpu

HALF = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def from_type(v, dtype):
    return (v.astype(np.uint32) << 16).view(np.float32).astype(np.float64) if dtype == "bf16" else v.astype(np.float64)


def u32(a):
    return to_dev(np.ascontiguousarray(a, dtype=np.uint32))


class Packed:
    """Sequences of nq rows and nk keys each, with `pad` rows before the first and behind the last that belong to none and
    hold NaN, in matrices whose strides go on with NaN."""

    def __init__(self, nq, nk, heads, kv, dim, dtype, gate=True, pad=2, seed=0, scale=None, size=1.0):
        rng = self.rng = np.random.default_rng(seed + sum(nq) * 31 + sum(nk) + dim)
        self.heads, self.kv, self.dim, self.dtype, self.pad = heads, kv, dim, dtype, pad
        self.scale = dim ** -0.5 if scale is None else scale
        self.q0 = pad + np.concatenate([[0], np.cumsum(nq)])
        self.k0 = pad + np.concatenate([[0], np.cumsum(nk)])
        self.rows, self.keys = int(self.q0[-1]) + pad, int(self.k0[-1]) + pad

        def matrix(rows, n, first, last, std):
            raw, x = to_type(rng.standard_normal((rows, n, dim)) * std, dtype)
            nan = to_type(np.full(1, np.nan), dtype)[0][0]
            raw[:first] = raw[last:] = nan
            x[:first] = x[last:] = np.nan
            return raw, x

        self.qr, self.q = matrix(self.rows, heads, pad, self.rows - pad, size)
        self.kr, self.k = matrix(self.keys, kv, pad, self.keys - pad, size)
        self.vr, self.v = matrix(self.keys, kv, pad, self.keys - pad, 1.0)
        self.g = (rng.standard_normal((self.rows, heads * dim)) * 2).astype(np.float32) if gate else None

    def device(self, extra=8):
        self.lds = [self.heads * self.dim + extra, self.kv * self.dim + 2 * extra, self.kv * self.dim + extra]
        self.d = []
        for raw, ld in zip((self.qr, self.kr, self.vr), self.lds):
            wide = np.full((len(raw), ld), to_type(np.full(1, np.nan), self.dtype)[0][0])
            wide[:, :raw.shape[1] * self.dim] = raw.reshape(len(raw), -1)
            self.d.append(to_dev(wide))
        self.ldg = self.heads * self.dim + 4
        self.gd = None
        if self.g is not None:
            wide = np.full((self.rows, self.ldg), np.nan, np.float32)
            wide[:, :-4] = self.g
            self.gd = to_dev(wide)
        self.ldy = self.heads * self.dim + 4
        self.q0d, self.k0d = u32(self.q0), u32(self.k0)
        self.batch = PackedBatch((self.q0d, 0), (self.k0d, 0), len(self.q0) - 1, self.rows, self.keys,
                                 int(np.diff(self.k0).max(initial=0)))

    def call(self, kernels, stream, y):
        q, k, v = self.d
        kernels.attn.packed(stream, self.batch, (q, 0), self.lds[0], (k, 0), self.lds[1], (v, 0), self.lds[2], self.dtype,
                            self.heads, self.kv, self.dim, self.scale, (y, 0), self.ldy,
                            None if self.gd is None else (self.gd, 0), self.ldg if self.gd is not None else 0)

    def blank(self):
        return full((self.rows, self.ldy), np.uint16, 0x1234)

    def run(self, kernels, stream):
        self.device()
        y = self.blank()
        self.call(kernels, stream, y)
        sync()
        return self.taken(to_host(y))

    def taken(self, raw):
        """The outputs, after checking that nothing else was written."""
        a, b = int(self.q0[0]), int(self.q0[-1])
        assert (raw[:a] == 0x1234).all() and (raw[b:] == 0x1234).all() and (raw[:, self.heads * self.dim:] == 0x1234).all()
        out = raw[:, :self.heads * self.dim]
        return from_type(out if self.dtype == "bf16" else out.view(np.float16), self.dtype)

    def want(self):
        y, err = ref.attention(self.q, self.k, self.v, self.g, self.scale, self.q0, self.k0, self.heads, self.kv,
                               HALF[self.dtype])
        return y.reshape(self.rows, -1), err.reshape(self.rows, -1)

    def check(self, kernels, stream):
        got, (want, err) = self.run(kernels, stream), self.want()
        a, b = int(self.q0[0]), int(self.q0[-1])
        got, want, err = got[a:b], want[a:b], err[a:b]
        assert np.array_equal(np.isnan(got), np.isnan(want))
        fine = np.isfinite(want)
        off = np.abs(got[fine] - want[fine]) / (err[fine] + 2.0 ** -24)
        assert (off <= 1.0).all(), off.max()
        return got


LAYOUTS = [(16, 4, 256, "f16"), (8, 2, 128, "bf16"), (6, 2, 64, "f16"), (5, 1, 64, "bf16"), (3, 3, 128, "f16"),
           (4, 4, 256, "bf16")]


@pytest.mark.parametrize("heads,kv,dim,dtype", LAYOUTS)
@pytest.mark.parametrize("nq,nk", [
    ([1], [1]), ([1], [64]), ([1, 1, 1], [65, 1, 200]), ([5], [5]), ([64], [64]), ([65, 3, 130], [65, 3, 130]),
    ([7, 20], [300, 20]), ([0, 4, 0, 0, 9], [3, 4, 0, 7, 40]), ([10, 3], [4, 0]), ([70], [69]), ([2, 2], [0, 2]),
])
def test_sequences_of_all_kinds(gpu, kernels, stream, heads, kv, dim, dtype, nq, nk):
    Packed(nq, nk, heads, kv, dim, dtype, gate=len(nq) % 2 == 0).check(kernels, stream)


@pytest.mark.parametrize("heads,kv,dim,dtype,nq,nk", [
    (16, 4, 256, "f16", [300], [300]), (8, 2, 128, "bf16", [200, 333], [200, 333]), (8, 1, 64, "f16", [400, 100], [400, 600]),
    (4, 1, 128, "f16", [1], [3000]), (4, 2, 64, "bf16", [1, 1, 1, 1], [2000, 5, 1300, 129]), (16, 4, 256, "bf16", [2], [1500]),
    (8, 8, 64, "f16", [130], [1000]), (32, 8, 128, "bf16", [1] * 9, [700, 1, 64, 65, 128, 129, 33, 512, 300]),
    (4, 1, 64, "f16", [40], [2500]), (1, 1, 128, "f16", [600], [600]), (8, 2, 256, "f16", [33, 1, 7], [900, 1100, 450]),
])
def test_longer_sequences(gpu, kernels, stream, heads, kv, dim, dtype, nq, nk):
    Packed(nq, nk, heads, kv, dim, dtype).check(kernels, stream)


WIDE = [  # enough (row, head) pairs for the tiles of many rows
    (32, 2, 128, "bf16", [610], [610]), (48, 6, 256, "f16", [300, 1, 170], [300, 500, 200]), (64, 64, 64, "f16", [400], [400]),
    (48, 2, 64, "bf16", [129, 0, 380], [700, 5, 380]), (24, 3, 128, "f16", [500, 65, 300], [500, 64, 1100]),
    (40, 8, 256, "bf16", [33, 600], [40, 600]),
]


@pytest.mark.parametrize("heads,kv,dim,dtype,nq,nk", WIDE)
def test_many_rows(gpu, kernels, stream, heads, kv, dim, dtype, nq, nk):
    assert sum(nq) * heads // 32 >= (9 if dim == 128 else 11) * 256 // 4  # the planner takes wide tiles from here on
    Packed(nq, nk, heads, kv, dim, dtype, gate=len(nq) > 1).check(kernels, stream)


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_many_rows_of_odd_scales_and_contents(gpu, kernels, stream, dim):
    """A negative scale and none; keys of -infinity and NaN; rows that see nothing; what is not finite in another sequence."""
    for scale in (-0.4, 0.0):
        Packed([90] * 3, [90] * 3, 96, 4, dim, "f16", scale=scale).check(kernels, stream)
    p = Packed([400], [400], 64, 2, dim, "f16", gate=False)
    p.qr[:], p.q[:] = np.abs(p.qr), np.abs(p.q)
    for at, value in ((p.k0[0] + 5, -np.inf), (p.k0[0] + 398, np.nan), (p.k0[0], -np.inf)):
        p.kr[at], p.k[at] = value, value
    got = p.check(kernels, stream)
    assert np.isnan(got[[0, -1, -2]]).all() and np.isfinite(got[1:-2]).all()
    clean, bad = (Packed([200, 100, 100], [200, 20, 100], 64, 4, dim, "bf16") for _ in range(2))
    bad.kr[bad.k0[1]:bad.k0[2]:7] = bad.vr[bad.k0[1]:bad.k0[2]:5] = 0x7f80
    bad.qr[bad.q0[1]:bad.q0[1] + 9] = 0x7fc0
    bad.g[bad.q0[1]:bad.q0[1] + 9] = np.nan
    a, b = clean.run(kernels, stream), bad.run(kernels, stream)
    for s in (0, 2):
        rows = slice(int(clean.q0[s]), int(clean.q0[s + 1]))
        assert np.array_equal(a[rows], b[rows]) and np.isfinite(a[rows]).all()
    assert (b[bad.q0[1]:bad.q0[1] + 80] == 0).all() and (a[bad.q0[1]:bad.q0[1] + 80] == 0).all()


@pytest.mark.parametrize("heads", [100, 257])
def test_groups_wider_than_a_tile(gpu, kernels, stream, heads):
    Packed([1, 3], [70, 3], heads, 1, 64, "f16").check(kernels, stream)


@pytest.mark.parametrize("n", [70, 500])
def test_many_short_sequences(gpu, kernels, stream, n):
    rng = np.random.default_rng(n)
    nk = rng.integers(1, 40, n).tolist()
    Packed([min(int(rng.integers(0, 9)), v) for v in nk], nk, 4, 2, 64, "f16").check(kernels, stream)


@pytest.mark.parametrize("nq,nk", [([150], [150]), ([1], [700])])
@pytest.mark.parametrize("scale,size", [(-0.3, 1.0), (0.0, 1.0), (2.0, 3.0), (0.125, 0.01)])
def test_scales_and_sharp_weights(gpu, kernels, stream, nq, nk, scale, size):
    for dim, dtype in ((64, "f16"), (256, "bf16")):
        Packed(nq, nk, 4, 2, dim, dtype, scale=scale, size=size).check(kernels, stream)


FAR = [(4, 2, [100], [100]), (4, 1, [3], [2000]), (4, 2, [5, 1], [5, 1]), (64, 2, [400], [400])]  # narrow tiles, runs, wide tiles


@pytest.mark.parametrize("scale", [2.0 ** -127, -(2.0 ** -128), 2.0 ** -149, 0.0])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("heads,kv,nq,nk", FAR)
def test_scales_below_the_normal_numbers(gpu, kernels, stream, dim, heads, kv, nq, nk, scale):
    """bf16's products of 2^124 and such a scale: scores of about 1/8. The factor of the exponent is rounded to a multiple of 2^-149,
    which moves no score by more than 2^-22, within the 2^-20 that the bound leaves."""
    Packed(nq, nk, heads, kv, dim, "bf16", scale=scale, size=2.0 ** 60).check(kernels, stream)


def winners_mean(p, winner):
    """What rows are whose seen keys t with winner(t) weigh the same and the others nothing: the mean of their values. The weights
    are 1 exactly; `seen` additions of them and of their values are off by 2 U each at most, in numerator and denominator."""
    want, err = np.full((2, p.rows, p.heads, p.dim), np.nan)
    for s in range(len(p.q0) - 1):
        for i in range(p.q0[s], p.q0[s + 1]):
            n = p.k0[s + 1] - p.k0[s] - (p.q0[s + 1] - 1 - i)
            v = p.v[p.k0[s] + np.flatnonzero(winner(np.arange(n)))]
            want[i] = np.repeat(v.mean(0), p.heads // p.kv, 0)
            err[i] = (4 * n + 8) * 2.0 ** -24 * np.repeat(np.abs(v).mean(0), p.heads // p.kv, 0)
    err = err * (1 + HALF[p.dtype]) + HALF[p.dtype] * np.abs(want) + 2.0 ** -25
    rows = slice(p.q0[0], p.q0[-1])
    return want.reshape(p.rows, -1)[rows], err.reshape(p.rows, -1)[rows]


@pytest.mark.parametrize("scale", [300.0, 1e5, 1e25])
@pytest.mark.parametrize("dim,dtype", [(64, "bf16"), (128, "f16"), (256, "bf16"), (256, "f16")])
@pytest.mark.parametrize("heads,kv,nq,nk", FAR)
def test_scores_far_from_zero_weigh_as_others_do(gpu, kernels, stream, dim, dtype, heads, kv, nq, nk, scale):
    """Scores of 2^22.6 times the scale, whose fp32 steps are 2^6 and more: every third key has the largest, or all have the same."""
    for sign, step in ((1.0, 3), (-1.0, 1)):
        p = Packed(nq, nk, heads, kv, dim, dtype, gate=False, scale=scale)
        p.q[:], p.k[:] = 0.0, 0.0
        p.q[..., 3] = 127.0  # (odd: a power of two's product with the scale has no rounding)
        for s in range(len(nq)):
            t = np.arange(nk[s])
            p.k[p.k0[s]:p.k0[s + 1], :, 3] = (sign * np.where(t % step == 0, 201 * 2.0 ** 8, 200 * 2.0 ** 8))[:, None]
        p.qr, p.kr = to_type(p.q, dtype)[0], to_type(p.k, dtype)[0]
        got = p.run(kernels, stream)[p.q0[0]:p.q0[-1]]
        want, err = winners_mean(p, lambda t: t % step == 0)
        assert (np.abs(got - want) <= err).all()


@pytest.mark.parametrize("dim,dtype", [(64, "f16"), (128, "bf16"), (256, "f16")])
@pytest.mark.parametrize("heads,kv,nq,nk", FAR)
def test_scores_far_from_zero_leave_other_rows_alone(gpu, kernels, stream, dim, dtype, heads, kv, nq, nk):
    """Every other row's scores are about 2^29; the rows between are, to the bit, as they are among rows like themselves."""
    clean, far = (Packed(nq, nk, heads, kv, dim, dtype, scale=0.9, size=0.5) for _ in range(2))
    for p in (clean, far):
        p.q[..., 3] = 0.0
        p.k[..., 3] = 201 * 2.0 ** 7
    far.q[1::2, :, 3] = 203 * 2.0 ** 7
    for p in (clean, far):
        p.qr, p.kr = to_type(p.q, dtype)[0], to_type(p.k, dtype)[0]
    a, b = clean.run(kernels, stream), far.run(kernels, stream)
    rows = np.arange(far.q0[0], far.q0[-1])
    assert np.array_equal(a[rows[rows % 2 == 0]], b[rows[rows % 2 == 0]]) and np.isfinite(b[rows]).all()


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("nq,nk", [([90, 90, 90], [90, 90, 90]), ([1, 1, 1], [500, 700, 300])])
def test_what_is_not_finite_stays_in_its_sequence(gpu, kernels, stream, dim, nq, nk):
    clean, bad = (Packed(nq, nk, 4, 2, dim, "f16") for _ in range(2))
    inf = np.float16(np.inf)
    for m, raw in ((bad.k, bad.kr), (bad.v, bad.vr)):
        raw[bad.k0[1]:bad.k0[2]:7] = inf
    bad.qr[bad.q0[1]] = np.float16(np.nan)
    a, b = clean.run(kernels, stream), bad.run(kernels, stream)
    for s in (0, 2):
        rows = slice(int(clean.q0[s]), int(clean.q0[s + 1]))
        assert np.array_equal(a[rows], b[rows]) and np.isfinite(a[rows]).all()
    assert np.isnan(b[int(bad.q0[1])]).all()


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("nq,nk", [([100], [100]), ([3], [400])])
def test_keys_of_infinite_score_are_followed(gpu, kernels, stream, dim, nq, nk):
    """A key of -infinity weighs nothing; a row that sees no other is NaN; a key that is NaN makes the rows that see it NaN
    and no others."""
    p = Packed(nq, nk, 2, 1, dim, "f16", gate=False)
    p.qr[:] = np.abs(p.qr)
    p.q[:] = np.abs(p.q)
    for at, value in ((p.k0[0] + 5, -np.inf), (p.k0[0] + nk[0] - 2, np.nan)):
        p.kr[at], p.k[at] = value, value
    if nq[0] == nk[0]:
        p.kr[p.k0[0]], p.k[p.k0[0]] = -np.inf, -np.inf
    got = p.check(kernels, stream)
    assert np.isnan(got[-2:]).all() and np.isfinite(got[1 if nq[0] == nk[0] else 0:-2]).all()
    assert np.isnan(got[0]).all() == (nq[0] == nk[0])


HIDDEN = [  # narrow tiles, runs, rows that see nothing, wide tiles
    (4, 2, [100], [100]), (4, 1, [37, 5], [90, 300]), (4, 2, [3], [2000]), (4, 2, [40], [11]), (64, 2, [400], [400]),
    (64, 2, [150, 250], [60, 700]),
]


@pytest.mark.parametrize("dim,dtype", [(64, "bf16"), (128, "f16"), (256, "bf16")])
@pytest.mark.parametrize("heads,kv,nq,nk", HIDDEN)
def test_values_that_a_row_does_not_see_may_be_anything(gpu, kernels, stream, dim, dtype, heads, kv, nq, nk):
    """The last keys of each sequence have values of NaN and infinity in some columns: the rows before them, and other columns,
    are as they would be without, to the bit; what sees an infinity is one, what sees a NaN or both infinities is NaN."""
    clean, bad = (Packed(nq, nk, heads, kv, dim, dtype, size=0.1) for _ in range(2))
    want = clean.run(kernels, stream)
    marks = np.zeros((3, bad.keys, kv, dim), bool)  # +infinity, -infinity, NaN
    for s in range(len(nq)):
        k1 = bad.k0[s + 1]
        for back, col, what in ((1, 5, 0), (2, dim - 1, 2), (9, 3, 1), (4, 3, 0), (7, 9, 1), (nk[s] // 8, 40, 2)):
            marks[what, max(k1 - back - 1, bad.k0[s]), :, col] = True
    for what, value in enumerate((np.inf, -np.inf, np.nan)):
        bad.vr[marks[what]] = to_type(np.full(1, value), dtype)[0][0]
    got = bad.run(kernels, stream)
    seen = np.zeros((3, bad.rows, heads, dim), bool)
    for s in range(len(nq)):
        for i in range(nq[s]):
            n = max(nk[s] - nq[s] + i + 1, 0)
            seen[:, bad.q0[s] + i] = np.repeat(marks[:, bad.k0[s]:bad.k0[s] + n].any(1), heads // kv, 1)
    plus, minus, nan = seen.reshape(3, bad.rows, -1)
    rows = slice(bad.q0[0], bad.q0[-1])
    nan = nan | plus & minus
    want = np.where(nan, np.nan, np.where(plus, np.inf, np.where(minus, -np.inf, want)))
    assert np.array_equal(got[rows], want[rows], equal_nan=True)


@pytest.mark.parametrize("dim,dtype", [(64, "f16"), (128, "bf16"), (256, "f16")])
@pytest.mark.parametrize("heads,kv,nq,nk", HIDDEN)
def test_infinite_values_of_keys_that_weigh_next_to_nothing(gpu, kernels, stream, dim, dtype, heads, kv, nq, nk):
    """Sharp weights, many of them zero as an operand, and infinite values: the first key's and another's that every row sees if it
    sees any, and the last two keys'. Their columns are infinite or NaN in the rows that see them, never finite; all else is as it
    would be without, to the bit."""
    clean, bad = (Packed(nq, nk, heads, kv, dim, dtype, size=3.0) for _ in range(2))
    want = clean.run(kernels, stream)
    marks = np.zeros((2, bad.keys, kv, dim), bool)  # +infinity, -infinity
    for s in range(len(nq)):
        k0, k1 = int(bad.k0[s]), int(bad.k0[s + 1])
        for key, col, what in ((k0, 5, 0), (k0 + max(nk[s] - nq[s], 0), dim - 1, 1), (k1 - 1, 7, 0), (k1 - 2, 40, 1)):
            marks[what, key, :, col] = True
    for what, value in enumerate((np.inf, -np.inf)):
        bad.vr[marks[what]] = to_type(np.full(1, value), dtype)[0][0]
    got = bad.run(kernels, stream)
    seen = np.zeros((2, bad.rows, heads, dim), bool)
    for s in range(len(nq)):
        for i in range(nq[s]):
            n = max(nk[s] - nq[s] + i + 1, 0)
            seen[:, bad.q0[s] + i] = np.repeat(marks[:, bad.k0[s]:bad.k0[s] + n].any(1), heads // kv, 1)
    plus, minus = seen.reshape(2, bad.rows, -1)[:, bad.q0[0]:bad.q0[-1]]
    got, want = got[bad.q0[0]:bad.q0[-1]], want[bad.q0[0]:bad.q0[-1]]
    assert (np.isnan(got[plus]) | (got[plus] == np.inf)).all() and (np.isnan(got[minus]) | (got[minus] == -np.inf)).all()
    assert np.array_equal(got[~(plus | minus)], want[~(plus | minus)]) and np.isfinite(got[~(plus | minus)]).all()


def test_rows_that_see_nothing_are_zero_whatever_they_hold(gpu, kernels, stream):
    for dim in (64, 128, 256):
        p = Packed([9, 300], [4, 0], 4, 2, dim, "bf16")
        p.qr[p.q0[0]:p.q0[0] + 5] = 0x7fc0
        p.g[p.q0[0]:p.q0[0] + 5] = np.nan
        got = p.run(kernels, stream)
        assert (got[p.q0[0]:p.q0[0] + 5] == 0).all() and (got[p.q0[1]:p.q0[2]] == 0).all()
        assert np.isfinite(got[p.q0[0] + 5:p.q0[1]]).all()


def test_as_many_heads_and_sequences_as_a_launch_takes(gpu, kernels, stream):
    nq = [0] * 2040 + [1, 2, 0]
    Packed(nq, [0] * 2040 + [3, 2, 1], 1024, 1024, 64, "f16", gate=False).check(kernels, stream)
    p = Packed(nq, [0] * 2040 + [3, 2, 1], 1024, 1024, 64, "bf16", gate=False)
    want = p.run(kernels, stream)
    p.batch.c.max_k = 5000  # the hint that would have long sequences divided
    y = p.blank()
    p.call(kernels, stream, y)
    sync()
    assert np.array_equal(p.taken(to_host(y)), want, equal_nan=True)


def test_k0_may_be_q0_and_entries_past_the_rows_end_there(gpu, kernels, stream):
    p = Packed([50, 40], [50, 40], 4, 2, 128, "f16", pad=0)
    want = p.run(kernels, stream)
    for q0 in (p.q0, [0, 50, 0xffffffff], [0, 50, 91]):
        d = u32(q0)
        p.batch = PackedBatch((d, 0), (d, 0), 2, p.rows, p.keys, 50)
        y = p.blank()
        p.call(kernels, stream, y)
        sync()
        assert np.array_equal(p.taken(to_host(y)), want)


@pytest.mark.parametrize("max_k", [0, 1, 700, 0xffffffff])
def test_the_longest_length_is_a_hint(gpu, kernels, stream, max_k):
    p = Packed([1, 3], [700, 90], 8, 2, 128, "f16")
    p.device()
    p.batch = PackedBatch((p.q0d, 0), (p.k0d, 0), 2, p.rows, p.keys, max_k)
    y = p.blank()
    p.call(kernels, stream, y)
    sync()
    got, (want, err) = p.taken(to_host(y)), p.want()
    rows = slice(int(p.q0[0]), int(p.q0[-1]))
    assert (np.abs(got - want)[rows] <= err[rows] + 2.0 ** -24).all()


def test_nothing_is_launched_for_no_rows(gpu, stream):
    k = Kernels()
    p = Packed([3], [3], 4, 2, 64, "f16", pad=0)
    p.device()
    y = p.blank()
    for seqs, rows in ((0, 3), (1, 0)):
        p.batch = PackedBatch((p.q0d, 0), (p.k0d, 0), seqs, rows, p.keys, 3)
        p.call(k, stream, y)
    sync()
    assert (to_host(y) == 0x1234).all() and k.gemm.fast_pipelines() == 0
    k.ctx.close()


def test_warm_up_loads_packed_attention(gpu, stream):
    k = Kernels()
    k.gemm.warm_up(stream, 64)
    loaded = k.gemm.fast_pipelines()
    for nq, nk, heads in (([1], [3000], 4), ([700], [700], 32), ([5], [5], 4)):
        Packed(nq, nk, heads, 2, 128, "f16").run(k, stream)
    assert k.gemm.fast_pipelines() == loaded
    k.ctx.close()


def test_the_same_call_gives_the_same_bits_on_any_stream(gpu):
    k = Kernels()
    ps = [Packed(nq, nk, 8, 2, 128, "bf16", seed=i) for i, (nq, nk) in
          enumerate([([1, 1], [3000, 700]), ([1] * 5, [900] * 5), ([2000, 700], [2000, 700]), ([200, 70], [200, 70])])]
    wants = [p.run(k, 0) for p in ps]
    streams = [Stream() for _ in ps]
    ys = [p.blank() for p in ps]
    for _ in range(4):
        for p, s, y in zip(ps, streams, ys):
            p.call(k, s.handle, y)
    for p, s, y, want in zip(ps, streams, ys, wants):
        s.synchronize()
        assert np.array_equal(p.taken(to_host(y)), want)
    k.ctx.close()


@pytest.mark.parametrize("heads,kv,dim", [(8, 2, 128), (16, 4, 256), (8, 1, 64)])
def test_a_step_replays_from_a_graph(gpu, heads, kv, dim):
    """The sizing call holds what the step needs; lengths change between replays, and eager work runs."""
    k = Kernels()
    p = Packed([1, 1, 1], [3000, 40, 900], heads, kv, dim, "f16")
    lens = [p.k0.copy(), np.concatenate([[2], 2 + np.cumsum([1200, 1500, 7])]), np.concatenate([[2], 2 + np.cumsum([1, 0, 64])])]
    wants = []
    p.device()
    for k0 in lens:
        p.k0d.copy_from(k0.astype(np.uint32))
        y = p.blank()
        p.call(k, 0, y)
        sync()
        wants.append(p.taken(to_host(y)))
    s, y = Stream(), p.blank()
    k.attn.packed_ws(s.handle, p.rows, 3, heads, kv, dim)
    g, ge = ctypes.c_void_p(), ctypes.c_void_p()
    check(rt().hipStreamBeginCapture(s.handle, 0), "begin")
    try:
        p.call(k, s.handle, y)
    finally:
        check(rt().hipStreamEndCapture(s.handle, ctypes.byref(g)), "end")
    check(rt().hipGraphInstantiate(ctypes.byref(ge), g, None, None, 0), "instantiate")
    for i in (0, 1, 2, 1, 0):
        p.k0d.copy_from(lens[i].astype(np.uint32))
        y.copy_from(np.full((p.rows, p.ldy), 0x1234, np.uint16))
        check(rt().hipGraphLaunch(ge, s.handle), "launch")
        s.synchronize()
        assert np.array_equal(p.taken(to_host(y)), wants[i])
        Packed([5], [90], heads, kv, dim, "f16").run(k, 0)
    rt().hipGraphExecDestroy(ge)
    k.ctx.close()


def test_keys_past_4_gib(gpu, kernels, stream):
    """Rows of 2^24 elements: a sequence's keys lie 2^32 bytes and more apart, the last at 9 GB."""
    p = Packed([6, 1], [150, 130], 4, 2, 64, "f16", gate=False, pad=0)
    ld = 1 << 24
    p.device()
    kd, vd = DeviceArray((p.keys * ld,), np.uint16), p.d[2]
    for r in range(p.keys):
        row = np.ascontiguousarray(p.kr[r])
        check(rt().hipMemcpy(kd.ptr + r * ld * 2, row.ctypes.data, row.nbytes, 1), "copy")
    want, err = p.want()
    y = p.blank()
    kernels.attn.packed(stream, p.batch, (p.d[0], 0), p.lds[0], (kd, 0), ld, (vd, 0), p.lds[2], "f16", 4, 2, 64, p.scale,
                        (y, 0), p.ldy)
    sync()
    assert (np.abs(p.taken(to_host(y)) - want) <= err + 2.0 ** -24).all()
    kd.free()


# ---- a layer's attention in 8 bits, over the packed prompts of three requests ---------------------------------------
def test_a_layer_over_packed_prompts(gpu, kernels, stream):
    """norm + code -> q | k | v | gate product -> rope -> packed attention -> code -> out product added to the residual.

    Each step is compared with its definition on the step's own inputs as the device holds them: codes exactly, products and
    attention within their bounds."""
    hidden, heads, kv, dim, lens = 384, 4, 2, 128, [70, 1, 33]
    rng = np.random.default_rng(3)
    t, wide = sum(lens), heads * dim
    n = 2 * wide + 2 * kv * dim
    x = rng.standard_normal((t, hidden)).astype(np.float32)
    norm = rng.standard_normal(hidden).astype(np.float32) * 0.1
    w_in = (rng.standard_normal((n, hidden)) * 0.05).astype(np.float16)
    w_out = (rng.standard_normal((hidden, wide)) * 0.05).astype(np.float16)

    def matrix(rows, k, each):
        lds = up(up(rows, each) // each, 4)
        c, s = full((rows, up(k, 128)), np.uint8, 0xff), full((up(k, 512) // 512, lds, 4), np.uint8, 0xff)
        return c, s, Fp8Matrix((c, 0), up(k, 128), (s, 0), lds)

    def coded(c, s, rows, each, k):
        nb = ref.blocks(k)
        e = to_host(s).transpose(1, 0, 2).reshape(-1, to_host(s).shape[0] * 4)[:up(rows, each) // each, :nb].astype(int) - 127
        return to_host(c), e, ref.values(to_host(c), e, each, k)

    xd, nd, wi, wo = to_dev(x), to_dev(norm), to_dev(w_in), to_dev(w_out)
    ci, si, mi = matrix(n, hidden, 128)
    co, so, mo = matrix(hidden, wide, 128)
    cx, sx, mx = matrix(t, hidden, 1)
    ca, sa, ma = matrix(t, wide, 1)
    kernels.fp8.quant_blocks(stream, (wi, 0), hidden, "f16", mi, n, hidden)
    kernels.fp8.quant_blocks(stream, (wo, 0), wide, "f16", mo, hidden, wide)
    kernels.fp8.quant_rows(stream, (xd, 0), hidden, "f32", mx, t, hidden, (nd, 0), True, 1e-6)
    p = full((t, n), np.float32, 0)
    kernels.fp8.gemm(stream, mx, mi, (p, 0), n, t, n, hidden, Epilogue.StoreF32)
    pos = u32(np.concatenate([np.arange(v) for v in lens]))
    fr, amp = rope_freqs(64, 1e6)
    fd = to_dev(np.array(fr, np.float32))
    qkv = full((t, wide + 2 * kv * dim), np.float16, 0)
    row = wide + 2 * kv * dim
    kernels.rope.rope(stream, (p, 0), n, "f32", (qkv, 0), row, "f16", (pos, 0), t, heads + kv, RopeSpec((fd, 0), dim, 64))
    none = RopeSpec((to_dev(np.zeros(32, np.float32)), 0), dim, 64)  # values as fp16, not turned
    kernels.rope.rope(stream, (p, 4 * (wide + kv * dim)), n, "f32", (qkv, 2 * (wide + kv * dim)), row, "f16", (pos, 0), t, kv,
                      none)
    q0 = u32(np.concatenate([[0], np.cumsum(lens)]))
    batch = PackedBatch((q0, 0), (q0, 0), len(lens), t, t, max(lens))
    y = full((t, wide), np.float16, 0)
    kernels.attn.packed(stream, batch, (qkv, 0), row, (qkv, 2 * wide), row, (qkv, 2 * (wide + kv * dim)), row, "f16", heads, kv,
                        dim, dim ** -0.5, (y, 0), wide, (p, 4 * (wide + 2 * kv * dim)), n)
    kernels.fp8.quant_rows(stream, (y, 0), wide, "f16", ma, t, wide)
    kernels.fp8.gemm(stream, ma, mo, (xd, 0), hidden, t, hidden, wide, Epilogue.AddF32)
    sync()

    u = 2.0 ** -24
    hc, he, hv = coded(cx, sx, t, 1, hidden)
    want_c, want_e = ref.quant(ref.normed(x, norm, True, np.float64(np.float32(1e-6))), 1)
    assert np.array_equal(hc, want_c) and np.array_equal(he, want_e)
    ic, ie, iv = coded(ci, si, n, 128, hidden)
    assert all(np.array_equal(a, b) for a, b in zip((ic, ie), ref.quant(w_in.astype(np.float64), 128)))
    got_p = to_host(p).astype(np.float64)
    assert (np.abs(got_p - hv @ iv.T) <= 2 * u * (hidden + 32) * (np.abs(hv) @ np.abs(iv).T) + u * np.abs(got_p)).all()
    got = to_host(qkv).astype(np.float64)
    assert np.array_equal(got[:, wide + kv * dim:], to_host(p)[:, wide + kv * dim:row].astype(np.float16).astype(np.float64))
    want, err = ref.attention(got[:, :wide].reshape(t, heads, dim), got[:, wide:wide + kv * dim].reshape(t, kv, dim),
                              got[:, wide + kv * dim:].reshape(t, kv, dim), to_host(p)[:, row:], dim ** -0.5,
                              to_host(q0).astype(int), to_host(q0).astype(int), heads, kv, HALF["f16"])
    got_y = to_host(y).astype(np.float64)
    assert (np.abs(got_y - want.reshape(t, -1)) <= err.reshape(t, -1) + 2.0 ** -24).all()
    ac, ae, av = coded(ca, sa, t, 1, wide)
    assert all(np.array_equal(a, b) for a, b in zip((ac, ae), ref.quant(got_y, 1)))
    _, _, ov = coded(co, so, hidden, 128, wide)
    out = av @ ov.T
    assert (np.abs(to_host(xd) - x - out) <= 2 * u * (wide + 32) * (np.abs(av) @ np.abs(ov).T) + 2 * u * (np.abs(out) + np.abs(x))).all()
