"""8-bit floating point with block scales on the GPU against its definition in 64 bits (packed_reference.py)."""

import ctypes

import numpy as np
import pytest

import packed_reference as ref
from decide_amd.hip import Stream, check, rt
from decide_amd.kernels import Epilogue, Fp8Matrix, Kernels
from gpu_util import full, sync, to_dev, to_host

pytestmark = pytest.mark.gpu

U = 2.0 ** -24  # half a step of fp32, relative
NUMPY = {"f16": np.float16, "bf16": np.uint16, "f32": np.float32}


def to_type(x, dtype):
    """x as values of dtype, and what they are in float64 (bf16: float32 cut to 16 bits)."""
    if dtype == "bf16":
        b = (np.asarray(x, np.float32).view(np.uint32) >> 16).astype(np.uint16)
        return b, (b.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    with np.errstate(over="ignore"):
        v = np.asarray(x, NUMPY[dtype])
    return v, v.astype(np.float64)


def up(x, n):
    return -(-x // n) * n


# ---- coding ---------------------------------------------------------------------------------------------------------
def run_quant(kernels, stream, of, raw, ldx, dtype, rows, k, norm_w=None, add_one=True, eps=1e-6):
    """Codes and scale bytes, after checking that nothing behind them was written."""
    each = 1 if of == "rows" else ref.BLOCK
    groups, words = up(rows, each) // each, up(k, 512) // 512
    ld, lds = up(k, 128) + 48, up(groups, 4) + 4
    codes, scales = full((rows + 1, ld), np.uint8, 0xA5), full((words, lds, 4), np.uint8, 0xA5)
    out, xd = Fp8Matrix((codes, 0), ld, (scales, 0), lds), to_dev(raw)
    if of == "rows":
        wd = None if norm_w is None else to_dev(norm_w)
        kernels.fp8.quant_rows(stream, (xd, 0), ldx, dtype, out, rows, k, None if wd is None else (wd, 0), add_one, eps)
    else:
        kernels.fp8.quant_blocks(stream, (xd, 0), ldx, dtype, out, rows, k)
    sync()
    c, s = to_host(codes), to_host(scales)
    assert (c[rows:] == 0xA5).all() and (c[:, up(k, 128):] == 0xA5).all() and (s[:, groups:] == 0xA5).all()
    return c[:rows, :up(k, 128)], s[:, :groups]


def want_quant(x, of, k):
    codes, e = ref.quant(x, 1 if of == "rows" else ref.BLOCK)
    return codes, ref.scale_bytes(e, len(e))


@pytest.mark.parametrize("of", ["rows", "blocks"])
@pytest.mark.parametrize("rows,k,dtype", [
    (1, 1, "f32"), (1, 128, "f16"), (3, 1001, "f16"), (17, 513, "bf16"), (130, 511, "f32"), (129, 640, "bf16"),
    (5, 2560, "f32"), (257, 130, "f16"), (2, 9216, "f16"),
])
def test_values_are_coded_as_defined(gpu, kernels, stream, of, rows, k, dtype):
    rng = np.random.default_rng(rows * 7 + k)
    ldx = up(k, 8) + 8
    raw, x = to_type(rng.standard_normal((rows, ldx)) * np.exp(3 * rng.standard_normal((rows, ldx))), dtype)
    codes, scales = run_quant(kernels, stream, of, raw, ldx, dtype, rows, k)
    want, bytes_ = want_quant(x[:, :k], of, k)
    assert np.array_equal(scales, bytes_)
    assert np.array_equal(codes, want)


@pytest.mark.parametrize("rows,k,dtype,add_one", [
    (1, 16, "f32", True), (3, 1001, "f16", False), (9, 2560, "f32", True), (2, 4097, "bf16", True),
    (5, 10241, "f16", True), (40, 520, "f32", False),
])
def test_rows_are_normed_before_they_are_coded(gpu, kernels, stream, rows, k, dtype, add_one):
    """The normed values are within a few 2^-52 of the reference's before either rounds to fp32, and a code falls elsewhere
    only where a value then lies that near to a border of both roundings: codes are equal."""
    rng = np.random.default_rng(rows + k)
    ldx = up(k, 8)
    raw, x = to_type(rng.standard_normal((rows, ldx)) * 30 + 1, dtype)
    w = rng.standard_normal(k).astype(np.float32) * 0.3
    codes, scales = run_quant(kernels, stream, "rows", raw, ldx, dtype, rows, k, w, add_one, 1e-5)
    want, bytes_ = want_quant(ref.normed(x[:, :k], w, add_one, np.float64(np.float32(1e-5))), "rows", k)
    assert np.array_equal(scales, bytes_) and np.array_equal(codes, want)


@pytest.mark.parametrize("of", ["rows", "blocks"])
def test_coding_of_extreme_values(gpu, kernels, stream, of):
    """Borders of a scale (448 * 2^e and its neighbours), zeros, fp32's smallest and largest, what is not finite."""
    k = 128 * 9
    x = np.zeros((3, k), np.float32)
    b = x.reshape(3, 9, 128)
    b[0, 0, 5] = 448.0
    b[0, 1, 5] = np.nextafter(np.float32(448.0), np.float32(1000.0))
    b[0, 2, 5] = -448.0 * 2.0 ** -30
    b[0, 3, 5] = 2.0 ** -149
    b[0, 4] = np.float32(3.4028235e38)
    b[0, 5, :4] = [np.inf, -np.inf, np.nan, 3.0]
    b[0, 6, :3] = [np.float32(2.0) ** -100, 448 * 2.0 ** -100, 449 * 2.0 ** -100]
    b[0, 7, :2] = [-0.0, 1.0]
    b[0, 8] = np.inf
    b[1, 0] = np.float32(1e-30) * np.arange(128, dtype=np.float32)
    b[2, 3, 127] = np.float32(-2.0) ** 127
    codes, scales = run_quant(kernels, stream, of, x, k, "f32", 3, k)
    want, bytes_ = want_quant(x.astype(np.float64), of, k)
    assert np.array_equal(scales, bytes_)
    assert np.array_equal(codes, want)


def test_a_row_that_is_not_finite_keeps_to_itself_in_the_norm(gpu, kernels, stream):
    k = 700
    rng = np.random.default_rng(1)
    x = rng.standard_normal((4, 704)).astype(np.float32)
    x[1, 3], x[2, 9] = np.inf, np.nan
    w = np.zeros(k, np.float32)
    codes, scales = run_quant(kernels, stream, "rows", x, 704, "f32", 4, k, w)
    want, bytes_ = want_quant(ref.normed(x[[0, 3], :k], w, True, np.float64(np.float32(1e-6))), "rows", k)
    assert np.array_equal(codes[[0, 3]], want) and np.array_equal(scales[:, [0, 3]], bytes_)
    # x * 0 but for infinity itself, which is infinity * 0; a row with NaN is NaN
    assert (codes[1, :k] & 0x7f == np.where(np.arange(k) == 3, 0x7f, 0)).all() and (codes[2, :k] == 0x7f).all()
    assert (codes[:, k:] == 0).all()


def test_nothing_is_coded_for_no_rows(gpu, stream):
    k = Kernels()
    c = full((4, 128), np.uint8, 7)
    m = Fp8Matrix((c, 0), 128, (c, 256), 4)
    k.fp8.quant_rows(stream, (c, 0), 128, "f16", m, 0, 100)
    k.fp8.quant_blocks(stream, (c, 0), 128, "f16", m, 0, 100)
    k.fp8.quant_rows(stream, (c, 0), 128, "f16", m, 3, 0)
    k.fp8.gemm(stream, m, m, (c, 0), 64, 0, 64, 128, Epilogue.StoreF32)
    k.fp8.gemm(stream, m, m, (c, 0), 64, 3, 0, 128, Epilogue.StoreF32)
    sync()
    assert (to_host(c) == 7).all() and k.gemm.fast_pipelines() == 0
    k.ctx.close()


# ---- the product ----------------------------------------------------------------------------------------------------
class Product:
    """Codes of m and n rows of k columns, in buffers whose strides, rows and scales go on with what must not be read."""

    def __init__(self, m, n, k, seed=0, spread=1.0, codes=None):
        rng = np.random.default_rng(seed + m + n + k)
        self.m, self.n, self.k, wide = m, n, k, up(k, 128)
        if codes is None:
            x, self.ex = ref.quant(rng.standard_normal((m, k)) * np.exp(spread * rng.standard_normal(k)), 1)
            w, self.ew = ref.quant(rng.standard_normal((n, k)) * np.exp(spread * rng.standard_normal((n, 1))), 128)
        else:
            x, w = codes(rng, (m, k)), codes(rng, (n, k))
            x, w = (np.pad(ref.encode(v), ((0, 0), (0, wide - k))) for v in (x, w))
            self.ex = rng.integers(-3, 4, (m, ref.blocks(k)))
            self.ew = rng.integers(-3, 4, (up(n, 128) // 128, ref.blocks(k)))
        self.x, self.w = x, w
        self.ld = wide + 32

    def device(self):
        def matrix(codes, e):
            c = np.full((len(codes) + 1, self.ld), 0x7f, np.uint8)
            c[:-1, :codes.shape[1]] = codes
            lds = up(len(e), 4) + 4
            self.keep = getattr(self, "keep", []) + [to_dev(c), to_dev(ref.scale_bytes(e, lds))]
            return Fp8Matrix((self.keep[-2], 0), self.ld, (self.keep[-1], 0), lds)

        return matrix(self.x, self.ex), matrix(self.w, self.ew)

    def want(self):
        return ref.values(self.x, self.ex, 1, self.k) @ ref.values(self.w, self.ew, 128, self.k).T

    def bound(self, f16):
        """How far the sums may be off. In fp32, each of at most k additions is off by 2 U of the terms' sum. With fp16 outputs
        sums of eight neighbours are cut 13 bits below the largest's leading bit, each of the other seven by one of
        those bits."""
        x, w = (np.abs(np.pad(ref.values(*a, self.k), ((0, 0), (0, up(self.k, 128) - self.k))))
                for a in ((self.x, self.ex, 1), (self.w, self.ew, 128)))
        err = 2 * U * (self.k + 32) * (x @ w.T)
        if f16 and x.shape[0] * w.shape[0] > 1 << 21:  # at most the largest of each side's eight
            err += 7 * 2.0 ** -13 * (x.reshape(len(x), -1, 8).max(2) @ w.reshape(len(w), -1, 8).max(2).T)
        elif f16:
            for c in range(0, x.shape[1], 8):
                err += 7 * 2.0 ** -13 * (x[:, None, c:c + 8] * w[None, :, c:c + 8]).max(2)
        return err

    def run(self, kernels, stream, epi, y0=None, ldy=None):
        wide = self.n // 2 if epi == Epilogue.SwigluF16 else self.n
        ldy = ldy or up(wide, 4) + 4
        f32 = epi in (Epilogue.StoreF32, Epilogue.AddF32)
        y = np.full((self.m + 1, ldy), 77, np.float32 if f32 else np.float16)
        if y0 is not None:
            y[:-1, :wide] = y0
        yd = to_dev(y)
        xm, wm = self.device()
        kernels.fp8.gemm(stream, xm, wm, (yd, 0), ldy, self.m, self.n, self.k, epi)
        sync()
        got = to_host(yd)
        assert (got[-1] == 77).all() and (got[:, wide:] == 77).all()
        return got[:-1, :wide].astype(np.float64)


def as_fp16(got, want, err):
    """Whether fp16 results are `want` within err and one rounding. From 65,520 on what is nearest is infinity; next to that,
    either."""
    far, over = np.abs(want) + err, np.abs(want) - err >= 65520.0
    near = np.abs(got - want) <= err + 2.0 ** -11 * far + 2.0 ** -25
    infinite = got == np.copysign(np.inf, want)
    return np.where(over, infinite, near | (infinite & (far >= 65504.0))).all()


SIZES = [  # every tile, ragged in each direction, K undivided and divided, one and several of what LDS holds of the scales
    (1, 1, 1), (1, 32, 128), (16, 160, 640), (17, 33, 100), (33, 300, 1025), (64, 96, 9216), (65, 129, 65), (127, 64, 4000),
    (300, 257, 777), (500, 128, 8200), (1025, 160, 130), (1300, 300, 1000), (1030, 64, 8320),
]


@pytest.mark.parametrize("m,n,k", SIZES)
def test_product_with_fp32_outputs(gpu, kernels, stream, m, n, k):
    p = Product(m, n, k)
    want, bound = p.want(), p.bound(False)
    got = p.run(kernels, stream, Epilogue.StoreF32)
    assert (np.abs(got - want) <= bound + U * np.abs(want)).all(), (np.abs(got - want) / (bound + 1e-300)).max()
    y0 = np.random.default_rng(m).standard_normal((m, n)).astype(np.float32)
    got = p.run(kernels, stream, Epilogue.AddF32, y0)
    assert (np.abs(got - (want + y0)) <= bound + 2 * U * (np.abs(want) + np.abs(y0))).all()


@pytest.mark.parametrize("m,n,k", [s for s in SIZES if s[0] * s[1] * s[2] <= 1300 * 300 * 1000])
def test_product_with_fp16_outputs(gpu, kernels, stream, m, n, k):
    p = Product(m, n, k)
    want, bound = p.want(), p.bound(True)
    got = p.run(kernels, stream, Epilogue.StoreF16)
    assert as_fp16(got, want, bound)
    if n % 32 == 0:
        # silu's slope is at most 1.1; its exp, reciprocal and products are a few roundings in fp32
        got = p.run(kernels, stream, Epilogue.SwigluF16)
        g = want.reshape(m, -1, 2, 16)
        b = bound.reshape(m, -1, 2, 16)
        with np.errstate(over="ignore"):
            silu = np.abs(g[:, :, 0] / (1.0 + np.exp(-g[:, :, 0])))
        err = 1.1 * b[:, :, 0] * (np.abs(g[:, :, 1]) + b[:, :, 1]) + silu * b[:, :, 1]
        err = err.reshape(m, -1) + 16 * U * np.abs(ref.swiglu(want))
        sw = ref.swiglu(want)
        assert as_fp16(got, sw, err)


def test_product_with_fp16_outputs_in_the_largest_tiles(gpu, kernels, stream):
    m, n, k = 2053, 4128, 650
    p = Product(m, n, k, spread=0.3)
    want, bound = p.want(), p.bound(True)
    assert as_fp16(p.run(kernels, stream, Epilogue.StoreF16), want, bound)
    p = Product(m, 4099, k, codes=lambda rng, shape: rng.integers(-8, 9, shape).astype(np.float64))
    with np.errstate(over="ignore"):
        assert np.array_equal(p.run(kernels, stream, Epilogue.StoreF16), p.want().astype(np.float16).astype(np.float64))
    p = Product(m, n, k, codes=lambda rng, shape: rng.integers(-2, 3, shape).astype(np.float64) / 64)
    want = p.want()
    sw = ref.swiglu(want)  # exact sums: silu's and the product's own roundings
    assert as_fp16(p.run(kernels, stream, Epilogue.SwigluF16), sw, 16 * U * np.abs(sw))


@pytest.mark.parametrize("m,n,k", [(5, 40, 300), (70, 130, 512), (200, 200, 2050), (1100, 96, 700), (1200, 257, 384)])
@pytest.mark.parametrize("epi", [Epilogue.StoreF32, Epilogue.StoreF16])
def test_small_whole_numbers_are_exact(gpu, kernels, stream, m, n, k, epi):
    """Codes of -8 .. 8: eight products' sums lie within the instruction's window, sums stay below 2^24 steps. Scales are
    powers of two between 2^-3 and 2^3."""
    p = Product(m, n, k, codes=lambda rng, shape: rng.integers(-8, 9, shape).astype(np.float64))
    want = p.want()
    got = p.run(kernels, stream, epi)
    with np.errstate(over="ignore"):
        assert np.array_equal(got, want.astype(np.float32 if epi == Epilogue.StoreF32 else np.float16).astype(np.float64))


@pytest.mark.parametrize("m,n", [(1300, 2600), (2050, 4100)])
@pytest.mark.parametrize("epi", [Epilogue.StoreF32, Epilogue.StoreF16])
def test_more_columns_than_their_scales_have_room_for(gpu, kernels, stream, m, n, epi):
    """Small whole numbers again, exact, over 6,700 columns that few or no workgroups share; scales that all differ."""
    k = 6700
    p = Product(m, n, k, codes=lambda rng, shape: rng.integers(-4, 5, shape).astype(np.float64))
    got, want = p.run(kernels, stream, epi), p.want()
    with np.errstate(over="ignore"):
        assert np.array_equal(got, want if epi == Epilogue.StoreF32 else want.astype(np.float16).astype(np.float64))


@pytest.mark.parametrize("m,n,k", [(9, 64, 1100), (150, 140, 300), (1100, 300, 200)])
@pytest.mark.parametrize("epi", [Epilogue.StoreF32, Epilogue.StoreF16])
def test_nan_codes_reach_their_row_and_column_alone(gpu, kernels, stream, m, n, k, epi):
    p = Product(m, n, k, spread=0.0)
    clean = p.run(kernels, stream, epi)
    p.x[m // 2, k - 1] = 0x7f
    p.w[n // 3, 0] = 0xff
    got = p.run(kernels, stream, epi)
    hit = np.zeros((m, n), bool)
    hit[m // 2], hit[:, n // 3] = True, True
    assert np.isnan(got[hit]).all() and np.array_equal(got[~hit], clean[~hit])


def test_all_scales_are_followed(gpu, kernels, stream):
    """Scales from 2^-126 to 2^100 whose products stay within fp32: single codes of 1 and 2."""
    m, n, k = 66, 300, 640
    for epi in (Epilogue.StoreF32, Epilogue.StoreF16):
        for ex, ew in ((-126, 100), (100, -120), (60, -60), (-8, -1)):
            p = Product(m, n, k, codes=lambda rng, s: np.where(rng.random(s) < 0.1, rng.integers(1, 3, s), 0).astype(float))
            p.ex[:], p.ew[:] = ex, ew
            want = p.want()
            got = p.run(kernels, stream, epi)
            t = np.float32 if epi == Epilogue.StoreF32 else np.float16
            assert np.array_equal(got, want.astype(t).astype(np.float64)), (epi, ex, ew)


@pytest.mark.parametrize("value", [448.0, 2.0 ** -9])
@pytest.mark.parametrize("m,n", [(66, 300), (300, 260), (1100, 4100)])
@pytest.mark.parametrize("epi,ends", [(Epilogue.StoreF32, (119, -124)), (Epilogue.StoreF16, (127, -126))])
def test_the_ends_of_the_scales_are_followed(gpu, kernels, stream, m, n, epi, ends, value):
    """The largest and the smallest code at the largest and the smallest scale that all codes are exact with, as x's and as w's;
    the others are of 1 and the inverse scale. Few terms, sums exact."""
    for e in ends:
        for of_x in (True, False):
            p = Product(m, n, 320, codes=lambda rng, s: np.where(rng.random(s) < 0.1, rng.choice([-1.0, 1.0], s), 0.0))
            far, near = (p.x, p.w) if of_x else (p.w, p.x)
            far[(far & 0x7f) == 0x38] += ref.encode(value) - 0x38  # (the sign stays)
            (p.ex if of_x else p.ew)[:], (p.ew if of_x else p.ex)[:] = e, max(-e, -126)
            want, got = p.want(), p.run(kernels, stream, epi)
            assert np.abs(want).max() >= value and np.array_equal(got, want), (e, of_x)


def test_coded_values_past_bfloat16_are_infinite_with_fp32_outputs(gpu, kernels, stream):
    """fp32's largest value is coded as 256 x 2^120: times 2^-120 finite in an fp16 output. The largest that is coded within
    bfloat16's range is finite in both."""
    x = np.zeros((2, 128), np.float64)
    x[0, 0], x[1, 0] = np.float32(3.4028235e38), np.float32(1.93 * 2.0 ** 127)
    p = Product(2, 32, 128)
    p.x, p.ex = ref.quant(x, 1)
    p.w, p.ew = ref.encode(np.ones((32, 128))), np.full((1, 1), -120)
    want = p.want()
    assert (want[:, 0] == (256, 240)).all() and (p.ex == 120).all()
    assert np.array_equal(p.run(kernels, stream, Epilogue.StoreF16), want)
    got = p.run(kernels, stream, Epilogue.StoreF32)
    assert np.isinf(got[0]).all() and np.array_equal(got[1], want[1])


@pytest.mark.parametrize("m,n", [(1, 32), (17, 64), (300, 96), (1100, 4128)])
def test_no_columns_sum_to_zero(gpu, kernels, stream, m, n):
    """K = 0, with codes, scales or neither: zeros are stored, nothing is added, SwiGLU of zeros is zero, as dh_gemm_nt's."""
    some = full((4096,), np.uint8, 0x7f)
    lds = max(up(m, 4), up(up(n, 128) // 128, 4))
    nt_x, nt_w = full((m, 8), np.float16, np.nan), full((n, 8), np.float16, np.nan)
    kernels.fp8.gemm_ws(stream, m, n, 0)
    for x in (Fp8Matrix((some, 0), 0, (some, 0), lds), Fp8Matrix((0, 0), 0, (0, 0), lds), Fp8Matrix((0, 0), 128, (0, 0), lds)):
        for epi in Epilogue:
            wide, f32 = n // 2 if epi == Epilogue.SwigluF16 else n, epi in (Epilogue.StoreF32, Epilogue.AddF32)
            before = np.random.default_rng(m).standard_normal((m + 1, wide + 4)).astype(np.float32 if f32 else np.float16)
            yd, nt = to_dev(before), to_dev(before)
            kernels.fp8.gemm(stream, x, x, (yd, 0), wide + 4, m, n, 0, epi)
            kernels.gemm.gemm(stream, (nt_x, 0), (nt_w, 0), (nt, 0), m, n, 0, 8, 8, wide + 4, epi)
            sync()
            want = before.copy()
            if epi != Epilogue.AddF32:
                want[:m, :wide] = 0
            assert np.array_equal(to_host(yd), want) and np.array_equal(to_host(nt), want)


@pytest.mark.parametrize("n", [(1 << 32) - 4, (1 << 32) - 32, (1 << 32) - 256, 1 << 31])
def test_more_columns_than_a_launch_takes_are_refused(gpu, kernels, stream, n):
    d = full((64,), np.uint8, 7)
    for epi, ldy in ((Epilogue.StoreF32, n), (Epilogue.SwigluF16, n // 2)):
        if epi == Epilogue.StoreF32 or n % 32 == 0:
            m = Fp8Matrix((d, 0), 0, (d, 0), 1 << 26)
            with pytest.raises(AssertionError, match="exceed one launch"):
                kernels.fp8.gemm(stream, m, m, (d, 0), ldy, 1, n, 0, epi)
    sync()
    assert (to_host(d) == 7).all()


def test_a_row_has_the_same_bits_wherever_it_stands(gpu, kernels, stream):
    p = Product(300, 96, 1030)
    p.x[:], p.ex[:] = p.x[0], p.ex[0]
    for epi in (Epilogue.StoreF32, Epilogue.SwigluF16):
        got = p.run(kernels, stream, epi)
        assert (got == got[0]).all()
        assert np.array_equal(got, p.run(kernels, stream, epi))  # and again


def test_product_on_two_streams_at_once_and_after_growth(gpu):
    k = Kernels()
    ps = [Product(40, 64, 9000, seed=i) for i in range(2)]
    more = Product(80, 200, 9000, seed=9)
    alone = [p.run(k, 0, Epilogue.StoreF32) for p in ps]
    streams = [Stream(), Stream()]
    ys = [full((40, 64), np.float32, 0) for _ in ps]
    ms = [p.device() for p in ps]
    y2, m2 = full((80, 200), np.float32, 0), more.device()
    for _ in range(5):
        for s, y, (a, b) in zip(streams, ys, ms):
            k.fp8.gemm(s.handle, a, b, (y, 0), 64, 40, 64, 9000, Epilogue.StoreF32)
        k.fp8.gemm(streams[0].handle, *m2, (y2, 0), 200, 80, 200, 9000, Epilogue.StoreF32)
    for s in streams:
        s.synchronize()
    for y, want in zip(ys, alone):
        assert np.array_equal(to_host(y).astype(np.float64), want)
    k.ctx.close()


def test_a_divided_product_replays_from_a_graph(gpu):
    """Sized by gemm_ws, refused where it would have to grow; every replay is the eager result for what the buffers hold."""
    k = Kernels()
    p, other = Product(33, 64, 9000), Product(33, 64, 9000, seed=5)
    eager = [q.run(k, 0, Epilogue.StoreF32) for q in (p, other)]
    s, y = Stream(), full((33, 64), np.float32, 0)
    xm, wm = p.device()
    codes, scales = p.keep[-4:-2]
    g, ge = ctypes.c_void_p(), ctypes.c_void_p()

    def capture():
        check(rt().hipStreamBeginCapture(s.handle, 0), "begin")
        try:
            k.fp8.gemm(s.handle, xm, wm, (y, 0), 64, 33, 64, 9000, Epilogue.StoreF32)
        finally:
            check(rt().hipStreamEndCapture(s.handle, ctypes.byref(g)), "end")

    with pytest.raises(AssertionError, match="being captured"):
        capture()
    k.fp8.gemm_ws(s.handle, 64, 64, 9000)
    capture()
    check(rt().hipGraphInstantiate(ctypes.byref(ge), g, None, None, 0), "instantiate")
    om, _ = other.device()
    first = [to_host(codes), to_host(scales)]
    second = [to_host(other.keep[0]), to_host(other.keep[1])]
    both = ref.values(other.x, other.ex, 1, 9000) @ ref.values(p.w, p.ew, 128, 9000).T
    for i in range(4):
        for d, h in zip((codes, scales), first if i % 2 == 0 else second):
            d.copy_from(h)
        check(rt().hipGraphLaunch(ge, s.handle), "launch")
        s.synchronize()
        got = to_host(y).astype(np.float64)
        if i % 2 == 0:
            assert np.array_equal(got, eager[0])
        else:
            assert np.allclose(got, both, rtol=0, atol=1e-3 * np.abs(both).max()) and not np.array_equal(got, eager[0])
        other.run(k, 0, Epilogue.StoreF32)  # eager work between replays
    rt().hipGraphExecDestroy(ge)
    k.ctx.close()


@pytest.mark.parametrize("n,k", [(64, 9000), (2560, 9216), (18432, 2560), (257, 4100), (2560, 4096), (1, 16000), (96, 0)])
def test_the_sizing_call_holds_every_call_up_to_its_rows(gpu, n, k):
    """A call that would have to grow the workspace is refused while its stream is captured: none is, of any epilogue."""
    kk, s, most = Kernels(), Stream(), 300
    wide = up(k, 128)
    c, e = full((max(most, n), max(wide, 16)), np.uint8, 0), full((max(up(k, 512) // 512, 1), 304, 4), np.uint8, 127)
    y = full((most, up(n, 4)), np.float32, 0)
    m = Fp8Matrix((c, 0), max(wide, 16), (e, 0), 304)
    kk.fp8.gemm_ws(s.handle, most, n, k)
    g = ctypes.c_void_p()
    check(rt().hipStreamBeginCapture(s.handle, 0), "begin")
    try:
        for rows in [*range(1, 20), *range(20, most, 23), 256, 257, most]:
            for epi in Epilogue:
                if epi != Epilogue.SwigluF16 or n % 32 == 0:
                    kk.fp8.gemm(s.handle, m, m, (y, 0), up(n, 4), rows, n, k, epi)
    finally:
        check(rt().hipStreamEndCapture(s.handle, ctypes.byref(g)), "end")
    rt().hipGraphDestroy(g)
    kk.ctx.close()


def test_rows_past_4_gib(gpu, kernels, stream):
    """Row strides of 2^23 bytes: the last tile's rows lie 2^32 bytes and more behind the first's."""
    from decide_amd.hip import DeviceArray

    m, n, k, ld = 600, 64, 200, 1 << 23
    p = Product(m, n, k)
    xd, wd = DeviceArray((m * ld,), np.uint8), DeviceArray((n * ld,), np.uint8)
    for d, codes in ((xd, p.x), (wd, p.w)):
        c = np.ascontiguousarray(codes)
        for r in range(len(c)):
            check(rt().hipMemcpy(d.ptr + r * ld, c[r].ctypes.data, c.shape[1], 1), "copy")
    sx, sw = to_dev(ref.scale_bytes(p.ex, 600)), to_dev(ref.scale_bytes(p.ew, 4))
    y = full((m, n), np.float32, 0)
    kernels.fp8.gemm(stream, Fp8Matrix((xd, 0), ld, (sx, 0), 600), Fp8Matrix((wd, 0), ld, (sw, 0), 4), (y, 0), n, m, n, k,
                     Epilogue.StoreF32)
    sync()
    want = p.want()
    assert (np.abs(to_host(y) - want) <= p.bound(False) + U * np.abs(want)).all()
    xd.free()
    wd.free()


@pytest.mark.parametrize("rows,of_w", [(515, False), (601, False), (607, False), (601, True), (607, True)])
@pytest.mark.parametrize("epi", [Epilogue.StoreF32, Epilogue.StoreF16])
def test_an_odd_number_of_rows_past_4_gib(gpu, kernels, stream, rows, of_w, epi):
    """X's, or W's, rows 2^23 bytes apart and not a multiple of eight of them: from some row the distance to the last one, in
    bytes, is small again modulo 2^32. Small whole numbers, exact."""
    from decide_amd.hip import DeviceArray

    few, k, ld = 40, 200, 1 << 23
    m, n = (few, rows) if of_w else (rows, few)
    p = Product(m, n, k, codes=lambda rng, shape: rng.integers(-8, 9, shape).astype(np.float64))
    big = DeviceArray((rows * ld,), np.uint8)
    far, near = (p.w, p.x) if of_w else (p.x, p.w)
    for r in range(rows):
        row = np.ascontiguousarray(far[r])
        check(rt().hipMemcpy(big.ptr + r * ld, row.ctypes.data, row.nbytes, 1), "copy")
    nd, sx, sw = to_dev(near), to_dev(ref.scale_bytes(p.ex, up(m, 4))), to_dev(ref.scale_bytes(p.ew, up(len(p.ew), 4)))
    x, w = ((nd, 0), (big, 0)) if of_w else ((big, 0), (nd, 0))
    lds = [near.shape[1], ld] if of_w else [ld, near.shape[1]]
    y = full((m, up(n, 4)), np.float32 if epi == Epilogue.StoreF32 else np.float16, 0)
    kernels.fp8.gemm(stream, Fp8Matrix(x, lds[0], (sx, 0), up(m, 4)), Fp8Matrix(w, lds[1], (sw, 0), up(len(p.ew), 4)), (y, 0),
                     up(n, 4), m, n, k, epi)
    sync()
    got = to_host(y)[:, :n]
    big.free()
    with np.errstate(over="ignore"):
        assert np.array_equal(got, p.want().astype(got.dtype))


def test_warm_up_loads_the_8_bit_kernels(gpu, stream):
    k = Kernels()
    k.gemm.warm_up(stream, 64)
    loaded = k.gemm.fast_pipelines()
    for m, n, kk in SIZES:
        p = Product(m, n, kk) if m * n * kk < 1e7 else None
        for epi in (Epilogue.StoreF32, Epilogue.StoreF16) if p else ():
            p.run(k, stream, epi)
    raw = np.ones((3, 128), np.float32)
    run_quant(k, stream, "rows", raw, 128, "f32", 3, 100)
    run_quant(k, stream, "blocks", raw, 128, "f32", 3, 100)
    assert k.gemm.fast_pipelines() == loaded
    k.ctx.close()
