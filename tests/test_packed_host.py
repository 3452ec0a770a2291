"""What the 8-bit products' and packed attention's entry points refuse, and the reference's own pins. No GPU."""

import ctypes

import numpy as np
import pytest

import packed_reference as ref
from decide_amd import _lib

MATRIX = dict(codes=16, scales=16, ld=2560, lds=16)
BATCH = dict(q0=4, k0=4, seqs=2, q_rows=10, k_rows=12, max_k=6)


def _refused(rc, msg):
    assert rc == _lib.DH_EINVAL
    assert msg in _lib.last_error(), _lib.last_error()


def _rows(out={}, **kw):
    a = {**dict(x=16, ldx=2560, dtype=2, w=16, add=1, eps=1e-6, rows=3, k=2560), **kw}
    m = _lib.DhFp8Matrix(**{**MATRIX, **out})
    return _lib.load().dh_fp8_quant_rows(None, None, a["x"], a["ldx"], a["dtype"], a["w"], a["add"], a["eps"],
                                         ctypes.byref(m), a["rows"], a["k"])


def _blocks(out={}, **kw):
    a = {**dict(x=16, ldx=2560, dtype=2, n=300, k=2560), **kw}
    m = _lib.DhFp8Matrix(**{**MATRIX, **out})
    return _lib.load().dh_fp8_quant_blocks(None, None, a["x"], a["ldx"], a["dtype"], ctypes.byref(m), a["n"], a["k"])


def _gemm(x={}, w={}, **kw):
    a = {**dict(y=16, ldy=512, m=16, n=512, k=2560, epi=0), **kw}
    xm, wm = _lib.DhFp8Matrix(**{**MATRIX, **x}), _lib.DhFp8Matrix(**{**MATRIX, **w})
    return _lib.load().dh_gemm_fp8(None, None, ctypes.byref(xm), ctypes.byref(wm), a["y"], a["ldy"], a["m"], a["n"], a["k"],
                                   a["epi"])


def _attn(batch={}, **kw):
    a = {**dict(q=16, ldq=1024, k=16, ldk=256, v=16, ldv=256, dtype=0, heads=8, kv=2, dim=128, scale=0.1, gate=16, ldg=1024,
                y=16, ldy=1024), **kw}
    b = _lib.DhPackedBatch(**{**BATCH, **batch})
    return _lib.load().dh_attention_packed(None, None, ctypes.byref(b), a["q"], a["ldq"], a["k"], a["ldk"], a["v"], a["ldv"],
                                           a["dtype"], a["heads"], a["kv"], a["dim"], a["scale"], a["gate"], a["ldg"],
                                           a["y"], a["ldy"])


@pytest.mark.parametrize("call", [_rows, _blocks, _gemm, _attn])
def test_a_valid_call_gets_as_far_as_its_missing_context(call):
    _refused(call(), "null context")


@pytest.mark.parametrize("kw,msg", [
    (dict(dtype=3), "dtype 3"), (dict(ldx=2552), "covering K"), (dict(ldx=2564), "multiple of 8"), (dict(x=8), "16-byte"),
    (dict(out=dict(ld=2544)), "covering 2560 columns"), (dict(out=dict(ld=2568)), "multiple of 16"),
    (dict(k=2561, ldx=2568), "covering 2688 columns"), (dict(out=dict(lds=0)), "multiple of 4 covering"),
    (dict(out=dict(lds=18)), "multiple of 4 covering"), (dict(out=dict(codes=8)), "16-byte"),
    (dict(out=dict(scales=4)), "16-byte"), (dict(w=4), "norm_w"), (dict(eps=0.0), "eps"), (dict(eps=float("nan")), "eps"),
    (dict(out=dict(ld=(1 << 23) + 16)), "2^23"), (dict(rows=17), "covering its 17"),
    (dict(rows=1 << 26, out=dict(lds=1 << 26)), "exceed one launch"),
])
def test_coding_rows_refuses(kw, msg):
    _refused(_rows(**kw), msg)


@pytest.mark.parametrize("kw,msg", [
    (dict(dtype=9), "dtype 9"), (dict(ldx=2000), "covering K"), (dict(n=2049), "covering its 17"),
    (dict(out=dict(ld=100)), "covering 2560"), (dict(n=0xffffffff, out=dict(lds=1 << 26)), "exceed one launch"),
])
def test_coding_weights_refuses(kw, msg):
    _refused(_blocks(**kw), msg)


@pytest.mark.parametrize("kw,msg", [
    (dict(epi=4), "epilogue 4"), (dict(epi=3, n=48), "multiple of 32"), (dict(x=dict(ld=2048)), "of x must"),
    (dict(w=dict(ld=2050)), "of w must"), (dict(x=dict(lds=12)), "of x must"), (dict(w=dict(lds=0)), "of w must"),
    (dict(m=17), "of x must"), (dict(n=2049, ldy=2052), "of w must"), (dict(ldy=508), "ldy = 508"), (dict(ldy=514), "ldy = 514"),
    (dict(y=8), "multiple of 16"), (dict(y=4, epi=1), "multiple of 8"), (dict(x=dict(codes=24)), "16-byte"),
    (dict(k=2561), "covering 2688"),
])
def test_the_product_refuses(kw, msg):
    _refused(_gemm(**kw), msg)


@pytest.mark.parametrize("kw,msg", [
    (dict(dim=96, ldq=4096), "head_dim = 96"), (dict(kv=0), "kv_heads = 0"), (dict(heads=7), "multiple of the 2"),
    (dict(heads=4096, kv=2, ldq=1 << 20, ldg=1 << 20, ldy=1 << 20), "at most 1024"), (dict(dtype=2), "dtype 2"),
    (dict(scale=float("inf")), "scale"), (dict(ldq=1016), "of q must"), (dict(ldq=1028), "of q must"), (dict(ldk=248), "of k"),
    (dict(ldv=260), "of v"), (dict(ldy=1022), "of y"), (dict(ldg=1022), "of gate"), (dict(q=8), "q must be 16"),
    (dict(k=4), "k must be 16"), (dict(v=2), "v must be 16"), (dict(y=4), "y must be 8"), (dict(gate=8), "gate must be 16"),
    (dict(ldk=1 << 25), "2^24"), (dict(batch=dict(q0=2)), "4-byte"), (dict(batch=dict(k0=1)), "4-byte"),
    (dict(batch=dict(q_rows=1 << 30)), "exceed one launch"),
    (dict(heads=2, ldq=256, batch=dict(seqs=1 << 23)), "exceed one launch"),
])
def test_packed_attention_refuses(kw, msg):
    _refused(_attn(**kw), msg)


@pytest.mark.parametrize("scale", [1.8e38, -1.8e38, 3.4e38, -3.4e38, float("nan"), float("-inf")])
def test_scales_past_2_to_the_127_are_refused(scale):
    """Times log2(e), by which the exponents are taken, they would be infinite."""
    _refused(_attn(scale=scale), "scale")
    for fine in (2.0 ** 127, -(2.0 ** 127), 2.0 ** -149, 0.0):
        _refused(_attn(scale=fine), "null context")


def test_scale_strides_past_their_addressing_are_refused():
    wide = dict(lds=(1 << 26) + 4)
    _refused(_rows(out=wide), "exceeds 2^26")
    _refused(_blocks(out=wide), "exceeds 2^26")
    _refused(_gemm(x=wide), "of x exceeds 2^26")
    _refused(_gemm(w=wide), "of w exceeds 2^26")


def test_sizing_calls_refuse():
    lib = _lib.load()
    _refused(lib.dh_gemm_fp8_ws(None, None, 16, 64, 64), "null context")
    _refused(lib.dh_attention_packed_ws(None, None, 16, 1, 8, 3, 64), "multiple of the 3")
    _refused(lib.dh_attention_packed_ws(None, None, 16, 1, 8, 2, 32), "head_dim = 32")
    _refused(lib.dh_attention_packed_ws(None, None, 16, 1, 8, 2, 64), "null context")


def test_the_reference_codes_as_the_format_says():
    assert ref.E4M3[0x7e] == 448.0 and ref.E4M3[1] == 2.0 ** -9 and ref.E4M3[0x38] == 1.0 and ref.E4M3[0xb8] == -1.0
    fine = np.array([c for c in range(256) if c & 127 != 127])
    assert np.array_equal(ref.encode(ref.E4M3[fine]), fine)
    # halfway goes to the even code, a little beyond to the nearer one
    assert ref.encode(1.0625) == 0x38 and ref.encode(1.1875) == 0x3a and ref.encode(1.0626) == 0x39
    assert ref.encode(2.0 ** -10) == 0 and ref.encode(3 * 2.0 ** -10) == 2 and ref.encode(-np.inf) == 0x7f
    assert list(ref.exponent(np.array([0.0, 448.0, 448.1, 224.0, 225.0, 1.0]))) == [-100, 0, 1, -1, 0, -8]


def test_the_reference_attention_is_causal_from_the_end():
    """Equal keys: a row's output is the mean of the values that it sees."""
    q, k = np.ones((5, 1, 64)), np.ones((8, 1, 64))
    v = np.repeat(np.arange(8.0), 64).reshape(8, 1, 64)
    y, _ = ref.attention(q, k, v, None, 0.1, [0, 2, 5], [0, 4, 6], 1, 1, 0.0)
    assert np.allclose(y[:, 0, 0], [1.0, 1.5, 0.0, 4.0, 4.5])
