"""How the 8-bit product divides its work: its planner, called as the library exports it. No GPU."""

import ctypes

import pytest

from decide_amd import _lib
from decide_amd.kernels import Epilogue

WORD = 512  # columns whose scales lie in one word: K is divided at its multiples


class Plan(ctypes.Structure):  # dh::Fp8Plan (decide_amd/csrc/fp8.h)
    _fields_ = [("variant", ctypes.c_int), ("splits", ctypes.c_uint32), ("kps", ctypes.c_uint32), ("mtiles", ctypes.c_uint32),
                ("ntiles", ctypes.c_uint32), ("ws_bytes", ctypes.c_uint64)]


def plan(m, n, k, epi, cus=256):
    f = _lib.load()._ZN2dh13fp8_gemm_planEjjjjj  # fp8_gemm_plan(m, n, k, epi, cus)
    f.restype, f.argtypes = Plan, [ctypes.c_uint32] * 5
    return f(m, n, k, int(epi), cus)


def plan_of(variant, splits, m, n, k):
    f = _lib.load()._ZN2dh16fp8_gemm_plan_ofEijjjj  # fp8_gemm_plan_of(variant, splits, m, n, k)
    f.restype, f.argtypes = Plan, [ctypes.c_int] + [ctypes.c_uint32] * 4
    return f(variant, splits, m, n, k)


@pytest.mark.parametrize("epi", list(Epilogue))
@pytest.mark.parametrize("m,n", [(1, 32), (17, 64), (603, 2560), (16384, 18432)])
def test_no_columns_are_one_part(m, n, epi):
    p = plan(m, n, 0, epi)
    assert p.splits == 1 and p.ws_bytes == 0
    for splits in (1, 2, 16):
        assert plan_of(1, splits, m, n, 0).splits == 1


@pytest.mark.parametrize("epi", list(Epilogue))
@pytest.mark.parametrize("m", [1, 16, 65, 603, 5000])
@pytest.mark.parametrize("n", [32, 2560, 18432])
@pytest.mark.parametrize("k", [1, 512, 513, 2560, 9216, 8200])
def test_parts_cover_the_columns_and_none_is_empty(m, n, k, epi):
    p = plan(m, n, k, epi)
    assert p.kps % WORD == 0 and (p.splits - 1) * p.kps < k <= p.splits * p.kps
    assert p.ws_bytes == (p.splits * m * n * 4 if p.splits > 1 else 0)


@pytest.mark.parametrize("epi", [Epilogue.StoreF32, Epilogue.StoreF16])
@pytest.mark.parametrize("n", [(1 << 32) - 1, (1 << 32) - 4, (1 << 32) - 127, (1 << 32) - 255])
@pytest.mark.parametrize("k", [0, 128, 9216])
def test_columns_up_to_the_last_of_32_bits_are_counted(n, k, epi):
    """Rounding n up to whole tiles passes 32 bits; the caller's limit of one launch counts the tiles."""
    for v, columns in ((0, 256), (1, 128), (2, 128)):
        p = plan_of(v, 1, 1, n, k)
        assert p.ntiles == -(-n // columns) and p.mtiles == 1
    p = plan(1, n, k, epi)
    assert p.ntiles >= 1 << 24 and p.splits == 1
