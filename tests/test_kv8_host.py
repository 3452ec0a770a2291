"""The 8-bit cache's host side: what each entry point refuses, the rotary frequencies, and the page tables. No GPU."""

import ctypes
import math
import random

import numpy as np
import pytest

import kv8_reference as ref
from decide_amd import _lib
from decide_amd.kernels import Pages, kv8_page_bytes, rope_freqs

CACHE = dict(pool=128, pages=8, layers=2, kv_heads=4, head_dim=256, format=0)
BATCH = dict(table=4, row0=4, qpos=4, ld_table=4, seqs=2, rows=10)
ROPE = dict(inv_freq=4, norm_w=16, head_dim=256, rot=64, layout=0, add_one=1, eps=1e-6, amp=1.0)


def _refs(cache, batch, rope):
    return (_lib.DhKv8Cache(**{**CACHE, **cache}), _lib.DhKv8Batch(**{**BATCH, **batch}),
            _lib.DhRopeSpec(**{**ROPE, **rope}))


def _rope(spec={}, **kw):
    a = {**dict(x=16, ldx=4096, xd=2, y=32, ldy=4096, yd=0, pos=4, rows=3, heads=16), **kw}
    p = _refs({}, {}, spec)[2]
    return _lib.load().dh_rope(None, None, a["x"], a["ldx"], a["xd"], a["y"], a["ldy"], a["yd"], a["pos"], a["rows"],
                               a["heads"], ctypes.byref(p))


def _append(cache={}, batch={}, spec={}, **kw):
    a = {**dict(layer=0, k=16, ldk=1024, v=16, ldv=1024, dtype=2), **kw}
    c, b, p = _refs(cache, batch, spec)
    return _lib.load().dh_kv8_append(None, None, ctypes.byref(c), a["layer"], ctypes.byref(b), a["k"], a["ldk"], a["v"],
                                     a["ldv"], a["dtype"], ctypes.byref(p) if spec is not None else None)


def _attention(cache={}, batch={}, **kw):
    a = {**dict(layer=0, q=16, ldq=4096, heads=16, scale=0.0625, gate=16, ldg=4096, y=8, ldy=4096, most=100), **kw}
    c, b, _ = _refs(cache, batch, {})
    return _lib.load().dh_kv8_attention(None, None, ctypes.byref(c), a["layer"], ctypes.byref(b), a["q"], a["ldq"],
                                        a["heads"], a["scale"], a["gate"], a["ldg"], a["y"], a["ldy"], a["most"])


def _copy(cache={}, **kw):
    a = {**dict(src=4, dst=4, n=3), **kw}
    return _lib.load().dh_kv8_copy_pages(None, None, ctypes.byref(_refs(cache, {}, {})[0]), a["src"], a["dst"], a["n"])


def _refused(rc, msg):
    assert rc == _lib.DH_EINVAL
    assert msg in _lib.last_error(), _lib.last_error()


@pytest.mark.parametrize("call", [_rope, _append, _attention, _copy])
def test_a_valid_call_gets_as_far_as_its_missing_context(call):
    _refused(call(), "null context")


@pytest.mark.parametrize("kw,msg", [
    (dict(spec=dict(head_dim=0)), "head_dim"), (dict(spec=dict(head_dim=260)), "head_dim"),
    (dict(spec=dict(head_dim=6)), "head_dim"), (dict(spec=dict(rot=0)), "rot"), (dict(spec=dict(rot=63)), "rot"),
    (dict(spec=dict(rot=258)), "rot"), (dict(spec=dict(layout=2)), "layout"),
    (dict(spec=dict(inv_freq=None)), "inv_freq is null"), (dict(spec=dict(inv_freq=2)), "4-byte"),
    (dict(spec=dict(norm_w=8)), "16-byte"), (dict(spec=dict(amp=math.inf)), "amp"), (dict(spec=dict(eps=0.0)), "eps"),
    (dict(spec=dict(eps=math.nan)), "eps"), (dict(xd=3), "x_dtype"), (dict(yd=9), "y_dtype"),
    (dict(ldx=4092), "row stride"), (dict(ldx=4098), "row stride"), (dict(ldy=4092), "row stride"),
    (dict(x=8), "16-byte aligned"), (dict(y=4), "8-byte aligned"), (dict(pos=2), "pos"),
    (dict(rows=1 << 31), "one launch"), (dict(x=64, y=64), "y may be x only"),
])
def test_rope_refusals(kw, msg):
    _refused(_rope(**kw), msg)


@pytest.mark.parametrize("call", [_append, _attention, _copy])
@pytest.mark.parametrize("kw,msg", [
    (dict(kv_heads=0), "kv_heads"), (dict(kv_heads=1025), "kv_heads"), (dict(head_dim=96), "head_dim"),
    (dict(format=2), "format"), (dict(pages=0), "at least one page"), (dict(layers=0), "one layer"),
    (dict(pool=None), "pool is null"), (dict(pool=64), "128-byte"),
])
def test_cache_refusals(call, kw, msg):
    _refused(call(cache=kw), msg)


@pytest.mark.parametrize("call", [_append, _attention])
@pytest.mark.parametrize("kw,msg", [
    (dict(table=None), "null pointer"), (dict(row0=None), "null pointer"), (dict(qpos=None), "null pointer"),
    (dict(row0=2), "4-byte"), (dict(seqs=1 << 31), "one launch"),
])
def test_batch_refusals(call, kw, msg):
    _refused(call(batch=kw), msg)


@pytest.mark.parametrize("kw,msg", [
    (dict(layer=2), "layer 2 of 2"), (dict(dtype=3), "dtype"), (dict(spec=dict(head_dim=128)), "not the cache's 256"),
    (dict(spec=dict(rot=2, layout=3)), "layout"), (dict(ldk=1020), "row stride"), (dict(ldv=1022), "row stride"),
    (dict(k=8), "16-byte aligned"), (dict(v=4, dtype=0), "8-byte aligned"),
])
def test_append_refusals(kw, msg):
    _refused(_append(**kw), msg)


@pytest.mark.parametrize("kw,msg", [
    (dict(layer=7), "layer 7 of 2"), (dict(heads=0), "multiple of the 4 kv heads"), (dict(heads=18), "multiple of"),
    (dict(heads=4100), "at most 1024"), (dict(scale=math.nan), "scale"), (dict(q=8), "q must be"),
    (dict(ldq=4092), "ldq"), (dict(ldq=4100), "ldq"), (dict(y=4), "y must be"), (dict(ldy=4090), "ldy"),
    (dict(gate=8), "gate must be"), (dict(ldg=4000), "ldg"), (dict(batch=dict(rows=1 << 29)), "one launch"),
])
def test_attention_refusals(kw, msg):
    _refused(_attention(**kw), msg)


@pytest.mark.parametrize("kw,msg", [(dict(n=9), "9 pairs for 8 pages"), (dict(src=2), "4-byte"),
                                    (dict(cache=dict(pages=1 << 30, layers=64), n=1 << 30), "one launch")])
def test_copy_refusals(kw, msg):
    _refused(_copy(**kw), msg)


@pytest.mark.parametrize("call,kw", [
    (_rope, dict(rows=1 << 24)), (_append, dict(batch=dict(rows=1 << 28))), (_append, dict(batch=dict(seqs=1 << 23))),
    (_attention, dict(batch=dict(rows=1 << 31))), (_attention, dict(batch=dict(seqs=1 << 22))),
    (_copy, dict(cache=dict(pages=1 << 26), n=1 << 25))])
def test_what_exceeds_one_launch_is_refused(call, kw):
    """A launch's threads are counted in 32 bits; nothing is launched in part."""
    _refused(call(**kw), "one launch")


def test_null_descriptors_are_refused():
    lib = _lib.load()
    _refused(lib.dh_rope(None, None, 16, 64, 2, 16, 64, 2, 4, 1, 1, None), "null spec")
    _refused(lib.dh_kv8_append(None, None, None, 0, None, 16, 64, 16, 64, 2, None), "null cache")
    _refused(lib.dh_kv8_attention(None, None, None, 0, None, 16, 64, 1, 1.0, None, 0, 8, 64, 1), "null cache")
    _refused(lib.dh_kv8_copy_pages(None, None, None, 4, 4, 1), "null cache")
    c = _lib.DhKv8Cache(**CACHE)
    _refused(lib.dh_kv8_append(None, None, ctypes.byref(c), 0, None, 16, 1024, 16, 1024, 2, None), "null batch")


@pytest.mark.parametrize("kv,dim", [(1, 64), (4, 256), (8, 128), (3, 64)])
def test_page_bytes(kv, dim):
    assert kv8_page_bytes(kv, dim) == ref.page_bytes(kv, dim)
    assert kv8_page_bytes(kv, 96) == 0 and kv8_page_bytes(0, dim) == 0 and kv8_page_bytes(1025, dim) == 0


# ---- frequencies ----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("rot,base,scaling", [(64, 1e7, "plain"), (128, 1e4, "linear"), (64, 1e6, "base"),
                                              (128, 1e7, "parts"), (2, 1e4, "plain"), (4, 1e4, "base")])
def test_rope_freqs(rot, base, scaling):
    f, amp = rope_freqs(rot, base, scaling, factor=8.0, low=1.0, high=32.0, trained_len=4096)
    want = [base ** (-2.0 * i / rot) for i in range(rot // 2)]
    if scaling == "linear":
        want = [v / 8.0 for v in want]
    if scaling == "base":
        want = [(base * 8.0 ** (rot / (rot - 2.0))) ** (-2.0 * i / rot) for i in range(rot // 2)]
        assert f[0] == 1.0 and abs(f[-1] * 8.0 / base ** (-2.0 * (rot // 2 - 1) / rot) - 1.0) < 1e-6
    if scaling == "parts":
        keep = [min(1.0, max(0.0, (4096 * v / (2 * math.pi) - 1.0) / 31.0)) for v in want]
        want = [v / 8.0 * (1.0 - k) + v * k for v, k in zip(want, keep)]
        assert f[0] == np.float32(1.0) and abs(amp - (0.1 * math.log(8.0) + 1.0)) < 1e-6
    else:
        assert amp == 1.0
    # one rounding to fp32 of a value that the two sides form in 64 bits
    assert np.allclose(f, want, rtol=2.0 ** -24 + 1e-14, atol=0)


def test_rope_freqs_refusals():
    for kw, msg in ((dict(rot=3), "rot"), (dict(rot=0), "rot"), (dict(rot=258), "rot"), (dict(base=0.0), "base"),
                    (dict(scaling="linear", factor=0.5), "factor"), (dict(scaling="base", factor=math.inf), "factor"),
                    (dict(scaling="base", rot=2, factor=2.0), "rot > 2"),
                    (dict(scaling="parts", factor=2.0, low=3.0, high=3.0), "low < high"),
                    (dict(scaling="parts", factor=2.0, trained_len=0), "trained_len")):
        with pytest.raises(AssertionError, match=msg):
            rope_freqs(**{**dict(rot=64, base=1e4), **kw})


# ---- page tables ----------------------------------------------------------------------------------------------------
def test_pages_grow_fork_and_copy_on_write():
    p = Pages(10, 4)
    assert p.resize(0, 100) is None and p.table(0) == (100, [0, 1])
    p.fork(0, 1, 100)
    assert p.table(1) == (100, [0, 1]) and p.refs(0) == 2 and p.refs(1) == 2 and p.free() == 8
    # the next token of either goes into page 1, which both hold: whoever comes first gets a copy
    assert p.resize(1, 101) == (1, 2) and p.table(1) == (101, [0, 2]) and p.refs(1) == 1
    assert p.resize(0, 129) is None and p.table(0) == (129, [0, 1, 3])
    # a fork that ends with a whole page copies nothing
    p.fork(0, 2, 64)
    assert p.table(2) == (64, [0]) and p.resize(2, 65) is None and p.table(2) == (65, [0, 4]) and p.refs(0) == 3
    # shrinking into a shared page and growing again splits it too
    assert p.resize(1, 30) is None and p.table(1) == (30, [0])
    assert p.resize(1, 31) == (0, 2) and p.table(1) == (31, [2])
    assert p.resize(0, 0) is None and p.table(0) == (0, []) and p.refs(0) == 1


def test_pages_run_out_without_a_change():
    p = Pages(3, 2)
    p.resize(0, 150)
    p.fork(0, 1, 150)
    before = p.table(0), p.table(1), p.free()
    with pytest.raises(_lib.DecideHipError) as e:  # the split needs a page
        p.resize(1, 151)
    assert e.value.code == _lib.DH_ENOMEM and (p.table(0), p.table(1), p.free()) == before
    with pytest.raises(_lib.DecideHipError):
        p.resize(0, 1 << 63)
    assert (p.table(0), p.table(1), p.free()) == before


def test_pages_refusals():
    p = Pages(4, 2)
    p.resize(0, 10)
    for f, msg in ((lambda: Pages(0, 1), "at least one"), (lambda: Pages(1, 0), "at least one"),
                   (lambda: p.resize(2, 1), "sequence 2 of 2"), (lambda: p.fork(0, 0, 1), "sequences 0 and 0"),
                   (lambda: p.fork(0, 2, 1), "of 2"), (lambda: p.fork(0, 1, 11), "11 tokens of 10"),
                   (lambda: p.table(2), "sequence 2")):
        with pytest.raises(AssertionError, match=msg):
            f()
    p.fork(0, 1, 10)
    with pytest.raises(AssertionError, match="not empty"):
        p.fork(0, 1, 10)
    assert p.refs(99) == 0
    # no room for the moves: refused, nothing changed
    q = Pages(4, 2)
    q.resize(0, 64)
    q.resize(1, 128)
    q.resize(0, 0)
    n = ctypes.c_uint32(7)
    assert _lib.load().dh_pages_compact(q.handle, None, None, 0, ctypes.byref(n)) == _lib.DH_EINVAL
    assert "1 moves, room for 0" in _lib.last_error() and q.table(1) == (128, [1, 2])


@pytest.mark.parametrize("seed", range(6))
def test_pages_against_a_model(seed):
    """Random calls; the contents of pages are tracked by token names, copies and moves carried out as they are asked
    for: every sequence always reads back its own tokens, and no page is lost."""
    r = random.Random(seed)
    pages, seqs = 24, 5
    p = Pages(pages, seqs)
    mem = [[None] * ref.PAGE for _ in range(pages)]
    want = [[] for _ in range(seqs)]
    fresh = 0
    for _ in range(400):
        op, s = r.choice(["grow", "grow", "grow", "shrink", "fork", "free", "compact"]), r.randrange(seqs)
        if op == "grow":
            n = len(want[s]) + r.choice([1, 1, 5, 63, 64, 65, 130])
            try:
                c = p.resize(s, n)
            except _lib.DecideHipError:
                continue
            if c:
                mem[c[1]] = list(mem[c[0]])
            ids = p.table(s)[1]
            for t in range(len(want[s]), n):
                fresh += 1
                want[s].append(fresh)
                mem[ids[t // ref.PAGE]][t % ref.PAGE] = fresh
        elif op in ("shrink", "free"):
            n = r.randint(0, len(want[s])) if op == "shrink" else 0
            assert p.resize(s, n) is None
            del want[s][n:]
        elif op == "fork":
            d = r.randrange(seqs)
            if d != s and not want[d]:
                n = r.randint(0, len(want[s]))
                p.fork(s, d, n)
                want[d] = want[s][:n]
        else:
            moves = p.compact()
            assert not {a for a, _ in moves} & {b for _, b in moves}
            for a, b in moves:
                mem[b] = list(mem[a])
            held = pages - p.free()
            assert all(p.refs(i) > 0 for i in range(held)) and all(p.refs(i) == 0 for i in range(held, pages))
        count = [0] * pages
        for q in range(seqs):
            n, ids = p.table(q)
            assert n == len(want[q]) and len(ids) == -(-n // ref.PAGE)
            assert [mem[ids[t // ref.PAGE]][t % ref.PAGE] for t in range(n)] == want[q]
            for i in ids:
                count[i] += 1
        assert count == [p.refs(i) for i in range(pages)] and p.free() == count.count(0)


# ---- the reference itself -------------------------------------------------------------------------------------------
def test_reference_codes_are_the_nearest():
    rng = np.random.default_rng(3)
    x = np.concatenate([rng.uniform(-448, 448, 4000), rng.uniform(-0.1, 0.1, 4000), [0.0, 448.0, -448.0, 2.0 ** -10]])
    grid = np.sort(np.unique(ref.E4M3[np.isfinite(ref.E4M3)]))
    got = ref.values(ref.encode(x, "e4m3"), "e4m3")
    near = np.abs(x[:, None] - grid).min(1)
    assert np.array_equal(np.abs(got - x), near)
    x = rng.uniform(-127, 127, 4000)
    assert np.abs(ref.values(ref.encode(x, "int8"), "int8") - x).max() <= 0.5
    assert ref.scale_of(448.0, "e4m3") == 1.0 and ref.scale_of(448.1, "e4m3") == 2.0
    assert ref.scale_of(0.0, "e4m3") == ref.FLOOR and ref.scale_of(224.0, "e4m3") == 0.5


# ---- the attention's workspace --------------------------------------------------------------------------------------
class _Plan(ctypes.Structure):
    """``dh::KvAttnPlan`` (decide_amd/csrc/kv8.h)."""

    _fields_ = [("slots", ctypes.c_uint32), ("runs", ctypes.c_uint32), ("min_run", ctypes.c_uint32),
                ("wide", ctypes.c_bool), ("ws_bytes", ctypes.c_uint64)]


def _attention_sizes():
    """(plan of a call, bytes that the sizing call reserves): the library's own functions, by their linked names."""
    lib = ctypes.CDLL(_lib.LIB_PATH)
    plan = lib["_ZN2dh18kv8_attention_planEjjjjjjjj"]
    plan.restype, plan.argtypes = _Plan, [ctypes.c_uint32] * 8
    reserve = lib["_ZN2dh22kv8_attention_ws_bytesEjjjjjj"]
    reserve.restype, reserve.argtypes = ctypes.c_uint64, [ctypes.c_uint32] * 6
    return plan, reserve


@pytest.mark.parametrize("cus", [256, 304, 64])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_the_reserved_workspace_covers_the_call_and_every_smaller_one(dim, cus):
    plan, reserve = _attention_sizes()
    r = random.Random(dim + cus)
    sizes, runs, wide = 0, 0, 0
    for kv in range(1, 129):
        for group in (1, 2, 3, 8):
            for rows in (1, 17, 80, 200, 320, 432, r.randint(1, 700)):
                tokens = r.choice([5000, 8192, r.randint(1, 131072)])
                held = reserve(rows, kv * group, kv, dim, tokens, cus)
                for small in range(3):
                    n, g = (rows, group) if small < 2 else (r.randint(1, rows), r.randint(1, group))
                    t = tokens if small < 2 else r.randint(1, tokens)
                    seqs = 1 if small == 0 else r.randint(1, n)
                    p = plan(n, seqs, kv * g, kv, dim, r.choice([0xFFFFFF, tokens // 64 + 2]), t, cus)
                    assert p.ws_bytes <= held, (kv, group, rows, tokens, n, g, t, seqs, p.wide, p.ws_bytes, held)
                    sizes, runs, wide = sizes + 1, runs + (p.runs > 0), wide + (p.wide and p.runs > 0)
    assert runs > sizes // 20 and (wide > 50 or dim == 64)  # the sweep meets what it is for


@pytest.mark.parametrize("cus", [256, 304, 64])
def test_runs_whose_pages_round_up_past_32_bits_are_not_taken(cus):
    """The device counts the tiles' pages in 32 bits (at most one more than the table has, each), rounds their number up to
    whole runs and adds a run's share to where it starts."""
    plan, _ = _attention_sizes()
    end = 1 << 32
    for rows in (1, 63, 65, 200):
        slots = rows + rows // 16
        for ld_table in (end // slots - 1 - i for i in (0, 1, 2, 5, 100, 300, 1000)):
            p = plan(rows, rows, 4, 4, 64, ld_table, 8192, cus)
            pages = slots * (ld_table + 1)
            assert p.slots == slots and (p.runs or pages > end - 1000)
            if p.runs:
                share = max(-(-pages // p.runs), p.min_run)
                assert pages + p.runs - 1 < end and -(-pages // share) * share < end
