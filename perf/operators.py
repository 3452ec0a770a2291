"""What the operators of the 8-bit paged key/value cache are timed on and compared over: rotary positions, the append
that turns key and value rows into 8-bit pages, the attention that reads them, and the copy that moves pages.

A cache is a pool of pages, uint8 [layers][pages][page bytes]. A page holds 64 tokens of every kv head: K codes
[kv][64][D], V codes [kv][D][64], then float32 scales [kv][2][4] (K's, then V's, one for 16 tokens each), padded to a
multiple of 128 bytes. A code is an e4m3 number whose scale is a power of two, or (int8) a byte b that stands for
b - 128 with scale amax / 127. Sequences name their pages in rows of a table; the rows of a call are those of sequence 0,
then 1, and so on (row0), each with its position (qpos), and see the tokens up to it.
"""

from __future__ import annotations

import functools
import math
import random

import torch

own = False

PAGE, BLOCK = 64, 16  # tokens of a page, tokens that share a scale
NONE = 0xFFFFFFFF  # the position of a row that sees no token
EPS = 1e-6
TORCH = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
# (query heads, kv heads, head dims, rotated dims): the decoder's attention layers, and other usual layouts
LAYOUTS = [(16, 4, 256, 64), (32, 8, 128, 128), (12, 4, 128, 64), (8, 1, 64, 32), (8, 8, 64, 64), (20, 4, 256, 64)]
LAYERS = 8  # attention layers of the 32-layer model


def listed():
    a = {"heads": 16, "kv": 4, "dim": 256}
    return [
        # queries of a follow-up question about a cached state
        {"name": "rope_followup", "op": "rope", "rows": 41, "heads": 16, "dim": 256, "rot": 64, "layout": "half",
         "scaling": "plain", "norm": True, "far": 2348, "src": "f32", "dst": "f16"},
        # interleaved pairs over the whole head, frequencies stretched by parts, positions up to a million
        {"name": "rope_far", "op": "rope", "rows": 8191, "heads": 32, "dim": 128, "rot": 128, "layout": "interleaved",
         "scaling": "parts", "norm": False, "far": 1000000, "src": "f16", "dst": "f16"},
        # one new token for each of 64 sequences: every block but a few is already started
        {"name": "append_step", "op": "append", "seqs": 64, "rows": 1, "len": 8192, "kv": 4, "dim": 256, "rot": 64,
         "rope": True, "src": "f32", "format": "e4m3", "ragged": 3},
        # a long document's prompt, normed and rotated on the way in
        {"name": "append_prompt", "op": "append", "seqs": 1, "rows": 2307, "len": 2307, "kv": 4, "dim": 256,
         "rot": 64, "rope": True, "src": "f32", "format": "e4m3", "ragged": 0},
        # chunks of several prompts at once, rows stored as they are
        {"name": "append_chunks", "op": "append", "seqs": 17, "rows": 603, "len": 1500, "kv": 8, "dim": 128, "rot": 0,
         "rope": False, "src": "f16", "format": "int8", "ragged": 5},
        # one token behind a ticket's prompt: latency
        {"name": "attn_step", "op": "attn", "seqs": 1, "rows": 1, "len": 603, "gate": True, "format": "e4m3",
         "ragged": 0, "blank": False, **a},
        # one token for each of 64 sequences
        {"name": "attn_step_batch", "op": "attn", "seqs": 64, "rows": 1, "len": 8192, "gate": True, "format": "e4m3",
         "ragged": 3, "blank": False, **a},
        # one token behind a very long context: few rows, all of the card
        {"name": "attn_step_far", "op": "attn", "seqs": 1, "rows": 1, "len": 131072, "gate": False, "format": "int8",
         "ragged": 0, "blank": False, "heads": 32, "kv": 8, "dim": 128},
        # a follow-up question behind a cached long document
        {"name": "attn_followup", "op": "attn", "seqs": 1, "rows": 41, "len": 2348, "gate": True, "format": "e4m3",
         "ragged": 0, "blank": False, **a},
        # a long document's whole causal square, some rows padding
        {"name": "attn_prompt", "op": "attn", "seqs": 1, "rows": 2307, "len": 2307, "gate": True, "format": "e4m3",
         "ragged": 0, "blank": True, **a},
        # forks of 20 sequences: each copies its started page, in every layer
        {"name": "copy_fork", "op": "copy", "pages": 64, "moves": 20, "kv": 4, "dim": 256},
        # a pool is compacted
        {"name": "copy_compact", "op": "copy", "pages": 1024, "moves": 400, "kv": 4, "dim": 256},
    ]


def _log_uniform(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rope", "append", "append", "attn", "attn", "attn", "copy"])
    heads, kv, dim, rot = rng.choice(LAYOUTS)
    if op == "rope":
        return {"op": op, "rows": _log_uniform(rng, 1, 8191 * 4096 // max(4096, heads * dim)), "heads": heads,
                "dim": dim, "rot": rot, "layout": rng.choice(["half", "interleaved"]),
                "scaling": rng.choice(["plain", "linear", "base", "parts"]), "norm": rng.random() < 0.5,
                "far": _log_uniform(rng, 1, 1000000), "src": rng.choice(["f32", "f16", "bf16"]),
                "dst": rng.choice(["f16", "bf16"])}
    if op == "copy":
        pages = _log_uniform(rng, 3, 1024)
        return {"op": op, "pages": pages, "moves": _log_uniform(rng, 1, min(400, pages // 2)), "kv": kv, "dim": dim}
    if op == "append":
        seqs = _log_uniform(rng, 1, 64)
        rows = _log_uniform(rng, 1, max(1, 2307 // seqs))
        rope = rng.random() < 0.5
        return {"op": op, "seqs": seqs, "rows": rows, "len": rows + rng.randint(0, 4096), "kv": kv, "dim": dim,
                "rot": rot if rope else 0, "rope": rope, "src": rng.choice(["f32", "f16", "bf16"]),
                "format": rng.choice(["e4m3", "int8"]), "ragged": rng.randint(1, 1000)}
    seqs = _log_uniform(rng, 1, 64)
    most = min(131072, 64 * 8192 * 1024 // (seqs * kv * dim))
    length = _log_uniform(rng, 1, most)
    rows = _log_uniform(rng, 1, max(1, min(length, 2307, 16 * 2307 * 2307 // (seqs * heads * length))))
    return {"op": op, "seqs": seqs, "rows": rows, "len": length, "heads": heads, "kv": kv, "dim": dim,
            "gate": rng.random() < 0.5, "format": rng.choice(["e4m3", "int8"]), "ragged": rng.randint(0, 1000),
            "blank": rng.random() < 0.3}


# ---- the batch a case stands for, on the host -----------------------------------------------------------------------
def _batch(case):
    """(rows, tokens after the call) of every sequence, from the case alone; ragged 0: all alike."""
    n, rows, length = case["seqs"], case["rows"], case["len"]
    if not case["ragged"]:
        return [rows] * n, [length] * n
    r = random.Random(case["ragged"])
    count = [rows] + [r.randint(0 if rows > 1 and i % 5 == 4 else 1, rows) for i in range(1, n)]
    lens = [length] + [max(c, 1, int(length ** r.uniform(0.3, 1.0))) for c in count[1:]]
    return count, lens


def _page_bytes(kv, dim):
    return -(-kv * (2 * PAGE * dim + 32) // 128) * 128


# ---- the pool's parts, as views -------------------------------------------------------------------------------------
def _views(pool, kv, dim):
    """K codes [pages, kv, 4, 16, D], V codes [pages, kv, D, 4, 16], scales [pages, kv, 2, 4] of one layer's pool."""
    kb = kv * PAGE * dim
    k = pool[:, :kb].unflatten(1, (kv, 4, BLOCK, dim))
    v = pool[:, kb:2 * kb].unflatten(1, (kv, dim, 4, BLOCK))
    s = pool[:, 2 * kb:2 * kb + 32 * kv].view(torch.float32).unflatten(1, (kv, 2, 4))
    return k, v, s


def _value(codes, fmt):
    """The numbers that code bytes stand for, without their scale, in float32."""
    if fmt == "e4m3":
        return codes.contiguous().view(torch.float8_e4m3fn).float()
    return codes.float() - 128.0


def _scale(amax, fmt):
    """The scale of blocks whose largest value is amax (float32)."""
    if fmt == "int8":
        return torch.clamp(amax / 127.0, min=2.0 ** -100)
    m, e = torch.frexp(amax)  # amax = m 2^e, m in [1/2, 1): m 2^e <= 448 2^x from x = e - 9 on, or e - 8 past 0.875
    x = torch.where(amax > 0, e - 9 + (m > 0.875).int(), -100)
    return torch.ldexp(torch.ones_like(amax), torch.clamp(x, min=-100))


def _code(x, fmt):
    """x (already divided by its scale) as code bytes."""
    if fmt == "e4m3":
        return x.to(torch.float8_e4m3fn).view(torch.uint8)
    return (torch.round(x) + 128.0).to(torch.uint8)


# ---- inputs ---------------------------------------------------------------------------------------------------------
def _normal(g, shape, dtype=torch.float32, mean=0.0, std=1.0):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).mul_(std).add_(mean).to(dtype)


def _u32(values):
    return torch.tensor(values, device="cuda", dtype=torch.int64).to(torch.uint32)


def _freqs(rot, scaling):
    """inv_freq float32 [rot / 2] and the amplitude; stretched scalings take a model trained on 32,768 tokens 32 times
    further."""
    base, factor, orig, low, high = 1e7, 32.0, 32768.0, 1.0, 32.0
    if scaling == "base":
        base *= factor ** (rot / (rot - 2.0))
    f = [base ** (-2.0 * i / rot) for i in range(rot // 2)]
    if scaling == "linear":
        f = [v / factor for v in f]
    if scaling == "parts":
        keep = [min(1.0, max(0.0, (orig * v / (2 * math.pi) - low) / (high - low))) for v in f]
        f = [v / factor * (1.0 - c) + v * c for v, c in zip(f, keep)]
    return torch.tensor(f, device="cuda", dtype=torch.float32), 0.1 * math.log(factor) + 1.0 if scaling == "parts" else 1.0


def _filled_pool(g, pages, kv, dim, fmt):
    """One layer's pool whose every block holds 16 tokens: unit keys, values of differing size."""
    pool = torch.zeros(pages, _page_bytes(kv, dim), device="cuda", dtype=torch.uint8)
    k, v, s = _views(pool, kv, dim)
    for lo in range(0, pages, 512):
        part = slice(lo, min(pages, lo + 512))
        n = part.stop - lo
        x = _normal(g, (n, kv, 4, BLOCK, dim))
        sc = _scale(x.abs().amax((3, 4)), fmt)
        k[part] = _code(x / sc[..., None, None], fmt)
        s[part, :, 0] = sc
        x = _normal(g, (n, kv, dim, 4, BLOCK)) * torch.exp(0.5 * _normal(g, (n, kv, 1, 4, BLOCK)))
        sc = _scale(x.abs().amax((2, 4)), fmt)
        v[part] = _code(x / sc[:, :, None, :, None], fmt)
        s[part, :, 1] = sc
    return pool


def _inputs(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    op = case["op"]
    if op == "copy":
        pages, n = case["pages"], case["moves"]
        order = torch.randperm(pages, generator=g, device="cuda")
        pool = torch.randint(0, 256, (LAYERS, pages, _page_bytes(case["kv"], case["dim"])), generator=g, device="cuda",
                             dtype=torch.uint8)
        return {"pool": pool, "src": order[:n].to(torch.uint32), "dst": order[n:2 * n].to(torch.uint32)}
    if op == "rope":
        rows, wide = case["rows"], case["heads"] * case["dim"]
        x = _normal(g, (rows, wide), TORCH[case["src"]])
        f, amp = _freqs(case["rot"], case["scaling"])
        return {"x": x, "freq": f, "amp": amp, "norm_w": _normal(g, (case["dim"],), std=0.1) if case["norm"] else None,
                "pos": torch.randint(0, case["far"], (rows,), generator=g, device="cuda").to(torch.uint32)}
    kv, dim, fmt = case["kv"], case["dim"], case["format"]
    count, lens = _batch(case)
    need = [-(-v // PAGE) for v in lens]
    wide = max(need) + 1
    ids = torch.randperm(sum(need) + 3, generator=g, device="cuda")
    table = torch.zeros(len(need), wide, device="cuda", dtype=torch.int64)
    at = 0
    for i, c in enumerate(need):
        table[i, :c] = ids[at:at + c]
        at += c
    rows, start = sum(count), [0]
    for c in count:
        start.append(start[-1] + c)
    first = torch.repeat_interleave(torch.tensor([v - c for v, c in zip(lens, count)]), torch.tensor(count))
    pos = (first + torch.arange(rows) - torch.repeat_interleave(torch.tensor(start[:-1]), torch.tensor(count))).cuda()
    if case.get("blank"):
        pos[5::11] = NONE
    i = {"pool": _filled_pool(g, sum(need) + 3, kv, dim, fmt), "table": table.to(torch.uint32), "row0": _u32(start),
         "qpos": pos.to(torch.uint32), "rows": rows, "count": count, "lens": lens}
    if op == "append":
        wide_kv = 2 * kv * dim  # keys, then values, in one projection's rows
        i["kv"] = _normal(g, (rows, wide_kv), TORCH[case["src"]])
        if case["rope"]:
            i["freq"], i["amp"] = _freqs(case["rot"], "plain")
            i["norm_w"] = _normal(g, (dim,), std=0.1)
        return i
    heads = case["heads"]
    i["q"] = _normal(g, (rows, heads * dim), torch.float16)
    i["gate"] = _normal(g, (rows, heads * dim)) if case["gate"] else None
    return i


def prepare(case, seed):
    i = _inputs(case, seed)
    s = {"case": case, "i": i, "stream": int(torch.cuda.current_stream().cuda_stream)}
    op = case["op"]
    if op == "rope":
        s["y"] = torch.empty(i["x"].shape, device="cuda", dtype=TORCH[case["dst"]])
    if op == "attn":
        s["y"] = torch.empty(i["q"].shape, device="cuda", dtype=torch.float16)
        rows = torch.arange(i["rows"], device="cuda")
        s["seq"] = torch.repeat_interleave(torch.arange(case["seqs"]), torch.tensor(i["count"])).cuda()
        s["slot"] = rows - i["row0"].long()[s["seq"]]  # a row's number within its sequence
    if op == "append":
        # the blocks that the call's rows fall into: page, block of the page, its rows (-1: none of this call's) and
        # how many tokens it held before
        page, block, rows, kept, at = [], [], [], [], 0
        table = i["table"].long().cpu()
        for q, (c, n) in enumerate(zip(i["count"], i["lens"])):
            p = n - c
            while p < n:
                b, k = p // BLOCK, p % BLOCK
                m = min(BLOCK - k, n - p)
                page.append(int(table[q, b // 4]))
                block.append(b % 4)
                rows.append([-1] * k + list(range(at, at + m)) + [-1] * (BLOCK - k - m))
                kept.append(k)
                p, at = p + m, at + m
        s["page"], s["block"], s["kept"] = (torch.tensor(v, device="cuda") for v in (page, block, kept))
        s["block_rows"] = torch.tensor(rows, device="cuda")
    return s


# ---- the framework's calls ------------------------------------------------------------------------------------------
@functools.lru_cache(maxsize=None)
def _kernels():
    from decide_amd.kernels import Kernels

    return Kernels()


def _held(s):
    """What a program keeps beside its tensors: the library's descriptors of its cache, its batch and its rotation."""
    from decide_amd.kernels import Kv8Batch, Kv8Cache, RopeSpec

    case, i = s["case"], s["i"]
    h = s["held"] = {}
    if "freq" in i:
        h["rope"] = RopeSpec((i["freq"], 0), case["dim"], case["rot"], case.get("layout", "half"), i["amp"],
                             None if i["norm_w"] is None else (i["norm_w"], 0), True, EPS)
    if case["op"] == "copy":
        h["cache"] = Kv8Cache((i["pool"], 0), case["pages"], LAYERS, case["kv"], case["dim"], "e4m3")
    elif case["op"] != "rope":
        h["cache"] = Kv8Cache((i["pool"], 0), i["pool"].shape[0], 1, case["kv"], case["dim"], case["format"])
        h["batch"] = Kv8Batch((i["table"], 0), i["table"].shape[1], (i["row0"], 0), (i["qpos"], 0), case["seqs"],
                              i["rows"])
    return h


def _run_own(s):
    case, i, st, k = s["case"], s["i"], s["stream"], _kernels()
    h = s.get("held") or _held(s)
    op = case["op"]
    if op == "rope":
        wide = case["heads"] * case["dim"]
        k.rope.rope(st, (i["x"], 0), wide, case["src"], (s["y"], 0), wide, case["dst"], (i["pos"], 0), case["rows"],
                    case["heads"], h["rope"])
        return s["y"]
    if op == "copy":
        k.kv8.copy_pages(st, h["cache"], (i["src"], 0), (i["dst"], 0), case["moves"])
        return i["pool"]
    kv, dim = case["kv"], case["dim"]
    if op == "append":
        size = i["kv"].element_size()
        k.kv8.append(st, h["cache"], 0, h["batch"], (i["kv"], 0), 2 * kv * dim, (i["kv"], size * kv * dim),
                     2 * kv * dim, case["src"], h.get("rope"))
        return _stored(i["pool"], case)
    wide = case["heads"] * dim
    gate = None if i["gate"] is None else (i["gate"], 0)
    k.kv8.attention(st, h["cache"], 0, h["batch"], (i["q"], 0), wide, case["heads"], dim ** -0.5, (s["y"], 0), wide,
                    case["len"], gate, wide if gate else 0)
    return s["y"]


def _stored(pool, case):
    """What an append leaves: the codes (e4m3 as the numbers that they are) and the scales."""
    k, v, sc = _views(pool, case["kv"], case["dim"])
    codes = pool[:, :2 * case["kv"] * PAGE * case["dim"]]
    return {"codes": codes.view(torch.float8_e4m3fn) if case["format"] == "e4m3" else codes, "scales": sc}


# ---- the plain form -------------------------------------------------------------------------------------------------
def _rope(x, pos, freq, amp, norm_w, rot, layout):
    """x [rows, heads, D] normed and rotated, in 64 bits."""
    x = x.double()
    if norm_w is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * (1.0 + norm_w.double())
    angle = (pos.double()[:, None] * freq.double())[:, None]
    c, s = torch.cos(angle) * amp, torch.sin(angle) * amp
    if layout == "half":
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        y = torch.cat([a * c - b * s, b * c + a * s], -1)
    else:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        y = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
    return torch.cat([y, x[..., rot:]], -1)


def _place(codes, scales, x, kept, new, fmt):
    """The codes and scales of blocks [n, kv, ...] that keep some tokens and take new ones: `codes` and `scales` before,
    x the new tokens' values (0 elsewhere), kept and new masks of tokens."""
    wide = lambda v: v[..., None, None]  # noqa: E731
    s = _scale(x.abs().amax((2, 3)), fmt)
    any_kept = kept.flatten(1).any(1)[:, None]
    s = torch.where(any_kept, torch.maximum(s, scales), s)
    old = _value(codes, fmt) * wide(scales / s)
    old = torch.where(wide(scales == s), codes, _code(old, fmt))
    zero = 0 if fmt == "e4m3" else 128
    out = torch.where(new, _code(x / wide(s), fmt), torch.where(kept, old, torch.full_like(codes, zero)))
    return out, s


def _plain_append(s):
    case, i = s["case"], s["i"]
    kv, dim, fmt = case["kv"], case["dim"], case["format"]
    k = i["kv"][:, :kv * dim].unflatten(1, (kv, dim))
    v = i["kv"][:, kv * dim:].unflatten(1, (kv, dim))
    if case["rope"]:
        k = _rope(k, i["qpos"], i["freq"], i["amp"], i["norm_w"], case["rot"], "half")
    kc, vc, sc = _views(i["pool"], kv, dim)
    page, block, rows = s["page"], s["block"], s["block_rows"]
    new = rows >= 0
    token = torch.arange(BLOCK, device="cuda")
    kept = token < s["kept"][:, None]
    at = rows.clamp(min=0)
    kx = torch.where(new[:, :, None, None], k.float()[at], 0.0).permute(0, 2, 1, 3)  # [blocks, kv, 16, D]
    vx = torch.where(new[:, :, None, None], v.float()[at], 0.0).permute(0, 2, 3, 1)  # [blocks, kv, D, 16]
    before = sc[page, :, :, block]
    kn, ks = _place(kc[page, :, block], before[:, :, 0], kx, kept[:, None, :, None], new[:, None, :, None], fmt)
    vn, vs = _place(vc[page, :, :, block], before[:, :, 1], vx, kept[:, None, None], new[:, None, None], fmt)
    kc[page, :, block], vc[page, :, :, block] = kn, vn
    sc[page, :, :, block] = torch.stack([ks, vs], -1)
    return _stored(i["pool"], case)


def _plain_attention(s):
    case, i = s["case"], s["i"]
    kv, dim, heads, fmt = case["kv"], case["dim"], case["heads"], case["format"]
    n, most, group = case["seqs"], case["rows"], heads // kv
    kc, vc, sc = _views(i["pool"], kv, dim)
    table = i["table"].long()[:, :-(-case["len"] // PAGE)]
    length = table.shape[1] * PAGE
    scale = sc[table]  # [seqs, pages, kv, 2, 4]
    k = (_value(kc[table], fmt) * scale[:, :, :, 0, :, None, None]).permute(0, 2, 5, 1, 3, 4)
    k = k.reshape(n, kv, dim, length)  # keys as columns
    v = (_value(vc[table], fmt) * scale[:, :, :, 1, None, :, None]).permute(0, 2, 1, 4, 5, 3)
    v = v.reshape(n, kv, length, dim)
    seq, slot = s["seq"], s["slot"]
    q = torch.zeros(n, kv, most, group, dim, device="cuda")
    q[seq, :, slot] = i["q"].float().unflatten(1, (kv, group, dim))
    seen = torch.zeros(n, most, device="cuda", dtype=torch.int64)
    pos = i["qpos"].long()
    seen[seq, slot] = torch.where(pos == NONE, 0, pos + 1)
    score = torch.matmul(q.view(n, kv, most * group, dim), k).view(n, kv, most, group, length) * dim ** -0.5
    hidden = torch.arange(length, device="cuda") >= seen[:, None, :, None, None]
    score = score.masked_fill(hidden, -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0.0, 1.0, total)
    o = torch.matmul(p.view(n, kv, most * group, length), v).view(n, kv, most, group, dim)[seq, :, slot]
    y = o.reshape(i["rows"], heads * dim)
    if i["gate"] is not None:
        y = y / (1.0 + torch.exp(-i["gate"]))
    return y.half()


def run(state):
    if own:
        return _run_own(state)
    case, i = state["case"], state["i"]
    op = case["op"]
    if op == "rope":
        x = i["x"].unflatten(1, (case["heads"], case["dim"]))
        y = _rope(x, i["pos"], i["freq"], i["amp"], i["norm_w"], case["rot"], case["layout"])
        return y.flatten(1).to(TORCH[case["dst"]])
    if op == "copy":
        i["pool"][:, i["dst"].long()] = i["pool"][:, i["src"].long()]
        return i["pool"]
    return _plain_append(state) if op == "append" else _plain_attention(state)


# ---- what a pass cannot do without ----------------------------------------------------------------------------------
def work(case):
    op, size = case["op"], {"f16": 2, "bf16": 2, "f32": 4}
    if op == "rope":
        values = case["rows"] * case["heads"] * case["dim"]
        return {"bytes": float(values * (size[case["src"]] + size[case["dst"]]) + 4 * case["rows"]),
                "flops": 6.0 * values}
    if op == "copy":
        return {"bytes": 2.0 * LAYERS * case["moves"] * _page_bytes(case["kv"], case["dim"]), "flops": 0.0}
    count, lens = _batch(case)
    kv, dim = case["kv"], case["dim"]
    if op == "append":
        rows = sum(count)
        kept = sum((n - c) % BLOCK for n, c in zip(lens, count) if c)  # tokens of started blocks, read back
        blocks = sum(-(-n // BLOCK) - (n - c) // BLOCK for n, c in zip(lens, count) if c)
        return {"bytes": float(2 * kv * dim * (rows * (size[case["src"]] + 1) + kept) + 8 * kv * blocks),
                "flops": 12.0 * 2 * kv * dim * rows}
    heads, rows = case["heads"], sum(count)
    seen = [n for n, c in zip(lens, count) if c]
    pairs = sum(c * (n - c) + c * (c + 1) / 2.0 for n, c in zip(lens, count))
    read = sum(2 * kv * dim * n + 8 * kv * -(-n // BLOCK) + 4 * -(-n // PAGE) for n in seen)
    return {"bytes": float(read + rows * heads * dim * (2 + 2 + (4 if case["gate"] else 0))),
            "flops": 4.0 * pairs * heads * dim}


# ---- the same from the definitions, in 64 bits ----------------------------------------------------------------------
def _numbers(codes, fmt):
    """Code bytes as 64-bit numbers, by their bits."""
    b = codes.long()
    if fmt == "int8":
        return (b - 128).double()
    e, m = (b >> 3) & 15, (b & 7).double()
    size = torch.where(e == 0, m * 2.0 ** -9, (8.0 + m) * torch.exp2((e - 10).double()))
    size = torch.where((b & 127) == 127, math.nan, size)
    return torch.where(b >= 128, -size, size)


def _tokens(pool, pages, kv, dim, fmt, n):
    """The first n keys and values [n, kv, D] of the sequence that holds `pages`, in 64 bits."""
    rec = pool[pages]
    kb = kv * PAGE * dim
    sc = rec[:, 2 * kb:2 * kb + 32 * kv].contiguous().view(torch.float32).double().view(-1, kv, 2, 4)
    sc = sc.repeat_interleave(BLOCK, 3)  # one for every token
    k = _numbers(rec[:, :kb], fmt).view(-1, kv, PAGE, dim) * sc[:, :, 0, :, None]
    v = _numbers(rec[:, kb:2 * kb], fmt).view(-1, kv, dim, PAGE) * sc[:, :, 1, None]
    return k.permute(0, 2, 1, 3).reshape(-1, kv, dim)[:n], v.permute(0, 3, 1, 2).reshape(-1, kv, dim)[:n]


def _exact_rope(x, pos, freq, amp, norm_w, rot, layout):
    x = x.double()
    if norm_w is not None:
        x = x / torch.sqrt(x.square().sum(-1, keepdim=True) / x.shape[-1] + EPS) * (norm_w.double() + 1.0)
    z = torch.polar(torch.full((len(x), 1, rot // 2), amp, device=x.device, dtype=torch.float64),
                    torch.outer(pos.double(), freq.double())[:, None])
    pairs = (x[..., :rot].unflatten(-1, (2, rot // 2)).transpose(-1, -2) if layout == "half"
             else x[..., :rot].unflatten(-1, (rot // 2, 2))).contiguous()
    turned = torch.view_as_real(torch.view_as_complex(pairs) * z)
    y = x.clone()
    y[..., :rot] = turned.transpose(-1, -2).flatten(-2) if layout == "half" else turned.flatten(-2)
    return y


def _to_grid(x, fmt):
    """64-bit numbers to the nearest code's number, ties to even."""
    if fmt == "int8":
        return torch.round(x)
    e = torch.clamp(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -300))), min=-6.0)
    step = torch.exp2(e - 3.0)
    return torch.round(x / step) * step


def _exact_append(case, i):
    kv, dim, fmt = case["kv"], case["dim"], case["format"]
    kb, pool = kv * PAGE * dim, i["pool"]
    rows = i["kv"].double().view(-1, 2, kv, dim)
    k, v = rows[:, 0], rows[:, 1]
    if case["rope"]:
        # stored keys are coded from float32: rounded to it once, then to the code
        k = _exact_rope(k, i["qpos"], i["freq"], i["amp"], i["norm_w"], case["rot"], "half").float().double()
    num = _numbers(pool[:, :2 * kb], fmt)
    kn = num[:, :kb].view(-1, kv, 4, BLOCK, dim)
    vn = num[:, kb:].view(-1, kv, dim, 4, BLOCK)
    sc = pool[:, 2 * kb:2 * kb + 32 * kv].contiguous().view(torch.float32).double().view(-1, kv, 2, 4)
    table, at = i["table"].long().cpu(), 0
    for q, (c, n) in enumerate(zip(i["count"], i["lens"])):
        p = n - c
        while p < n:
            b, o = p // BLOCK, p % BLOCK
            m = min(BLOCK - o, n - p)
            page, b = int(table[q, b // 4]), b % 4
            for w, (x, slot) in enumerate(((k[at:at + m], kn[page, :, b]),
                                           (v[at:at + m], vn[page, :, :, b].transpose(1, 2)))):
                x = x.transpose(0, 1)  # [kv, m, D]; slot [kv, 16, D]
                top = x.abs().amax((1, 2))
                if fmt == "int8":
                    s = (top / 127.0).float().double().clamp(min=2.0 ** -100)
                else:
                    s = torch.exp2(torch.clamp(torch.ceil(torch.log2(top / 448.0)), min=-100.0))
                if o:
                    s = torch.maximum(s, sc[page, :, w, b])
                    ratio = (sc[page, :, w, b] / s).float().double()[:, None, None]
                    slot[:, :o] = _to_grid((slot[:, :o] * ratio).float().double(), fmt)
                slot[:, o:o + m] = _to_grid((x / s[:, None, None]).float().double(), fmt)
                slot[:, o + m:] = 0.0
                sc[page, :, w, b] = s
            p, at = p + m, at + m
    codes = num if fmt == "e4m3" else (num + 128.0).to(torch.uint8)
    return {"codes": codes, "scales": sc}


def _exact_attention(case, i):
    kv, dim, heads, fmt = case["kv"], case["dim"], case["heads"], case["format"]
    y = torch.zeros(i["rows"], heads, dim, device="cuda", dtype=torch.float64)
    at = 0
    for s, (c, n) in enumerate(zip(i["count"], i["lens"])):
        if not c:
            continue
        k, v = _tokens(i["pool"], i["table"][s].long()[:-(-n // PAGE)], kv, dim, fmt, n)
        pos = i["qpos"][at:at + c].long()
        hidden = torch.arange(n, device="cuda")[None] >= torch.where(pos == NONE, 0, pos + 1)[:, None]
        for h in range(heads):
            q = i["q"][at:at + c, h * dim:(h + 1) * dim].double()
            w = (q @ k[:, h // (heads // kv)].t().contiguous() / math.sqrt(dim)).masked_fill(hidden, -math.inf)
            y[at:at + c, h] = torch.nan_to_num(torch.softmax(w, -1)) @ v[:, h // (heads // kv)].contiguous()
        at += c
    y = y.view(i["rows"], heads * dim)
    return y * torch.sigmoid(i["gate"].double()) if i["gate"] is not None else y


def exact(case, seed):
    i = _inputs(case, seed)
    op = case["op"]
    if op == "copy":
        return None  # bytes move: there is nothing to compute
    if op == "rope":
        return _exact_rope(i["x"].unflatten(1, (case["heads"], case["dim"])), i["pos"], i["freq"], i["amp"],
                           i["norm_w"], case["rot"], case["layout"]).flatten(1)
    return _exact_append(case, i) if op == "append" else _exact_attention(case, i)
