"""What the operators of packed prompts in 8 bits are timed on and compared over: the coding of rows and weights into
8-bit floating point, the matrix product of such codes, and causal attention over the packed rows of several sequences.

Codes are e4m3 numbers, rows of a stride that is a multiple of 128 columns, columns behind the last one zero. A scale is
a power of two, held as one byte (exponent + 127), for 128 columns of one row (activations) or of 128 rows (weights):
bytes [ceil(columns / 512)][rows or row blocks][4], the four of 512 columns next to each other, 127 behind the last.
"""

from __future__ import annotations

import functools
import math
import random

import torch

own = False

BLOCK = 128  # columns (for weights: rows too) that share a scale
EPS = 1e-6
TORCH = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
SIZE = {"f16": 2, "bf16": 2, "f32": 4}
# (query heads, kv heads, head dims): the decoder's attention layers, and other usual layouts
LAYOUTS = [(16, 4, 256), (32, 8, 128), (12, 4, 128), (8, 1, 64), (8, 8, 64), (20, 4, 256)]
# (columns of the output, columns summed over): the decoder's projections
PROJECTIONS = [(12352, 2560), (10240, 2560), (18432, 2560), (2560, 4096), (2560, 9216)]
SCORES = 32 * 8192 * 8192  # of one call's padded plain form, at most
PRODUCTS = 16384 * 18432 * 2560


def listed():
    a = {"heads": 16, "kv": 4, "dim": 256}
    return [
        # one token for each of 8 sequences: the norm before a layer's first product
        {"name": "code_step", "op": "code", "of": "rows", "rows": 8, "k": 2560, "src": "f32", "norm": True},
        # the MLP's products of a batch of prompts, before the down projection
        {"name": "code_prompts", "op": "code", "of": "rows", "rows": 16383, "k": 9216, "src": "f16", "norm": False},
        # a layer's gate|up weight, once when it is loaded
        {"name": "code_weight", "op": "code", "of": "blocks", "rows": 18432, "k": 2560, "src": "bf16", "norm": False},
        # one token for each of 16 sequences: the weights' bytes
        {"name": "gemm_step", "op": "gemm", "m": 16, "n": 18432, "k": 2560, "epi": "swiglu"},
        # a ticket's prompt through the down projection
        {"name": "gemm_ticket", "op": "gemm", "m": 603, "n": 2560, "k": 9216, "epi": "f32"},
        # nothing divides anything
        {"name": "gemm_odd", "op": "gemm", "m": 1777, "n": 5003, "k": 1001, "epi": "f16"},
        # a batch of prompts through the down projection and through gate|up
        {"name": "gemm_prompts_down", "op": "gemm", "m": 8192, "n": 2560, "k": 9216, "epi": "f32"},
        {"name": "gemm_prompts_up", "op": "gemm", "m": 16384, "n": 18432, "k": 2560, "epi": "swiglu"},
        # one token for each of 64 sequences
        {"name": "attn_step", "op": "attn", "seqs": 64, "rows": 1, "len": 4096, "heads": 32, "kv": 8, "dim": 128,
         "type": "bf16", "gate": False, "ragged": 3},
        # one ticket's prompt
        {"name": "attn_ticket", "op": "attn", "seqs": 1, "rows": 603, "len": 603, "type": "f16", "gate": True,
         "ragged": 0, **a},
        # a batch of prompts of different lengths
        {"name": "attn_prompts", "op": "attn", "seqs": 24, "rows": 2307, "len": 2307, "type": "f16", "gate": True,
         "ragged": 5, **a},
        # one long prompt
        {"name": "attn_long", "op": "attn", "seqs": 1, "rows": 8192, "len": 8192, "heads": 32, "kv": 8, "dim": 128,
         "type": "bf16", "gate": False, "ragged": 0},
    ]


def _log_uniform(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["code", "code", "gemm", "gemm", "gemm", "attn", "attn", "attn"])
    if op == "code":
        of = rng.choice(["rows", "rows", "blocks"])
        rows = _log_uniform(rng, 1, 18432)
        return {"op": op, "of": of, "rows": rows, "k": _log_uniform(rng, 16, min(16384, 16383 * 9216 // rows)),
                "src": rng.choice(["f32", "f16", "bf16"]), "norm": of == "rows" and rng.random() < 0.5}
    if op == "gemm":
        epi = rng.choice(["f32", "f16", "swiglu"])
        n, k = rng.choice(PROJECTIONS)
        if rng.random() < 0.5:
            n, k = _log_uniform(rng, 1, 18432), _log_uniform(rng, 1, 9216)
            if epi == "swiglu":
                n = -(-n // 32) * 32
        return {"op": op, "m": _log_uniform(rng, 1, min(16384, PRODUCTS // (n * k))), "n": n, "k": k, "epi": epi}
    heads, kv, dim = rng.choice(LAYOUTS)
    kind = rng.choice(["prompts", "prompts", "chunks", "steps"])
    seqs = _log_uniform(rng, 1, 64)
    length = _log_uniform(rng, 1, 8192 if kind == "prompts" else 16384)
    most = SCORES // (seqs * heads)
    if kind == "prompts":
        length = rows = min(length, math.isqrt(most))
    else:
        rows = 1 if kind == "steps" else _log_uniform(rng, 1, min(length, most // length))
    return {"op": op, "seqs": seqs, "rows": rows, "len": length, "heads": heads, "kv": kv, "dim": dim,
            "type": rng.choice(["f16", "bf16"]), "gate": rng.random() < 0.5, "ragged": rng.randint(0, 1000)}


# ---- the batch a case stands for, on the host -----------------------------------------------------------------------
def _batch(case):
    """(rows, keys) of every sequence, from the case alone; ragged 0: all alike. Whole prompts stay whole."""
    n, rows, length = case["seqs"], case["rows"], case["len"]
    if not case["ragged"]:
        return [rows] * n, [length] * n
    r = random.Random(case["ragged"])
    lens = [length] + [max(1, int(length ** r.uniform(0.6, 1.0))) for _ in range(1, n)]
    if rows == length:
        return list(lens), lens
    return [min(rows, lens[0])] + [r.randint(0 if rows > 1 and i % 5 == 4 else 1, min(rows, lens[i]))
                                   for i in range(1, n)], lens


# ---- codes and scales -----------------------------------------------------------------------------------------------
def _blocks(k):
    return -(-k // BLOCK)


def _exponent(amax):
    """The exponents (+ 127) of blocks whose largest value is amax (float32)."""
    m, e = torch.frexp(amax)  # amax = m 2^e, m in [1/2, 1): m 2^e <= 448 2^x from x = e - 9 on, or e - 8 past 0.875
    x = torch.where(amax > 0, e - 9 + (m > 0.875).int(), -100)
    return torch.clamp(x, min=-100) + 127


def _codes(x, exponent):
    """x (float32) over its scales as e4m3 numbers."""
    return torch.ldexp(x, 127 - exponent).to(torch.float8_e4m3fn)


def _split(x):
    """x [rows, k] as float32 [rows, blocks, 128], zeros behind the last column."""
    return torch.nn.functional.pad(x.float(), (0, _blocks(x.shape[1]) * BLOCK - x.shape[1])).unflatten(1, (-1, BLOCK))


def _scale_bytes(exponent):
    """Exponents [rows, blocks] in the order that the bytes have."""
    e = torch.nn.functional.pad(exponent, (0, -exponent.shape[1] % 4), value=127).to(torch.uint8)
    return e.unflatten(1, (-1, 4)).transpose(0, 1)


def _code_rows(x):
    """Codes [rows, padded columns] and scale bytes [words][rows][4] of x [rows, k]."""
    b = _split(x)
    e = _exponent(b.abs().amax(2))
    return _codes(b, e[:, :, None]).flatten(1), _scale_bytes(e)


def _code_blocks(w):
    """The same with a scale for 128 rows."""
    b = _split(w)
    rows = _blocks(w.shape[0])
    a = torch.nn.functional.pad(b.abs().amax(2), (0, 0, 0, rows * BLOCK - w.shape[0])).unflatten(0, (rows, BLOCK))
    e = _exponent(a.amax(1))
    of_row = e.repeat_interleave(BLOCK, 0)[:w.shape[0]]
    return _codes(b, of_row[:, :, None]).flatten(1), _scale_bytes(e)


def _values(codes, scales, rows_each, k):
    """The numbers [rows, k] that codes and scale bytes stand for."""
    e = scales.transpose(0, 1).flatten(1)[:, :_blocks(k)].int() - 127
    if rows_each > 1:
        e = e.repeat_interleave(rows_each, 0)[:codes.shape[0]]
    return torch.ldexp(codes.float().unflatten(1, (-1, BLOCK)), e[:, :, None]).flatten(1)[:, :k]


# ---- inputs ---------------------------------------------------------------------------------------------------------
def _normal(g, shape, dtype=torch.float32, mean=0.0, std=1.0):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).mul_(std).add_(mean).to(dtype)


def _u32(values):
    return torch.tensor(values, device="cuda", dtype=torch.int64).to(torch.uint32)


def _room(words, rows):
    """Scale bytes for a matrix of so many rows or row blocks; the library wants a multiple of four."""
    return torch.zeros(words, -(-rows // 4) * 4, 4, device="cuda", dtype=torch.uint8)


def _inputs(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    op = case["op"]
    if op == "code":
        rows, k = case["rows"], case["k"]
        ld = -(-k // 8) * 8
        x = torch.zeros(rows, ld, device="cuda", dtype=TORCH[case["src"]])
        # some columns are far larger than the others, as a model's are
        x[:, :k] = _normal(g, (rows, k)) * torch.exp(1.5 * _normal(g, (1, k)))
        return {"x": x, "norm_w": _normal(g, (k,), std=0.1) if case["norm"] else None}
    if op == "gemm":
        m, n, k = case["m"], case["n"], case["k"]
        x, sx = _code_rows(_normal(g, (m, k)) * torch.exp(_normal(g, (1, k))))
        w, sw = _code_blocks(_normal(g, (n, k), std=0.02) * torch.exp(0.5 * _normal(g, (n, 1))))
        xs, ws = _room(sx.shape[0], m), _room(sw.shape[0], _blocks(n))
        xs[:, :m], ws[:, :_blocks(n)] = sx, sw
        return {"x": x, "sx": xs, "w": w, "sw": ws}
    heads, kv, dim, t = case["heads"], case["kv"], case["dim"], TORCH[case["type"]]
    count, lens = _batch(case)
    q0, k0 = [0], [0]
    for c, n in zip(count, lens):
        q0.append(q0[-1] + c)
        k0.append(k0[-1] + n)
    kvs = _normal(g, (k0[-1], 2, kv, dim))  # a projection's rows: keys, then values
    kvs[:, 1] *= torch.exp(0.5 * _normal(g, (k0[-1], kv, 1)))
    return {"q": _normal(g, (q0[-1], heads * dim), t), "kv": kvs.flatten(1).to(t),
            "gate": _normal(g, (q0[-1], heads * dim)) if case["gate"] else None, "q0": _u32(q0), "k0": _u32(k0),
            "count": count, "lens": lens}


def prepare(case, seed):
    i = _inputs(case, seed)
    s = {"case": case, "i": i, "stream": int(torch.cuda.current_stream().cuda_stream)}
    op = case["op"]
    if op == "code":
        each = 1 if case["of"] == "rows" else BLOCK
        codes = torch.empty(case["rows"], _blocks(case["k"]) * BLOCK, device="cuda", dtype=torch.uint8)
        rows = -(-case["rows"] // each)
        scales = _room(-(-case["k"] // 512), rows)
        s["codes"], s["scales"] = codes, scales
        s["out"] = {"codes": codes.view(torch.float8_e4m3fn), "scales": scales[:, :rows]}
    if op == "gemm":
        wide = case["n"] // 2 if case["epi"] == "swiglu" else case["n"]
        s["y"] = torch.empty(case["m"], -(-wide // 4) * 4, device="cuda",
                             dtype=torch.float32 if case["epi"] == "f32" else torch.float16)
        s["out"] = s["y"][:, :wide]
    if op == "attn":
        s["y"] = torch.empty_like(i["q"])
        seq = torch.repeat_interleave(torch.arange(case["seqs"]), torch.tensor(i["count"]))
        s["seq"] = seq.cuda()  # of each row, and the row's number within it
        s["slot"] = (torch.arange(len(seq)) - i["q0"].long().cpu()[seq]).cuda()
        at = torch.repeat_interleave(torch.arange(case["seqs"]), torch.tensor(i["lens"]))
        s["key_seq"] = at.cuda()  # the same of each key
        s["key_slot"] = (torch.arange(len(at)) - i["k0"].long().cpu()[at]).cuda()
        s["seen"] = (torch.tensor(i["lens"])[seq] - torch.tensor(i["count"])[seq]).cuda() + s["slot"] + 1
    return s


# ---- the framework's calls ------------------------------------------------------------------------------------------
@functools.lru_cache(maxsize=None)
def _kernels():
    from decide_amd.kernels import Kernels

    return Kernels()


def _held(s):
    """What a program keeps beside its tensors: the library's descriptors of its matrices and its batch."""
    from decide_amd.kernels import Epilogue, Fp8Matrix, PackedBatch

    case, i = s["case"], s["i"]
    h = s["held"] = {}
    if case["op"] == "code":
        h["out"] = Fp8Matrix((s["codes"], 0), s["codes"].shape[1], (s["scales"], 0), s["scales"].shape[1])
    if case["op"] == "gemm":
        h["x"] = Fp8Matrix((i["x"], 0), i["x"].shape[1], (i["sx"], 0), i["sx"].shape[1])
        h["w"] = Fp8Matrix((i["w"], 0), i["w"].shape[1], (i["sw"], 0), i["sw"].shape[1])
        h["epi"] = {"f32": Epilogue.StoreF32, "f16": Epilogue.StoreF16, "swiglu": Epilogue.SwigluF16}[case["epi"]]
    if case["op"] == "attn":
        h["batch"] = PackedBatch((i["q0"], 0), (i["k0"], 0), case["seqs"], i["q"].shape[0], i["kv"].shape[0],
                                 max(i["lens"]))
    return h


def _run_own(s):
    case, i, st, k = s["case"], s["i"], s["stream"], _kernels()
    h = s.get("held") or _held(s)
    op = case["op"]
    if op == "code" and case["of"] == "rows":
        norm = None if i["norm_w"] is None else (i["norm_w"], 0)
        k.fp8.quant_rows(st, (i["x"], 0), i["x"].shape[1], case["src"], h["out"], case["rows"], case["k"], norm, True,
                         EPS)
    elif op == "code":
        k.fp8.quant_blocks(st, (i["x"], 0), i["x"].shape[1], case["src"], h["out"], case["rows"], case["k"])
    elif op == "gemm":
        k.fp8.gemm(st, h["x"], h["w"], (s["y"], 0), s["y"].shape[1], case["m"], case["n"], case["k"], h["epi"])
    else:
        wide, narrow = case["heads"] * case["dim"], case["kv"] * case["dim"]
        gate = None if i["gate"] is None else (i["gate"], 0)
        k.attn.packed(st, h["batch"], (i["q"], 0), wide, (i["kv"], 0), 2 * narrow, (i["kv"], 2 * narrow), 2 * narrow,
                      case["type"], case["heads"], case["kv"], case["dim"], case["dim"] ** -0.5, (s["y"], 0), wide,
                      gate, wide if gate else 0)
        return s["y"]
    return s["out"]


# ---- the plain form -------------------------------------------------------------------------------------------------
def _plain_code(s):
    case, i = s["case"], s["i"]
    x = i["x"][:, :case["k"]]
    if i["norm_w"] is not None:  # in 64 bits: a value next to a border decides a scale
        x = x.double()
        x = (x * torch.rsqrt((x * x).mean(1, keepdim=True) + EPS) * (1.0 + i["norm_w"].double())).float()
    codes, scales = _code_rows(x) if case["of"] == "rows" else _code_blocks(x)
    return {"codes": codes, "scales": scales}


def _plain_gemm(s):
    case, i = s["case"], s["i"]
    m, n, k = case["m"], case["n"], case["k"]
    x = _values(i["x"], i["sx"][:, :m], 1, k)
    w = _values(i["w"], i["sw"][:, :_blocks(n)], BLOCK, k)
    y = torch.matmul(x, w.t())
    if case["epi"] == "swiglu":  # columns alternate: 16 of the gate, 16 to be gated
        y = y.unflatten(1, (-1, 2, 16))
        y = (y[:, :, 0] / (1.0 + torch.exp(-y[:, :, 0])) * y[:, :, 1]).flatten(1)
    return y if case["epi"] == "f32" else y.half()


def _plain_attention(s):
    case, i = s["case"], s["i"]
    heads, kv, dim, n = case["heads"], case["kv"], case["dim"], case["seqs"]
    group, rows, length = heads // kv, max(i["count"]), max(i["lens"])
    seq, slot = s["seq"], s["slot"]
    q = torch.zeros(n, kv, rows, group, dim, device="cuda")
    q[seq, :, slot] = i["q"].float().unflatten(1, (kv, group, dim))
    k = torch.zeros(n, kv, dim, length, device="cuda")
    v = torch.zeros(n, kv, length, dim, device="cuda")
    both = i["kv"].float().unflatten(1, (2, kv, dim))
    k[s["key_seq"], :, :, s["key_slot"]] = both[:, 0]
    v[s["key_seq"], :, s["key_slot"]] = both[:, 1]
    seen = torch.zeros(n, rows, device="cuda", dtype=torch.int64)
    seen[seq, slot] = s["seen"]
    score = torch.matmul(q.view(n, kv, rows * group, dim), k).view(n, kv, rows, group, length) * dim ** -0.5
    score = score.masked_fill(torch.arange(length, device="cuda") >= seen[:, None, :, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0.0, 1.0, total)
    o = torch.matmul(p.view(n, kv, rows * group, length), v).view(n, kv, rows, group, dim)[seq, :, slot]
    y = o.reshape(len(seq), heads * dim)
    if i["gate"] is not None:
        y = y / (1.0 + torch.exp(-i["gate"]))
    return y.to(TORCH[case["type"]])


def run(state):
    if own:
        return _run_own(state)
    op = state["case"]["op"]
    return _plain_code(state) if op == "code" else _plain_gemm(state) if op == "gemm" else _plain_attention(state)


# ---- what a pass cannot do without ----------------------------------------------------------------------------------
def work(case):
    op = case["op"]
    if op == "code":
        rows, k = case["rows"], case["k"]
        scales = (rows if case["of"] == "rows" else _blocks(rows)) * _blocks(k)
        return {"bytes": float(rows * k * (SIZE[case["src"]] + 1) + scales + (4 * k if case["norm"] else 0)),
                "flops": (6.0 if case["norm"] else 2.0) * rows * k}
    if op == "gemm":
        m, n, k = case["m"], case["n"], case["k"]
        out = {"f32": 4 * n, "f16": 2 * n, "swiglu": n}[case["epi"]]
        return {"bytes": float((m + n) * k + m * out + (m + _blocks(n)) * _blocks(k)), "flops": 2.0 * m * n * k}
    count, lens = _batch(case)
    heads, kv, dim = case["heads"], case["kv"], case["dim"]
    pairs = sum(c * (n - c) + c * (c + 1) / 2.0 for n, c in zip(lens, count))
    read = sum(2 * kv * dim * 2 * n for n, c in zip(lens, count) if c)
    return {"bytes": float(read + sum(count) * heads * dim * (2 + 2 + (4 if case["gate"] else 0))),
            "flops": 4.0 * pairs * heads * dim}


# ---- the same from the definitions, in 64 bits ----------------------------------------------------------------------
def _numbers(codes):
    """e4m3 codes as 64-bit numbers, by their bits."""
    b = codes.view(torch.uint8).long()
    e, m = (b >> 3) & 15, (b & 7).double()
    size = torch.where(e == 0, m * 2.0 ** -9, (8.0 + m) * torch.exp2((e - 10).double()))
    return torch.where(b >= 128, -size, size)


def _exact_code(case, i):
    k, rows = case["k"], case["rows"]
    x = i["x"][:, :k].double()
    if i["norm_w"] is not None:
        # what is coded is the normed number in float32
        x = x / torch.sqrt(x.square().sum(1, keepdim=True) / k + EPS) * (i["norm_w"].double() + 1.0)
        x = x.float().double()
    nb = _blocks(k)
    wide = torch.zeros(rows, nb * BLOCK, device="cuda", dtype=torch.float64)
    wide[:, :k] = x
    top = wide.view(rows, nb, BLOCK).abs().max(2).values
    if case["of"] == "blocks":
        top = torch.stack([t.max(0).values for t in top.split(BLOCK)])
    # the smallest exponent with top <= 448 * 2^e; log2 of a number next to a border is put right by comparing
    e = torch.ceil(torch.log2(top.clamp(min=2.0 ** -120) / 448.0))
    e = torch.where(448.0 * torch.exp2(e - 1.0) >= top, e - 1.0, e)
    e = torch.where(448.0 * torch.exp2(e) < top, e + 1.0, e).clamp(min=-100.0)
    of_row = e if case["of"] == "rows" else e[torch.arange(rows, device="cuda") // BLOCK]
    y = wide / torch.exp2(of_row).repeat_interleave(BLOCK, 1)
    step = torch.exp2(torch.clamp(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -300))), min=-6.0) - 3.0)
    words = torch.full((e.shape[0], -(-nb // 4) * 4), 127, device="cuda", dtype=torch.uint8)
    words[:, :nb] = (e + 127.0).to(torch.uint8)
    return {"codes": torch.round(y / step) * step, "scales": words.view(e.shape[0], -1, 4).permute(1, 0, 2)}


def _exact_gemm(case, i):
    m, n, k = case["m"], case["n"], case["k"]
    column = torch.arange(k, device="cuda") // BLOCK

    def numbers(codes, scales, of_row):
        e = scales.permute(1, 0, 2).reshape(scales.shape[1], -1).double() - 127.0
        return _numbers(codes)[:, :k] * torch.exp2(e)[of_row][:, column]

    x = numbers(i["x"], i["sx"], torch.arange(m, device="cuda"))
    w = numbers(i["w"], i["sw"], torch.arange(n, device="cuda") // BLOCK)
    y = x @ w.t()
    if case["epi"] == "swiglu":
        at = torch.arange(n // 2, device="cuda")
        at = at // 16 * 32 + at % 16
        y = torch.nn.functional.silu(y[:, at]) * y[:, at + 16]
    return y


def _exact_attention(case, i):
    kv, dim, heads = case["kv"], case["dim"], case["heads"]
    y = torch.zeros(i["q"].shape[0], heads, dim, device="cuda", dtype=torch.float64)
    qa = ka = 0
    for c, n in zip(i["count"], i["lens"]):
        k, v = i["kv"][ka:ka + n].double().view(n, 2, kv, dim).unbind(1)
        hidden = torch.ones(c, n, device="cuda", dtype=torch.bool).triu(n - c + 1)
        for h in range(heads if c else 0):
            q = i["q"][qa:qa + c, h * dim:(h + 1) * dim].double()
            w = (q @ k[:, h // (heads // kv)].t().contiguous() / math.sqrt(dim)).masked_fill(hidden, -math.inf)
            y[qa:qa + c, h] = torch.softmax(w, -1) @ v[:, h // (heads // kv)].contiguous()
        qa, ka = qa + c, ka + n
    y = y.flatten(1)
    return y * torch.sigmoid(i["gate"].double()) if i["gate"] is not None else y


def exact(case, seed):
    i = _inputs(case, seed)
    return {"code": _exact_code, "gemm": _exact_gemm, "attn": _exact_attention}[case["op"]](case, i)
