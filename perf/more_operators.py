"""The 4-bit format's operators, as measurable cases.

MXFP4 holds 32 consecutive elements of a row as e2m1 codes (4 bits) beside one
power of two (e8m0, 8 bits): 4.25 bits an element. ``quantize_mxfp4`` and
``dequant_mxfp4`` turn rows into it and back, ``gemv_mxfp4`` multiplies a
weight in it by the 16-bit activations of a decode batch, ``gemm_mxfp4`` by
activations that are MXFP4 too (prompts), ``qk_norm_rope_paged`` appends keys
and values to a paged cache in it and ``attn_decode_paged`` attends over that
cache.

``listed()`` names the cases, ``draw(rng)`` draws more of the same ranges;
``prepare`` makes a case's inputs, ``run`` is one pass (through the binding
where ``own`` is true, else in elementary torch operations), ``work`` its
minimum bytes and operations, ``exact`` the result in 64 bits. Weights have the
benchmark's and the checkpoint's widths (5120 / 25600 and 6656 / 19968), heads
are theirs too (40 query / 8 kv heads of 128, 32 / 2).
"""
import math
import os
import random
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DEV = "cuda:0"
EPS = 1e-6
QK_SCALE = 3.87
THETA = 1e6
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}

own = False

_prims = None


def prims():
    """One context for the process, as a program keeps it."""
    global _prims
    if _prims is None:
        sys.path.insert(0, os.path.join(ROOT, "muse-glimmer-intel-serve_amd"))
        import mgprims
        _prims = mgprims.Prims(0)
    return _prims


def listed():
    return [
        # a projection's weight at load, and read back to check it: the largest of these
        {"name": "quant_weight", "kind": "quant", "rows": 25600, "in": 5120, "dtype": "bf16", "out": "bf16"},
        # the activations of one decode step of a batch
        {"name": "quant_acts_61", "kind": "quant", "rows": 61, "in": 19968, "dtype": "f16", "out": "f32"},
        # a projection at decode, one user
        {"name": "gemv_b1", "kind": "gemv", "rows": 25600, "in": 5120, "batch": 1, "dtype": "bf16", "out": "f32"},
        # the down projection for a batch of users
        {"name": "gemv_b48_f16", "kind": "gemv", "rows": 6656, "in": 19968, "batch": 48, "dtype": "f16", "out": "f16"},
        # the key projection of a few tokens to verify: latency
        {"name": "gemm_7", "kind": "gemm", "tokens": 7, "rows": 1024, "in": 5120, "out": "bf16"},
        # the down projection of a ragged prompt chunk, its result added up elsewhere in f32
        {"name": "gemm_333", "kind": "gemm", "tokens": 333, "rows": 5120, "in": 25600, "out": "f32"},
        # the up projection of a full prefill batch: the largest product
        {"name": "gemm_4096", "kind": "gemm", "tokens": 4096, "rows": 25600, "in": 5120, "out": "bf16"},
        # everything around RoPE of one decode step of a batch, padded for a captured graph
        {"name": "append_decode_61", "kind": "append", "tokens": 61, "pad": 3, "heads": 40, "kv": 8, "dim": 128,
         "page": 16, "dtype": "bf16", "most": 9000, "mix": 4},
        # the same of a prompt chunk
        {"name": "append_2000_f16", "kind": "append", "tokens": 2000, "pad": 0, "heads": 32, "kv": 2, "dim": 128,
         "page": 64, "dtype": "f16", "most": 20000, "mix": 5},
        # one user's token in an ordinary conversation: latency
        {"name": "decode_1x1500", "kind": "decode", "seqs": 1, "most": 1500, "ragged": False, "heads": 32, "kv": 2,
         "dim": 128, "page": 16, "dtype": "bf16", "out": "bf16", "window": 0, "mix": 7},
        # a batch of conversations of all lengths, an empty row among them
        {"name": "decode_64_ragged", "kind": "decode", "seqs": 64, "most": 8000, "ragged": True, "heads": 40, "kv": 8,
         "dim": 128, "page": 16, "dtype": "bf16", "out": "bf16", "window": 0, "mix": 8},
        # long documents
        {"name": "decode_5x100003", "kind": "decode", "seqs": 5, "most": 100003, "ragged": False, "heads": 32, "kv": 2,
         "dim": 128, "page": 64, "dtype": "bf16", "out": "bf16", "window": 0, "mix": 11},
    ]


def _log(rng, lo, hi):
    """An integer spread over the logarithm of [lo, hi]."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _weight(rng):
    """(rows, in) of a weight: the models' own widths, or any."""
    if rng.random() < 0.4:
        return rng.choice([(25600, 5120), (5120, 25600), (19968, 6656), (6656, 19968), (5120, 5120), (1024, 5120)])
    n = 32 * _log(rng, 2, 800)
    return _log(rng, 16, min(25600, 131072000 // n)), n


def draw(rng):
    kind = rng.choice(["quant", "gemv", "gemv", "gemm", "gemm", "append", "append", "decode", "decode", "decode"])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    if kind == "quant":
        rows, n = _weight(rng)
        return {"kind": kind, "rows": rows, "in": n, "dtype": rng.choice([dtype, dtype, "f32"]),
                "out": rng.choice([dtype, "f32"])}
    if kind == "gemv":
        rows, n = _weight(rng)
        return {"kind": kind, "rows": rows, "in": n, "batch": _log(rng, 1, 64), "dtype": dtype,
                "out": rng.choice([dtype, "f32"])}
    if kind == "gemm":
        rows, n = _weight(rng)
        return {"kind": kind, "tokens": _log(rng, 1, 4096), "rows": rows, "in": n, "out": rng.choice([dtype, "f32"])}
    mix, page, dim = rng.randrange(1 << 20), rng.choice([16, 32, 64, 128]), rng.choice([64, 128, 128])
    heads, kv = rng.choice([(40, 8), (32, 2)])
    if kind == "append":
        t = _log(rng, 1, 4096)
        return {"kind": kind, "tokens": t, "pad": rng.choice([0, 0, 5]), "heads": heads, "kv": kv, "dim": dim,
                "page": page, "dtype": dtype, "most": _log(rng, max(t, 64), 20000), "mix": mix}
    seqs = _log(rng, 1, 256)
    return {"kind": kind, "seqs": seqs, "most": _log(rng, 16, min(131072, 500000 // seqs)), "ragged": rng.random() < 0.7,
            "heads": heads, "kv": kv, "dim": dim, "page": page, "dtype": dtype, "out": rng.choice([dtype, dtype, "f32"]),
            "window": rng.choice([0, 0, 0, 1024]), "mix": mix}


def _seq_lens(c):
    """Key counts of a decode call."""
    rng, most = random.Random(c["mix"]), c["most"]
    if not c["ragged"]:
        return [most] * c["seqs"]
    lens = [rng.randint(1, most) for _ in range(c["seqs"])]
    if c["seqs"] > 8:
        lens[rng.randrange(c["seqs"])] = 0  # a padding row
    lens[rng.randrange(c["seqs"])] = most
    return lens


def _append_positions(c):
    """Runs of tokens of several requests, as a ragged batch holds them: (first position, tokens) of each."""
    rng, left, runs = random.Random(c["mix"]), c["tokens"], []
    while left:
        n = min(left, rng.choice([1, 1, 1, rng.randint(1, c["tokens"])]))
        runs.append((rng.randint(0, c["most"] - n) if c["most"] > n else 0, n))
        left -= n
    return runs


def _pages(n, page):
    return -(-n // page)


# ------------------------------------------------- the format, in plain steps
def _quantized(x):
    """MXFP4 codes and scales of x's rows: a block's scale is 2^(floor(log2 amax) - 2), a code the nearest of
    0 .5 1 1.5 2 3 4 6 (ties to the even code) with the sign in bit 3, past 6: 6."""
    b = x.float().unflatten(-1, (-1, 32))
    e = torch.frexp(b.abs().amax(-1, keepdim=True))[1] - 1
    amax0 = b.abs().amax(-1, keepdim=True) == 0
    s = torch.where(amax0, 0, (e - 2 + 127).clamp(0, 254))
    y = torch.ldexp(b, 127 - s)
    a = y.abs()
    code = torch.zeros_like(a, dtype=torch.uint8)
    for at, tie_up in ((0.25, False), (0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False)):
        code += (a >= at if tie_up else a > at).to(torch.uint8)
    code += torch.signbit(y).to(torch.uint8) * 8
    code = code.flatten(-2)
    return (code[..., 0::2] | (code[..., 1::2] << 4)).contiguous(), s.squeeze(-1).to(torch.uint8).contiguous()


_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)


def _values(qs, s):
    """What codes [.., n / 2] and scales [.., n / 32] stand for, in 32 bits."""
    lut = torch.tensor(_E2M1, dtype=torch.float32, device=qs.device)
    v = torch.stack((lut[(qs & 15).int()], lut[(qs >> 4).int()]), -1).flatten(-2)
    return torch.ldexp(v.unflatten(-1, (-1, 32)), s.int()[..., None] - 127).flatten(-2)


# ------------------------------------------------------------------- inputs
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(1_000_003 * (seed % 1_000_000_007) + 31)
    return g


def _randn(g, shape, dtype=torch.float32):
    return torch.randn(shape, generator=g, device=DEV, dtype=torch.float32).to(dtype)


def _i32(v):
    return torch.tensor(v, dtype=torch.int32).to(DEV)


def _i64(v):
    return torch.tensor(v, dtype=torch.int64).to(DEV)


def _acts(g, rows, n, dtype=torch.float32):
    """Activations: channels of different widths, rows of different sizes."""
    x = _randn(g, (rows, n)) * torch.exp(0.5 * _randn(g, (n,))) * torch.exp(0.3 * _randn(g, (rows, 1)))
    return x.to(dtype)


def _weights(g, rows, n):
    return _quantized((_randn(g, (rows, n)) / math.sqrt(n)).to(torch.bfloat16))


def _prepare_quant(c, g):
    n = c["in"]
    s = {"x": _acts(g, c["rows"], n, DTYPES[c["dtype"]])}
    s["qs"] = torch.empty((c["rows"], n // 2), dtype=torch.uint8, device=DEV)
    s["s"] = torch.empty((c["rows"], n // 32), dtype=torch.uint8, device=DEV)
    s["y"] = torch.empty((c["rows"], n), dtype=DTYPES[c["out"]], device=DEV)
    return s


def _prepare_gemv(c, g):
    s = {"x": _acts(g, c["batch"], c["in"], DTYPES[c["dtype"]])}
    s["qs"], s["s"] = _weights(g, c["rows"], c["in"])
    s["y"] = torch.empty((c["batch"], c["rows"]), dtype=DTYPES[c["out"]], device=DEV)
    return s


def _prepare_gemm(c, g):
    s = {}
    s["aq"], s["as"] = _quantized(_acts(g, c["tokens"], c["in"], torch.bfloat16))
    s["qs"], s["s"] = _weights(g, c["rows"], c["in"])
    s["y"] = torch.empty((c["tokens"], c["rows"]), dtype=DTYPES[c["out"]], device=DEV)
    return s


def _prepare_append(c, g):
    dt, T, hq, hk, D, ps = DTYPES[c["dtype"]], c["tokens"] + c["pad"], c["heads"], c["kv"], c["dim"], c["page"]
    s = {"q": _randn(g, (T, hq, D), dt), "k": _randn(g, (T, hk, D), dt), "v": _randn(g, (T, hk, D), dt)}
    runs = _append_positions(c)
    firsts = [(p // ps, _pages(p + n, ps) - p // ps) for p, n in runs]  # the pages a run writes
    pool = sum(n for _, n in firsts) + 16
    perm = torch.randperm(pool, generator=g, device=DEV)
    pos, page, at = [], [], 0
    for (p, n), (first, cnt) in zip(runs, firsts):
        pos += range(p, p + n)
        page += [at + j // ps - first for j in range(p, p + n)]
        at += cnt
    p = _i64(pos)
    s["pos"] = torch.cat((p, _i64([-1] * c["pad"])))
    s["slots"] = torch.cat((perm[_i64(page)] * ps + p % ps, _i64([-1] * c["pad"])))
    # the rotary table of every position, at the storage type (angles in 64 bits)
    inv = THETA ** (-torch.arange(0, D, 2, dtype=torch.float64, device=DEV) / D)
    ang = torch.arange(c["most"], dtype=torch.float64, device=DEV)[:, None] * inv
    s["cos"], s["sin"] = ang.cos().to(dt), ang.sin().to(dt)
    # the pool, with one more page behind it that the plain form lets unmapped tokens write
    for n in "kv":
        s[n + "all"] = torch.zeros((pool + 1, ps, hk, D // 2), dtype=torch.uint8, device=DEV)
        s[n + "dall"] = torch.zeros((pool + 1, ps, hk, D // 32), dtype=torch.uint8, device=DEV)
        s[n + "c"], s[n + "d"] = s[n + "all"][:pool], s[n + "dall"][:pool]
        s[n + "val"] = torch.zeros((pool, ps, hk, D), dtype=torch.float32, device=DEV)
    return s


def _prepare_decode(c, g):
    dt, hk, D, ps = DTYPES[c["dtype"]], c["kv"], c["dim"], c["page"]
    lens = _seq_lens(c)
    width = max(1, _pages(max(lens), ps))
    need = _i64([_pages(n, ps) for n in lens])
    pool = sum(_pages(n, ps) for n in lens) + 8
    # the pool's pages dealt to the requests in random order
    perm = torch.randperm(pool, generator=g, device=DEV).to(torch.int32)
    col = torch.arange(width, device=DEV)[None, :]
    off = (need.cumsum(0) - need)[:, None] + col
    table = torch.where(col < need[:, None], perm[off.clamp(max=pool - 1)], torch.full_like(off, -1, dtype=torch.int32))
    s = {"q": _randn(g, (c["seqs"], c["heads"], D), dt), "lens": _i32(lens), "table": table.contiguous()}
    for n in "kv":
        s[n + "c"], s[n + "d"] = _quantized(_randn(g, (pool, ps, hk, D), dt))
    s["o"] = torch.empty(s["q"].shape, dtype=DTYPES[c["out"]], device=DEV)
    return s


def _inputs(c, seed):
    return {"quant": _prepare_quant, "gemv": _prepare_gemv, "gemm": _prepare_gemm, "append": _prepare_append,
            "decode": _prepare_decode}[c["kind"]](c, _gen(seed))


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    s["scaling"] = 1.0 / math.sqrt(case.get("dim", 1))
    if own:
        s["P"] = prims()
    return s


# --------------------------------------------------------------- plain forms
def _plain_quant(s):
    s["qs"], s["s"] = _quantized(s["x"])
    s["y"].copy_(_values(s["qs"], s["s"]))


def _plain_gemv(s):
    s["y"].copy_(torch.matmul(s["x"].float(), _values(s["qs"], s["s"]).t()))


def _plain_gemm(s):
    s["y"].copy_(torch.matmul(_values(s["aq"], s["as"]), _values(s["qs"], s["s"]).t()))


def _plain_append(s):
    c = s["case"]
    dt, pos, slots = DTYPES[c["dtype"]], s["pos"], s["slots"]
    half, hk, D = c["dim"] // 2, c["kv"], c["dim"]

    # The operator is defined as the model's separate steps, each with its result stored at the storage type: the plain
    # form takes them one by one. The norm's sum runs in 64 bits: a value next to a border of two stored values goes by it.
    def stored(x):
        return x.float().to(dt).float()

    def normed(x):
        d = x.double()
        return stored(d * (1.0 / torch.sqrt((d * d).mean(-1, keepdim=True) + EPS)))

    turn = ((pos >= 0) & (pos < c["most"]))[:, None, None]
    row = pos.clamp(0, c["most"] - 1)
    cos, sin = s["cos"][row].float()[:, None, :], s["sin"][row].float()[:, None, :]

    def rotated(x):
        lo, hi = x[..., :half], x[..., half:]
        y = torch.cat((stored(lo * cos) + stored(-(hi * sin)), stored(hi * cos) + stored(lo * sin)), -1)
        return torch.where(turn, stored(y), x).to(dt)

    s["q"].copy_(rotated(stored(normed(s["q"]) * QK_SCALE)))
    s["k"].copy_(rotated(normed(s["k"])))
    at = torch.where(slots >= 0, slots, s["kc"].shape[0] * c["page"])
    for n in "kv":
        qs, d = _quantized(s[n])
        s[n + "all"].view(-1, hk, D // 2)[at] = qs
        s[n + "dall"].view(-1, hk, D // 32)[at] = d
        s[n + "val"].copy_(_values(s[n + "c"], s[n + "d"]))


def _plain_decode(s):
    c = s["case"]
    B, hk, g, D, ps = c["seqs"], c["kv"], c["heads"] // c["kv"], c["dim"], c["page"]
    page = s["table"].long().clamp(min=0)
    keys = page.shape[1] * ps

    def rows(n):  # every request's keys or values, [B, kv heads, keys, D]
        x = _values(s[n + "c"][page], s[n + "d"][page])
        return x.reshape(B, keys, hk, D).transpose(1, 2).contiguous()

    n = s["lens"].long()[:, None, None, None]
    j = torch.arange(keys, device=page.device)
    seen = j < n
    if c["window"]:
        seen = seen & (j >= n - c["window"])
    q = s["q"].float().reshape(B, hk, g, D)
    sc = (torch.matmul(q, rows("k").transpose(-1, -2).contiguous()) * s["scaling"]).masked_fill_(~seen, -math.inf)
    m = sc.amax(-1, keepdim=True)
    p = torch.where(seen, torch.exp(sc - m), 0.0)
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, rows("v")) / torch.where(total > 0, total, 1.0)
    s["o"].copy_(o.reshape(B, c["heads"], D))


# --------------------------------------------------------------------- pass
def run(s):
    kind, P = s["case"]["kind"], s.get("P")
    if kind == "quant":
        if own:
            P.quantize_mxfp4(s["x"], s["qs"], s["s"])
            P.dequant_mxfp4(s["qs"], s["s"], s["y"])  # the codes are returned as what they stand for
        else:
            _plain_quant(s)
        return s["y"]
    if kind == "gemv":
        if own:
            P.gemv_mxfp4(s["qs"], s["s"], s["x"], s["y"])
        else:
            _plain_gemv(s)
        return s["y"]
    if kind == "gemm":
        if own:
            P.gemm_mxfp4(s["aq"], s["as"], s["qs"], s["s"], s["y"])
        else:
            _plain_gemm(s)
        return s["y"]
    if kind == "append":
        if own:
            P.qk_norm_rope_paged(s["q"], s["k"], s["v"], EPS, QK_SCALE, s["cos"], s["sin"], s["pos"], s["slots"],
                                 s["kc"], s["vc"], s["kd"], s["vd"])
            for n in "kv":  # the pages' 4-bit values are read back as what they stand for
                D = s["case"]["dim"]
                P.dequant_mxfp4(s[n + "c"].view(-1, D // 2), s[n + "d"].view(-1, D // 32), s[n + "val"].view(-1, D))
        else:
            _plain_append(s)
        return s["q"], s["k"], s["kval"], s["vval"]
    if own:
        P.attn_decode_paged(s["q"], s["kc"], s["vc"], s["table"], s["lens"], s["scaling"], s["case"]["window"], s["kd"],
                            s["vd"], s["o"])
    else:
        _plain_decode(s)
    return s["o"]


# ------------------------------------------------------------------ measure
def _size(dtype):
    return 4 if dtype == "f32" else 2


def work(c):
    kind = c["kind"]
    if kind == "quant":
        # read, and what it stands for written: the codes between them are the pass's own
        n = c["rows"] * c["in"]
        return {"bytes": n * (_size(c["dtype"]) + _size(c["out"])) + n * 17 // 32, "flops": 0}
    if kind == "gemv":
        n, b = c["rows"] * c["in"], c["batch"]
        return {"bytes": n * 17 // 32 + 2 * b * c["in"] + _size(c["out"]) * b * c["rows"], "flops": 2 * b * n}
    if kind == "gemm":
        n, t = c["rows"] * c["in"], c["tokens"]
        return {"bytes": (n + t * c["in"]) * 17 // 32 + _size(c["out"]) * t * c["rows"], "flops": 2 * t * n}
    hq, hk, D = c["heads"], c["kv"], c["dim"]
    row = D * 17 // 32  # a head's row in the cache
    if kind == "append":
        T = c["tokens"] + c["pad"]
        pos = {p for first, n in _append_positions(c) for p in range(first, first + n)}
        q, k = T * hq * D, T * hk * D
        b = 2 * 2 * (q + k) + 2 * k + 2 * row * c["tokens"] * hk + 2 * D * len(pos) + 16 * T
        return {"bytes": b, "flops": 10 * (q + k)}
    lens = [min(n, c["window"]) if c["window"] else n for n in _seq_lens(c)]
    keys, table = sum(lens), sum(_pages(n, c["page"]) for n in lens)
    return {"bytes": 2 * row * keys * hk + (2 + _size(c["out"])) * c["seqs"] * hq * D + 4 * table + 4 * c["seqs"],
            "flops": 4 * D * hq * keys}


# ------------------------------------------------------------- 64-bit result
def _exact_rows(x):
    """What the quantizer keeps of rows x, from the distance to each value of the format."""
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64, device=DEV)
    out = torch.empty(x.shape, dtype=torch.float64, device=DEV)
    for at in range(0, x.shape[0], 512):
        b = x[at:at + 512].double().reshape(-1, 32)
        big = b.abs().max(1, keepdim=True).values
        step = torch.exp2((torch.floor(torch.log2(torch.where(big > 0, big, 1.0))) - 2.0).clamp(-127, 127))
        # log2 in 64 bits of a value just below a power of two may round up to it
        step = torch.where(big < 4.0 * step, step / 2, step)
        step = torch.where(big >= 8.0 * step, step * 2, step).clamp(min=2.0**-127)
        a = b.abs() / step
        best, val = torch.full_like(a, math.inf), torch.zeros_like(a)
        for i in (0, 2, 4, 6, 1, 3, 5, 7):  # even codes first: they win ties
            d = (a - grid[i]).abs()
            near = d < best
            best, val = torch.where(near, d, best), torch.where(near, grid[i], val)
        out[at:at + 512] = (val * step * b.sign()).reshape(-1, x.shape[1])
    return out


def _exact_values(qs, s):
    """Codes and scales, field by field: (-1)^sign 2^(exponent - 1) (1 + m / 2), or m / 2 where the exponent is 0."""
    v = torch.empty((*qs.shape[:-1], 2 * qs.shape[-1]), dtype=torch.float64, device=DEV)
    for i in range(2):
        c = (qs >> (4 * i)) & 15
        ex, m = ((c >> 1) & 3).double(), (c & 1).double()
        mag = torch.where(ex > 0, torch.exp2(ex - 1) * (1 + m / 2), m / 2)
        v[..., i::2] = torch.where(c >= 8, -mag, mag)
    return v * torch.exp2(s.double() - 127).repeat_interleave(32, -1)


def _exact_product(x, qs, s):
    """x [b, n] times every row of a weight, some rows at a time"""
    out = torch.empty((x.shape[0], qs.shape[0]), dtype=torch.float64, device=DEV)
    for at in range(0, qs.shape[0], 4096):
        out[:, at:at + 4096] = (_exact_values(qs[at:at + 4096], s[at:at + 4096]) @ x.t().contiguous()).t()
    return out


def _exact_append(c, s):
    dt, D = DTYPES[c["dtype"]], c["dim"]
    h = D // 2

    def at(x):  # a step's result as the operator defines it: a value of the storage type
        return x.to(torch.float32).to(dt).to(torch.float64)

    res = []
    for name, gain in (("q", QK_SCALE), ("k", None)):
        x = s[name].to(torch.float64)
        y = at(x / x.pow(2).mean(-1, keepdim=True).add(EPS).sqrt())
        if gain is not None:
            y = at(y * torch.tensor(gain, dtype=torch.float32, device=DEV).double())
        z = y.clone()
        live = s["pos"] >= 0
        co, si = (s[t].to(torch.float64)[s["pos"][live]].unsqueeze(1) for t in ("cos", "sin"))
        a, b = y[live][..., :h], y[live][..., h:]
        z[live] = at(torch.cat((at(a * co) - at(b * si), at(b * co) + at(a * si)), dim=-1))
        res.append(z)
    pool, ps, hk = s["kc"].shape[:3]
    live = s["slots"] >= 0
    caches = []
    for rows in (res[1], s["v"].to(torch.float64)):
        out = torch.zeros((pool * ps, hk, D), dtype=torch.float64, device=DEV)
        rows = rows[live]
        out[s["slots"][live]] = _exact_rows(rows.reshape(-1, D)).reshape(rows.shape)
        caches.append(out.view(pool, ps, hk, D))
    return (*res, *caches)


def _exact_decode(c, s):
    D, hk, ps = c["dim"], c["kv"], c["page"]
    g = c["heads"] // hk
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    for b, n in enumerate(_seq_lens(c)):
        lo = max(0, n - c["window"]) if c["window"] else 0
        if n <= lo:
            continue
        j = torch.arange(lo, n, device=DEV)
        slot = s["table"][b].long()[j // ps] * ps + j % ps
        k, v = (_exact_values(s[t + "c"].view(-1, hk, D // 2)[slot], s[t + "d"].view(-1, hk, D // 32)[slot]) for t in "kv")
        for h in range(hk):
            sc = (s["q"][b, h * g:(h + 1) * g].double() @ k[:, h].t().contiguous()) / math.sqrt(D)
            out[b, h * g:(h + 1) * g] = torch.softmax(sc, -1) @ v[:, h].contiguous()
    return out


def exact(case, seed):
    s = _inputs(case, seed)
    kind = case["kind"]
    if kind == "quant":
        return _exact_rows(s["x"])
    if kind == "gemv":
        return _exact_product(s["x"].double(), s["qs"], s["s"])
    if kind == "gemm":
        return _exact_product(_exact_values(s["aq"], s["as"]), s["qs"], s["s"])
    return _exact_append(case, s) if kind == "append" else _exact_decode(case, s)
