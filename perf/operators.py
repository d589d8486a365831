"""The paged KV cache's operators, as measurable cases.

A serving engine keeps the keys and values of many requests in one pool of
pages. Three operators keep and read it: ``kv_pages`` takes and gives back
pages as the requests' lengths change and maps their new tokens to slots,
``qk_norm_rope_paged`` runs the sequence around RoPE and appends through that
map, ``attn_decode_paged`` attends one new token per request over its pages.

``listed()`` names the cases, ``draw(rng)`` draws more of the same ranges;
``prepare`` makes a case's inputs, ``run`` is one pass (through the binding
where ``own`` is true, else in elementary torch operations), ``work`` its
minimum bytes and operations, ``exact`` the result in 64 bits. Head counts are
those of the benchmark (40 query / 8 kv heads of 128) and of the checkpoint
(32 / 2), request lengths run from one token to the benchmark's 131072.
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
        # one decode step of a small batch: every request one token longer, some into a new page
        {"name": "pages_decode_48", "kind": "pages", "requests": 48, "page": 16, "mode": "decode", "most": 9000, "mix": 1},
        # a step of continuous batching: most requests grow by a token, some finish, some start
        {"name": "pages_mixed_1000", "kind": "pages", "requests": 1000, "page": 16, "mode": "mixed", "most": 4000,
         "mix": 2},
        # admission of a wave of long prompts
        {"name": "pages_prompts_200", "kind": "pages", "requests": 200, "page": 32, "mode": "prompts", "most": 5000,
         "mix": 3},
        # everything around RoPE of one decode step of a batch, padded for a captured graph
        {"name": "append_decode_61", "kind": "append", "tokens": 61, "pad": 3, "heads": 40, "kv": 8, "dim": 128,
         "page": 16, "dtype": "bf16", "cache": "same", "most": 9000, "mix": 4},
        # the same of a prompt chunk into 8-bit pages
        {"name": "append_q8_2000", "kind": "append", "tokens": 2000, "pad": 0, "heads": 32, "kv": 2, "dim": 128,
         "page": 64, "dtype": "bf16", "cache": "q8_0", "most": 20000, "mix": 5},
        # a full prefill batch
        {"name": "append_4096_f16", "kind": "append", "tokens": 4096, "pad": 0, "heads": 40, "kv": 8, "dim": 128,
         "page": 16, "dtype": "f16", "cache": "same", "most": 4096, "mix": 6},
        # one user's token in an ordinary conversation: latency
        {"name": "decode_1x1500", "kind": "decode", "seqs": 1, "most": 1500, "ragged": False, "heads": 32, "kv": 2,
         "dim": 128, "page": 16, "dtype": "bf16", "cache": "same", "out": "bf16", "window": 0, "mix": 7},
        # a batch of conversations of all lengths, an empty row among them
        {"name": "decode_64_ragged", "kind": "decode", "seqs": 64, "most": 8000, "ragged": True, "heads": 40, "kv": 8,
         "dim": 128, "page": 16, "dtype": "bf16", "cache": "same", "out": "bf16", "window": 0, "mix": 8},
        # a large batch of short requests, the output in f32
        {"name": "decode_250_short", "kind": "decode", "seqs": 250, "most": 700, "ragged": True, "heads": 40, "kv": 8,
         "dim": 128, "page": 16, "dtype": "bf16", "cache": "same", "out": "f32", "window": 0, "mix": 9},
        # sliding-window layers of long requests
        {"name": "decode_window_f16", "kind": "decode", "seqs": 32, "most": 30000, "ragged": True, "heads": 40, "kv": 8,
         "dim": 64, "page": 32, "dtype": "f16", "cache": "same", "out": "f16", "window": 1024, "mix": 10},
        # long documents in 8-bit pages
        {"name": "decode_q8_5x100003", "kind": "decode", "seqs": 5, "most": 100003, "ragged": False, "heads": 32,
         "kv": 2, "dim": 128, "page": 64, "dtype": "bf16", "cache": "q8_0", "out": "bf16", "window": 0, "mix": 11},
        # the longest context for a batch: the largest call
        {"name": "decode_8x131072", "kind": "decode", "seqs": 8, "most": 131072, "ragged": False, "heads": 40, "kv": 8,
         "dim": 128, "page": 16, "dtype": "bf16", "cache": "same", "out": "bf16", "window": 0, "mix": 12},
    ]


def _log(rng, lo, hi):
    """An integer spread over the logarithm of [lo, hi]."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["pages", "append", "append", "decode", "decode", "decode"])
    mix = rng.randrange(1 << 20)
    page = rng.choice([16, 32, 64, 128])
    if kind == "pages":
        r = _log(rng, 1, 1000)
        return {"kind": kind, "requests": r, "page": page, "mode": rng.choice(["decode", "mixed", "prompts"]),
                "most": _log(rng, 20, min(131072, 1000000 // r)), "mix": mix}
    heads, kv = rng.choice([(40, 8), (32, 2)])
    dim, dtype, cache = rng.choice([64, 128, 128]), rng.choice(["bf16", "bf16", "f16"]), rng.choice(["same", "same", "q8_0"])
    if kind == "append":
        t = _log(rng, 1, 4096)
        return {"kind": kind, "tokens": t, "pad": rng.choice([0, 0, 5]), "heads": heads, "kv": kv, "dim": dim,
                "page": page, "dtype": dtype, "cache": cache, "most": _log(rng, max(t, 64), 20000), "mix": mix}
    seqs = _log(rng, 1, 256)
    return {"kind": kind, "seqs": seqs, "most": _log(rng, 16, min(131072, 800000 // seqs)), "ragged": rng.random() < 0.7,
            "heads": heads, "kv": kv, "dim": dim, "page": page, "dtype": dtype, "cache": cache,
            "out": rng.choice([dtype, dtype, "f32"]), "window": rng.choice([0, 0, 0, 1024]), "mix": mix}


# ---------------------------------------------------------- lengths of a case
def _old_new(c):
    """The request lengths before and after a step: the scheduler's, known with the case."""
    rng, r, most = random.Random(c["mix"]), c["requests"], c["most"]
    if c["mode"] == "prompts":
        return [0] * r, [rng.randint(1, most) for _ in range(r)]
    old = [rng.randint(1, most - 1) for _ in range(r)]
    new = [n + 1 for n in old]
    if c["mode"] == "mixed":
        for i in range(r):
            u = rng.random()
            if u < 0.05:  # finished
                new[i] = 0
            elif u < 0.1:  # started
                old[i], new[i] = 0, rng.randint(1, most)
            elif u < 0.13:  # rejected draft tokens rolled back
                new[i] = max(0, old[i] - rng.randint(1, 5))
            elif u < 0.15:  # an unused row of the batch
                old[i] = new[i] = 0
    return old, new


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


def _pages(n, page):
    return -(-n // page)


# ------------------------------------------------------------------- inputs
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(1_000_003 * (seed % 1_000_000_007) + 29)
    return g


def _randn(g, shape, dtype):
    return torch.randn(shape, generator=g, device=DEV, dtype=torch.float32).to(dtype)


def _i32(v):
    return torch.tensor(v, dtype=torch.int32).to(DEV)


def _i64(v):
    return torch.tensor(v, dtype=torch.int64).to(DEV)


def _table(g, lens, page, width, spare):
    """A pool's pages dealt to requests of the given lengths in random order: (table, the pages left, pool size)."""
    need = _i64([_pages(n, page) for n in lens])
    pool = int(sum(_pages(n, page) for n in lens)) + spare
    perm = torch.randperm(pool, generator=g, device=DEV).to(torch.int32)
    col = torch.arange(width, device=DEV)[None, :]
    off = (need.cumsum(0) - need)[:, None] + col
    table = torch.where(col < need[:, None], perm[off.clamp(max=pool - 1)], torch.full_like(off, -1, dtype=torch.int32))
    return table.contiguous(), perm[pool - spare:], pool


def _quantized(x):
    """Q8_0 quants and scales of x's rows, by 32 elements: d = amax / 127 in f32, stored as f16, q = x / d to the
    nearest whole number, halves away from zero."""
    b = x.float().unflatten(-1, (-1, 32))
    # (each step of the rule is one 32-bit rounding: quotients in 64 bits, then rounded)
    d = (b.abs().amax(-1, keepdim=True).double() / 127.0).float()
    y = b * torch.where(d != 0, 1.0 / d.double(), 0.0).float()
    q = torch.copysign((y.abs() + 0.5).floor(), y)
    return q.to(torch.int8).flatten(-2), d.squeeze(-1).half()


def _prepare_pages(c, g):
    old, new = _old_new(c)
    ps, r = c["page"], c["requests"]
    width = _pages(max(max(old), max(new)), ps) + 1
    takes = sum(max(0, _pages(n, ps) - _pages(o, ps)) for o, n in zip(old, new))
    table, left, pool = _table(g, old, ps, width, takes + 64)
    head = int(torch.randint(0, 4 * pool, (1,), generator=g, device=DEV))
    ring = torch.zeros(pool, dtype=torch.int32, device=DEV)
    ring[(head + torch.arange(left.numel(), device=DEV)) % pool] = left
    tokens = sum(max(0, n - o) for o, n in zip(old, new)) + 7  # the maps of a padded batch
    return {"table": table, "old": _i32(old), "new": _i32(new), "free": ring, "ends": _i64([head, head + left.numel()]),
            "lens": _i32([0] * r), "ends_out": _i64([0, 0]), "starts": _i32([0] * (r + 1)),
            "slots": _i64([0] * tokens), "pos": _i64([0] * tokens)}


def _append_positions(c):
    """Runs of tokens of several requests, as a ragged batch holds them: (request, position) of every token."""
    rng, left, runs = random.Random(c["mix"]), c["tokens"], []
    while left:
        n = min(left, rng.choice([1, 1, 1, rng.randint(1, c["tokens"])]))
        runs.append((rng.randint(0, c["most"] - n) if c["most"] > n else 0, n))
        left -= n
    return runs


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
    q8 = c["cache"] == "q8_0"
    # the pool, with one more page behind it that the plain form lets unmapped tokens write
    kv = [torch.zeros((pool + 1, ps, hk, D), dtype=torch.int8 if q8 else dt, device=DEV) for _ in range(2)]
    s["kall"], s["vall"] = kv
    s["kc"], s["vc"] = (t[:pool] for t in kv)
    s["kd"] = s["vd"] = s["kdall"] = s["vdall"] = None
    if q8:
        s["kdall"], s["vdall"] = (torch.zeros((pool + 1, ps, hk, D // 32), dtype=torch.float16, device=DEV)
                                  for _ in range(2))
        s["kd"], s["vd"] = s["kdall"][:pool], s["vdall"][:pool]
        s["kval"], s["vval"] = (torch.zeros((pool, ps, hk, D), dtype=torch.float32, device=DEV) for _ in range(2))
    return s


def _prepare_decode(c, g):
    dt, hk, D, ps = DTYPES[c["dtype"]], c["kv"], c["dim"], c["page"]
    lens = _seq_lens(c)
    width = max(1, _pages(max(lens), ps))
    table, _, pool = _table(g, lens, ps, width, 8)
    s = {"q": _randn(g, (c["seqs"], c["heads"], D), dt), "lens": _i32(lens), "table": table, "kd": None, "vd": None}
    for name in "kv":
        x = _randn(g, (pool, ps, hk, D), dt)
        if c["cache"] == "q8_0":
            x, s[name + "d"] = _quantized(x)
        s[name + "c"] = x
    s["o"] = torch.empty(s["q"].shape, dtype=DTYPES[c["out"]], device=DEV)
    return s


def _inputs(c, seed):
    return {"pages": _prepare_pages, "append": _prepare_append, "decode": _prepare_decode}[c["kind"]](c, _gen(seed))


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    s["scaling"] = 1.0 / math.sqrt(case.get("dim", 1))
    if own:
        s["P"] = prims()
    return s


# --------------------------------------------------------------- plain forms
def _plain_pages(s):
    ps, table, ring = s["case"]["page"], s["table"], s["free"]
    (R, W), N, T = table.shape, ring.numel(), s["slots"].numel()
    head, tail = s["ends"][0], s["ends"][1]
    o, n = s["old"].long().clamp(0, W * ps), s["new"].long().clamp(min=0)
    add = (n - o).clamp(min=0)
    ends = add.cumsum(0)
    starts = ends - add
    have, want = (o + ps - 1) // ps, (n + ps - 1) // ps
    fits = (n <= W * ps) & (ends <= T)
    grow = torch.where(fits, (want - have).clamp(min=0), 0)
    gend = grow.cumsum(0)
    ok = fits & ((grow == 0) | (gend <= (tail - head).clamp(0, N)))
    back = (have - want).clamp(min=0)
    bend = back.cumsum(0)
    # pages given back go behind the ring's tail, pages taken come from its head
    col = torch.arange(W, device=table.device)[None, :]
    gone = (col >= want[:, None]) & (col < have[:, None])
    to = torch.where(gone, (tail + (bend - back)[:, None] + col - want[:, None]) % N, N)
    longer = torch.cat((ring, ring[:1])).scatter_(0, to.flatten(), table.flatten())[:N]
    taken = ok[:, None] & (col >= have[:, None]) & (col < want[:, None])
    table.copy_(torch.where(taken, ring[(head + (gend - grow)[:, None] + col - have[:, None]) % N], table))
    ring.copy_(longer)
    s["lens"].copy_(torch.where(ok, n, o))
    s["ends_out"].copy_(torch.stack((head + torch.where(ok, grow, 0).sum(), tail + back.sum())))
    s["starts"].copy_(torch.cat((starts, ends[-1:])).clamp(max=T))
    t = torch.arange(T, device=table.device)
    i = torch.searchsorted(ends, t, right=True).clamp(max=R - 1)
    p = o[i] + t - starts[i]
    page = table[i, (p // ps).clamp(0, W - 1)].long()
    live = (t < ends[-1]) & ok[i]
    s["pos"].copy_(torch.where(live, p, -1))
    s["slots"].copy_(torch.where(live & (page >= 0) & (page < N), page * ps + p % ps, -1))


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
    if c["cache"] == "q8_0":
        for name in "kv":
            qs, d = _quantized(s[name])
            s[name + "all"].view(-1, hk, D)[at] = qs
            s[name + "dall"].view(-1, hk, D // 32)[at] = d
            s[name + "val"].copy_((s[name + "c"].float().unflatten(-1, (-1, 32)) * s[name + "d"].float()[..., None]).flatten(-2))
        return
    s["kall"].view(-1, hk, D)[at] = s["k"]
    s["vall"].view(-1, hk, D)[at] = s["v"]


def _plain_decode(s):
    c = s["case"]
    B, hk, g, D, ps = c["seqs"], c["kv"], c["heads"] // c["kv"], c["dim"], c["page"]
    page = s["table"].long().clamp(min=0)
    keys = page.shape[1] * ps

    def rows(name):  # every request's keys or values, [B, kv heads, keys, D]
        x = s[name + "c"][page].float()
        if c["cache"] == "q8_0":
            x = (x.unflatten(-1, (-1, 32)) * s[name + "d"][page].float()[..., None]).flatten(-2)
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
    c = s["case"]
    if c["kind"] == "pages":
        if own:
            s["P"].kv_pages(s["table"], s["old"], s["new"], c["page"], s["free"], s["ends"], s["lens"], s["ends_out"],
                            s["starts"], s["slots"], s["pos"])
        else:
            _plain_pages(s)
        return tuple(s[k] for k in ("table", "free", "lens", "ends_out", "starts", "slots", "pos"))
    if c["kind"] == "append":
        if own:
            s["P"].qk_norm_rope_paged(s["q"], s["k"], s["v"], EPS, QK_SCALE, s["cos"], s["sin"], s["pos"], s["slots"],
                                      s["kc"], s["vc"], s["kd"], s["vd"])
            if c["cache"] == "q8_0":  # the pages' 8-bit values are read back as what they stand for
                for name in "kv":
                    qs = s[name + "c"]
                    s["P"].dequant_q8_0(qs.view(-1, c["dim"]), s[name + "d"].view(-1, c["dim"] // 32),
                                        s[name + "val"].view(-1, c["dim"]))
        else:
            _plain_append(s)
        if c["cache"] == "q8_0":
            return s["q"], s["k"], s["kval"], s["vval"]
        return s["q"], s["k"], s["kc"], s["vc"]
    if own:
        s["P"].attn_decode_paged(s["q"], s["kc"], s["vc"], s["table"], s["lens"], s["scaling"], c["window"], s["kd"],
                                 s["vd"], s["o"])
    else:
        _plain_decode(s)
    return s["o"]


# ------------------------------------------------------------------ measure
def work(c):
    if c["kind"] == "pages":
        old, new = _old_new(c)
        ps, r = c["page"], c["requests"]
        tokens = sum(max(0, n - o) for o, n in zip(old, new)) + 7
        moved = sum(abs(_pages(n, ps) - _pages(o, ps)) for o, n in zip(old, new))
        kept = sum(n > o and o % ps != 0 for o, n in zip(old, new))  # new tokens in a page that was there
        return {"bytes": 8 * r + 4 * r + 4 * (r + 1) + 16 * tokens + 8 * moved + 4 * kept + 32, "flops": 0}
    hq, hk, D = c["heads"], c["kv"], c["dim"]
    row = D + D // 16 if c["cache"] == "q8_0" else 2 * D  # a head's row in the cache
    if c["kind"] == "append":
        T = c["tokens"] + c["pad"]
        pos = {p for first, n in _append_positions(c) for p in range(first, first + n)}
        q, k = T * hq * D, T * hk * D
        b = 2 * 2 * (q + k) + 2 * k + 2 * row * c["tokens"] * hk + 2 * D * len(pos) + 16 * T
        return {"bytes": b, "flops": 10 * (q + k)}
    lens = _seq_lens(c)
    keys = sum(min(n, c["window"]) if c["window"] else n for n in lens)
    table = sum(_pages(min(n, c["window"]) if c["window"] else n, c["page"]) for n in lens)
    out = 4 if c["out"] == "f32" else 2
    return {"bytes": 2 * row * keys * hk + (2 + out) * c["seqs"] * hq * D + 4 * table + 4 * c["seqs"],
            "flops": 4 * D * hq * keys}


# ------------------------------------------------------------- 64-bit result
def _exact_pages(c, s):
    """The step request by request, as a host's allocator takes it."""
    old, new = _old_new(c)
    ps = c["page"]
    table, ring = s["table"].cpu().tolist(), s["free"].cpu().tolist()
    head, tail = s["ends"].tolist()
    N, T, taken, lens, starts, slots, pos = len(ring), s["slots"].numel(), 0, [], [0], [], []
    avail = tail - head
    for i, (o, n) in enumerate(zip(old, new)):
        for j in range(_pages(n, ps), _pages(o, ps)):
            ring[tail % N] = table[i][j]
            tail += 1
        for j in range(_pages(o, ps), _pages(n, ps)):
            assert taken < avail
            table[i][j] = ring[head % N]
            head, taken = head + 1, taken + 1
        for p in range(o, n):
            pos.append(p)
            slots.append(table[i][p // ps] * ps + p % ps)
        lens.append(n)
        starts.append(len(pos))
    pad = [-1] * (T - len(pos))
    return (_i32(table), _i32(ring), _i32(lens), _i64([head, tail]), _i32(starts), _i64(slots + pad), _i64(pos + pad))


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
        rows = rows[live]
        if c["cache"] == "q8_0":
            # the rule is one of 32-bit steps: scale, its reciprocal and the product each rounded once
            blk = rows.reshape(-1, 32)
            d = (blk.abs().max(1, keepdim=True).values / 127.0).float()
            inv = torch.where(d == 0, 0.0, 1.0 / d.double()).float()
            t = (blk * inv.double()).float().double()
            rows = (t.sign() * (t.abs() + 0.5).floor() * d.half().double()).reshape(rows.shape)
        out = torch.zeros((pool * ps, hk, D), dtype=torch.float64, device=DEV)
        out[s["slots"][live]] = rows
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
        k, v = (s[t].view(-1, hk, D)[slot].double() for t in ("kc", "vc"))
        if c["cache"] == "q8_0":
            k, v = (x * s[t].view(-1, hk, D // 32)[slot].double().repeat_interleave(32, -1)
                    for x, t in ((k, "kd"), (v, "vd")))
        for h in range(hk):
            sc = (s["q"][b, h * g:(h + 1) * g].double() @ k[:, h].t().contiguous()) / math.sqrt(D)
            out[b, h * g:(h + 1) * g] = torch.softmax(sc, -1) @ v[:, h].contiguous()
    return out


def exact(case, seed):
    s = _inputs(case, seed)
    return {"pages": _exact_pages, "append": _exact_append, "decode": _exact_decode}[case["kind"]](case, s)
