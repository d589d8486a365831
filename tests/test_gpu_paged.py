"""GPU: the paged KV cache's operators against plain forms (tests/paged_oracle.py).

kv_pages is whole numbers: every output equal. qk_norm_rope_paged is bit for bit
qk_norm_rope (itself pinned to the twin by test_gpu_qk.py) with its rows where
the slot map says, Q8_0 pages by the quantizer's rule. attn_decode_paged is
gated on the bound counted in paged_oracle.attn_decode, plus half a step of a
16-bit output.
"""
import math

import numpy as np
import pytest

import oracle as O
import paged_oracle as PO
from util import BF16, F16, F32, from_dev, to_dev

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def i32(v):
    import torch
    return torch.tensor(np.asarray(v, np.int32), device=DEV)


def i64(v):
    import torch
    return torch.tensor(np.asarray(v, np.int64), device=DEV)


# ------------------------------------------------------------------ kv_pages
def pages_state(rng, R, W, ps, old, spare, head=0, owned=True):
    """a table that owns distinct pages for `old`, and the rest of the pool in the queue"""
    need = [PO.pages_of(min(max(o, 0), W * ps), ps) for o in old]
    N = sum(need) + spare
    perm = rng.permutation(N).tolist()
    table = np.full((R, W), -1, np.int32)
    for i, n in enumerate(need):
        table[i, :n] = [perm.pop() for _ in range(n)]
    ring = np.full(N, -7, np.int32)
    for k, p in enumerate(perm):
        ring[(head + k) % N] = p
    return table, ring, [head, head + len(perm)]


def run_pages(prims, table, old, new, ps, ring, ends, tokens, in_place=False, ldt=None):
    R, W = table.shape
    import torch
    ldt = ldt or W
    wide = torch.full((R, ldt), -99, dtype=torch.int32, device=DEV)
    t = wide[:, :W]
    t.copy_(i32(table))
    dold, dnew, dring, dends = i32(old), i32(new), i32(ring), i64(ends)
    lens = dold if in_place else i32([-5] * R)
    eout = dends if in_place else i64([-5, -5])
    starts, slots, pos = i32([-5] * (R + 1)), i64([-5] * tokens), i64([-5] * tokens)
    prims.kv_pages(t, dold, dnew, ps, dring, dends, lens, eout, starts, slots, pos)
    want = PO.kv_pages(table.tolist(), old, new, ps, ring.tolist(), ends, tokens)
    got = (t, dring, lens, eout, starts, slots, pos)
    for name, g, w in zip(("table", "ring", "lens", "ends", "starts", "slots", "pos"), got, want):
        assert np.array_equal(g.cpu().numpy(), np.asarray(w, g.cpu().numpy().dtype).reshape(tuple(g.shape))), name
    assert (wide[:, W:] == -99).all()
    return want


@pytest.mark.parametrize("R", (1, 5, 64, 1023, 1025, 4096))
@pytest.mark.parametrize("ps", (1, 16, 64))
def test_pages_mixed_steps(prims, R, ps):
    """growth by one and by prompts, finished requests, roll-backs and unused rows, a wrapped ring"""
    rng = np.random.default_rng(R * 100 + ps)
    W = 300 // ps + 2
    old = [int(x) for x in rng.integers(0, 290, R)]
    new = []
    for o in old:
        u = rng.random()
        new.append(o + 1 if u < 0.6 else 0 if u < 0.7 else max(0, o - int(rng.integers(0, 20))) if u < 0.8
                   else o if u < 0.9 else int(rng.integers(0, 301)))
    takes = sum(max(0, PO.pages_of(n, ps) - PO.pages_of(o, ps)) for o, n in zip(old, new))
    table, ring, ends = pages_state(rng, R, W, ps, old, takes + 9, head=10**12 + 3)
    tokens = sum(max(0, n - o) for o, n in zip(old, new))
    run_pages(prims, table, old, new, ps, ring, ends, tokens + 5, ldt=W + 3)
    run_pages(prims, table, old, new, ps, ring, ends, tokens, in_place=True)


def test_pages_refusals(prims):
    """too few pages (the one that does not fit and all behind it that need pages), a row too
    short, tokens past the maps (a shrinking request behind them still shrinks), and old
    lengths outside the row"""
    rng = np.random.default_rng(3)
    old = [16, 30, 0, 5, 40, 7, 64]
    new = [17, 33, 50, 6, 20, 8, 70]
    table, ring, ends = pages_state(rng, 7, 8, 16, old, 3)
    want = run_pages(prims, table, old, new, 16, ring, ends, 200)
    assert want[2] == [17, 33, 0, 6, 20, 8, 64]  # 1 + 1 pages of 3 taken, then 4 are asked for
    table, ring, ends = pages_state(rng, 7, 8, 16, old, 40)
    want = run_pages(prims, table, old, [17, 129, 50, 6, 20, 8, 128], 16, ring, ends, 60)
    assert want[2] == [17, 30, 0, 5, 20, 7, 64]
    want = run_pages(prims, table, [-3, 200, 128, 5, 0, 0, 0], [1, 128, 129, -7, 0, 0, 1], 16, ring, ends, 60)
    assert want[2] == [1, 128, 128, 0, 0, 0, 1]
    # an empty queue, a queue whose counters make no sense
    for e in ([4, 4], [9, 2], [-6, -1]):
        run_pages(prims, table, old, new, 16, ring, e, 200)


def test_pages_bad_table_entries(prims):
    """entries outside the pool give no slot"""
    rng = np.random.default_rng(4)
    table, ring, ends = pages_state(rng, 3, 4, 16, [20, 20, 20], 9)
    table[0, 1], table[1, 1], table[2, 1] = -1, len(ring), 2**31 - 1
    want = run_pages(prims, table, [20] * 3, [24, 40, 21], 16, ring, ends, 40)
    assert want[5][:4] == [-1] * 4 and want[5][16] >= 0


def test_pages_optional_outputs_and_no_requests(prims):
    import torch
    table, ring, ends = i32([[-1, -1]]), i32([3, 1, 0, 2]), i64([0, 4])
    lens, eo = i32([9]), i64([9, 9])
    prims.kv_pages(table, i32([0]), i32([17]), 16, ring, ends, lens, eo)  # no maps: 17 tokens do not fit 0
    assert lens.tolist() == [0] and eo.tolist() == [0, 4]
    pos = i64([5] * 20)
    prims.kv_pages(table, i32([0]), i32([17]), 16, ring, ends, lens, eo, positions=pos)
    assert lens.tolist() == [17] and eo.tolist() == [2, 4] and table.tolist() == [[3, 1]]
    assert pos.tolist() == list(range(17)) + [-1] * 3
    none = torch.empty((0, 4), dtype=torch.int32, device=DEV)
    starts, slots = i32([7]), i64([7, 7])
    prims.kv_pages(none, i32([]), i32([]), 16, ring, ends, i32([]), eo, starts, slots)
    assert starts.tolist() == [0] and slots.tolist() == [-1, -1] and eo.tolist() == [0, 4]


def test_pages_many_steps_keep_every_page(prims):
    """200 steps with the state in place: owned and free pages are the pool, none twice"""
    rng = np.random.default_rng(5)
    R, W, ps, N, T = 40, 20, 16, 300, 500
    table, ring = i32(np.full((R, W), -1)), i32(rng.permutation(N))
    lens, ends = i32([0] * R), i64([0, N])
    slots, pos = i64([0] * T), i64([0] * T)
    h = [0] * R
    state = ([[-1] * W for _ in range(R)], ring.tolist(), [0, N])
    for _ in range(200):
        new = [0 if rng.random() < 0.03 else min(W * ps, n + int(rng.choice([1, 1, 1, 30]))) for n in h]
        prims.kv_pages(table, lens, i32(new), ps, ring, ends, lens, ends, None, slots, pos)
        t, r, h2, e, _, sl, _ = PO.kv_pages(state[0], h, new, ps, state[1], state[2], T)
        state, h = (t, r, e), h2
        assert slots.tolist() == sl and lens.tolist() == h and ends.tolist() == e
    assert table.tolist() == state[0] and ring.tolist() == state[1]
    own = [p for row, n in zip(state[0], h) for p in row[:PO.pages_of(n, ps)]]
    free = [state[1][k % N] for k in range(*state[2])]
    assert sorted(own + free) == list(range(N))


def test_pages_errors(prims):
    table, ring, ends, lens = i32([[0, 0]] * 2), i32([0, 1]), i64([0, 2]), i32([0, 0])
    args = lambda **k: {**dict(page_table=table, old_lens=lens, new_lens=lens, page_size=16, free_ring=ring, ends=ends,
                               lens=lens, ends_out=ends), **k}
    prims.kv_pages(**args())
    for bad, match in ((dict(page_size=24), "power of two"), (dict(page_size=0), "power of two"),
                       (dict(page_size=1 << 21), "power of two"), (dict(new_lens=i32([0])), "int32"),
                       (dict(old_lens=i64([0, 0]).int().expand(2).to(DEV)[:1].expand(2)), "contiguous"),
                       (dict(ends=i32([0, 2])), "int64"), (dict(page_table=i32([[0, 0]])), "page_table"),
                       (dict(page_table=i32([[0, 0]]).expand(2, 2)), "overlap"), (dict(lens=lens.cpu()), "cpu"),
                       (dict(starts=i32([0, 0])), "int32"), (dict(slot_map=i32([0, 0])), "int64"),
                       (dict(slot_map=i64([0, 0]), positions=i64([0])), "int64")):
        with pytest.raises(Exception, match=match):
            prims.kv_pages(**args(**bad))
    many = i32(np.zeros((4097, 1)))
    l = i32(np.zeros(4097))
    with pytest.raises(Exception, match="4096 requests"):
        prims.kv_pages(**args(page_table=many, old_lens=l, new_lens=l, lens=l))
    with pytest.raises(Exception, match="2\\^30"):
        prims.kv_pages(**args(page_table=i32(np.zeros((2, 2048))), page_size=1 << 20))


# -------------------------------------------------------- qk_norm_rope_paged
def rows(seed, shape, dt):
    return to_dev(O.normal(seed, shape, 0.0, 1.0, dt), dt)


def rope_tables(T, D, dt):
    rc, rs = O.rope_table(1e6, D, T, dt)
    return to_dev(O.from_f64(rc, dt), dt), to_dev(O.from_f64(rs, dt), dt)


def q8_rule(x):
    """int8 quants and f16 scales of rows x (f32) by 32, one 32-bit rounding a step"""
    b = x.astype(np.float32).reshape(*x.shape[:-1], -1, 32)
    d = np.fmax.reduce(np.abs(b), axis=-1, keepdims=True) / np.float32(127)
    with np.errstate(divide="ignore", over="ignore", invalid="ignore"):
        y = b * np.where(d != 0, np.float32(1) / d, np.float32(0)).astype(np.float32)
        q = np.copysign(np.floor(np.abs(y) + np.float32(0.5)), y)
        return np.nan_to_num(q, nan=0.0).astype(np.int8).reshape(x.shape), d[..., 0].astype(np.float16)


def run_append(prims, dt, T, qh, kh, D, ps, q8, seed=7, pad=0, use_rope=True, offset=0):
    import torch
    rng = np.random.default_rng(seed)
    pos = rng.integers(0, 500, T)
    pos[T - pad:] = -1
    pages = T // ps + 3
    slot = rng.permutation(pages * ps)[:T].astype(np.int64)
    slot[T - pad:] = -1
    if T > 8:
        slot[3], slot[5] = pages * ps, -(2**40)  # outside the pool
        pos[4] = 10**6                           # outside the table
    # row strides wider than the rows
    base = [rows(seed + i, (T, (qh if i == 0 else kh) + 1, D), dt) for i in range(3)]
    q, k, v = base[0][:, offset:offset + qh], base[1][:, offset:offset + kh], base[2][:, :kh]
    eq, ek = q.clone(), k.clone()
    co, si = rope_tables(500, D, dt) if use_rope else (None, None)
    dpos, dslot = i64(pos), i64(slot)
    prims.qk_norm_rope(eq, ek, 1e-6, 3.87, co, si, dpos)
    if q8:
        kc, vc = (torch.full((pages, ps, kh, D), 77, dtype=torch.int8, device=DEV) for _ in range(2))
        kd, vd = (torch.full((pages, ps, kh, D // 32), 0.5, dtype=torch.float16, device=DEV) for _ in range(2))
    else:
        kc, vc = (torch.full((pages, ps, kh, D), 0.25, dtype=q.dtype, device=DEV) for _ in range(2))
        kd = vd = None
    want = [t.clone().view(-1, kh, t.shape[-1]) if t is not None else None for t in (kc, vc, kd, vd)]
    prims.qk_norm_rope_paged(q, k, v, 1e-6, 3.87, co, si, dpos, dslot, kc, vc, kd, vd)
    assert torch.equal(q.contiguous().view(torch.int16), eq.view(torch.int16))
    assert torch.equal(k.contiguous().view(torch.int16), ek.view(torch.int16))
    live = torch.from_numpy((slot >= 0) & (slot < pages * ps)).to(DEV)
    for c, d, x in ((0, 2, ek), (1, 3, v)):
        if q8:
            qs, sc = q8_rule(x.float().cpu().numpy())
            want[c][dslot[live]] = torch.from_numpy(qs).to(DEV)[live]
            want[d][dslot[live]] = torch.from_numpy(sc).to(DEV)[live]
        else:
            want[c][dslot[live]] = x[live]
    for g, w in zip((kc, vc, kd, vd), want):
        if g is not None:
            bits = torch.int8 if g.dtype == torch.int8 else torch.int16
            assert torch.equal(g.view(-1, kh, g.shape[-1]).view(bits), w.view(bits))


@pytest.mark.parametrize("dt", (BF16, F16))
@pytest.mark.parametrize("q8", (False, True))
@pytest.mark.parametrize("T,qh,kh,D,ps", ((1, 40, 8, 128, 16), (61, 32, 2, 128, 16), (130, 4, 1, 64, 32), (33, 3, 3, 256, 1)))
def test_append(prims, dt, q8, T, qh, kh, D, ps):
    run_append(prims, dt, T, qh, kh, D, ps, q8, pad=2 if T > 40 else 0)


@pytest.mark.parametrize("dt", (BF16, F16))
def test_append_other_head_dims_and_no_rope(prims, dt):
    """the general kernel: head_dim 18 and 80; no rotation"""
    run_append(prims, dt, 21, 4, 2, 18, 8, False)
    run_append(prims, dt, 21, 4, 2, 80, 8, False)
    run_append(prims, dt, 21, 4, 2, 128, 8, True, use_rope=False)


def test_append_specials(prims):
    """NaN, infinities and zero blocks of v in Q8_0 pages, by the rule; k's scale ties"""
    import torch
    v = torch.randn((2, 1, 128), generator=torch.Generator().manual_seed(3)).bfloat16()
    v[0, 0, 3], v[0, 0, 40] = float("nan"), float("inf")
    v[0, 0, 64:96] = 0.0
    v[0, 0, 96:] = torch.arange(32).bfloat16() - 0.5  # halves
    v[0, 0, 127] = 127.0
    v[1] = 3e38
    q, k = torch.ones((2, 1, 128), dtype=torch.bfloat16, device=DEV), torch.ones((2, 1, 128), dtype=torch.bfloat16, device=DEV)
    kc, vc = (torch.zeros((1, 2, 1, 128), dtype=torch.int8, device=DEV) for _ in range(2))
    kd, vd = (torch.zeros((1, 2, 1, 4), dtype=torch.float16, device=DEV) for _ in range(2))
    prims.qk_norm_rope_paged(q, k, v.to(DEV), 1e-6, 1.0, None, None, i64([0, 1]), i64([1, 0]), kc, vc, kd, vd)
    qs, sc = q8_rule(v.float().numpy())
    assert np.array_equal(vc[0].flip(0).cpu().numpy(), qs.reshape(2, 1, 128))
    assert np.array_equal(vd[0].flip(0).cpu().numpy().view(np.uint16), sc.reshape(2, 1, 4).view(np.uint16))


def test_append_errors(prims):
    import torch
    q, k = (torch.zeros((2, h, 128), dtype=torch.bfloat16, device=DEV) for h in (4, 2))
    kc = torch.zeros((3, 16, 2, 128), dtype=torch.bfloat16, device=DEV)
    p = i64([0, 1])
    args = lambda **kw: {**dict(q=q, k=k, v=k.clone(), eps=1e-6, qk_scale=1.0, cos=None, sin=None, positions=p,
                                slot_map=p, k_cache=kc, v_cache=kc.clone()), **kw}
    prims.qk_norm_rope_paged(**args())
    q8, sc = kc.to(torch.int8), torch.zeros((3, 16, 2, 4), dtype=torch.float16, device=DEV)
    f32 = torch.zeros((2, 4, 128), device=DEV)
    for bad, match in ((dict(slot_map=i32([0, 1])), "int64"), (dict(slot_map=i64([0])), "int64"),
                       (dict(k_cache=kc[:, :, :1].contiguous()), "caches must be"), (dict(v_cache=kc[:2]), "shape"),
                       (dict(k_cache=kc.half(), v_cache=kc.half()), "needed"), (dict(k_scale=sc), "both"),
                       (dict(k_cache=q8, v_cache=q8, k_scale=sc, v_scale=sc[..., :2].contiguous()), "scales"),
                       (dict(k_scale=sc, v_scale=sc), "needed"), (dict(k=k[:1]), "must be"),
                       (dict(q=f32, k=f32[:, :2], v=f32[:, :2], k_cache=kc.float(), v_cache=kc.float()), "bf16 or f16"),
                       (dict(q=q[:1].expand(2, 4, 128)), "overlap"),
                       (dict(v=k.clone().cpu()), "cpu")):
        with pytest.raises(Exception, match=match):
            prims.qk_norm_rope_paged(**args(**bad))
    small = lambda h: torch.zeros((2, h, 32), dtype=torch.bfloat16, device=DEV)
    with pytest.raises(Exception, match="head_dim 64, 128 or 256"):
        c = torch.zeros((1, 16, 2, 32), dtype=torch.int8, device=DEV)
        d = torch.zeros((1, 16, 2, 1), dtype=torch.float16, device=DEV)
        prims.qk_norm_rope_paged(small(4), small(2), small(2), 1e-6, 1.0, None, None, p, p, c, c.clone(), d, d.clone())


# --------------------------------------------------------- attn_decode_paged
def decode_case(prims, lens, nq, nkv, D, ps, dt=BF16, q8=False, out=None, window=0, seed=61, scaling=None, gap=0,
                poison=True, bad=None, ws=None):
    """a pool whose unused slots hold NaN (or quants with a NaN scale): only the requests' own keys may count"""
    import torch
    rng = np.random.default_rng(seed)
    R = len(lens)
    W = max(1, max(PO.pages_of(n, ps) for n in lens)) + 1
    need = sum(PO.pages_of(n, ps) for n in lens)
    N = need + 2
    perm = rng.permutation(N)
    table = rng.integers(-5, 2 * N, (R, W)).astype(np.int32)  # entries past a request's pages: anything
    used = np.zeros((N, ps), bool)
    at = 0
    for r, n in enumerate(lens):
        for i in range(PO.pages_of(n, ps)):
            table[r, i] = perm[at]
            used[perm[at], :min(ps, n - i * ps)] = True
            at += 1
    if bad:
        for r, i, page in bad:
            table[r, i] = page
    qb = O.normal(seed, (R, nq, D), 0.0, 1.0, dt)
    fill = []
    for s in (1, 2):
        x = rng.standard_normal((N, ps, nkv, D)).astype(np.float32)
        if q8:
            qs, d = q8_rule(x)
            vals = qs.astype(np.float64).reshape(N, ps, nkv, -1, 32) * d.astype(np.float64)[..., None]
            if poison:
                d[~used] = np.nan
            fill.append((torch.from_numpy(qs).to(DEV), torch.from_numpy(d).to(DEV), vals.reshape(x.shape)))
        else:
            b = O.from_f64(x.astype(np.float64), dt)
            vals = O.to_f64(b, dt)
            if poison:
                b[~used] = 0x7fc0 if dt == BF16 else 0x7e00
            fill.append((to_dev(b, dt), None, vals))
    (kc, kd, K), (vc, vd, V) = fill
    scaling = 1.0 / math.sqrt(D) if scaling is None else scaling
    dq = to_dev(qb, dt)
    od = {None: torch.float32, "same": dq.dtype}[out]
    wide = torch.full((R + 1, nq + gap, D), 7.5, dtype=od, device=DEV)
    o = wide[:R, :nq]
    wt = torch.full((R, W + gap), 5, dtype=torch.int32, device=DEV)
    wt[:, :W] = i32(table)
    (ws or prims).attn_decode_paged(dq, kc, vc, wt[:, :W], i32(lens), scaling, window, kd, vd, o)
    assert (wide[R:] == 7.5).all() and (wide[:, nq:] == 7.5).all()
    ref, bound = PO.attn_decode(O.to_f64(qb, dt), K, V, table, lens, ps, window, scaling)
    got = o.double().cpu().numpy()
    if out == "same":
        bound = bound + np.abs(ref) * (2.0**-8 if dt == BF16 else 2.0**-11) + 2.0**-24
    err = np.abs(got - ref)
    assert np.all(err <= bound * 1.0000001 + 1e-30), (float(err.max()), np.argwhere(~(err <= bound))[:4].tolist())
    return got


FORMS = ((BF16, False), (F16, False), (BF16, True), (F16, True))


@pytest.mark.parametrize("dt,q8", FORMS)
@pytest.mark.parametrize("D", (64, 128))
@pytest.mark.parametrize("ps", (1, 16, 64))
def test_decode_ragged(prims, dt, q8, D, ps):
    """lengths from none to many, at the edges of pages and of the tiles"""
    decode_case(prims, [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 500, 0, 1025], 10, 2, D, ps, dt, q8)


@pytest.mark.parametrize("dt,q8", FORMS)
@pytest.mark.parametrize("nq,nkv", ((1, 1), (7, 7), (40, 8), (32, 2), (9, 1), (20, 1), (64, 2)))
def test_decode_heads(prims, dt, q8, nq, nkv):
    """group sizes of 1 to 32 heads, in strided tensors, the output at q's dtype"""
    decode_case(prims, [70, 0, 333], nq, nkv, 128, 16, dt, q8, out="same", gap=2, seed=nq)


@pytest.mark.parametrize("dt,q8", FORMS)
@pytest.mark.parametrize("window", (1, 20, 128, 1000))
def test_decode_window(prims, dt, q8, window):
    decode_case(prims, [0, 1, 19, 20, 21, 300, 1500, 999, 1000, 1001], 10, 2, 64, 16, dt, q8, window=window)


@pytest.mark.parametrize("dt,q8", FORMS)
def test_decode_long(prims, dt, q8):
    """one long request, split over many work-groups, next to short ones; one alone"""
    decode_case(prims, [20011, 3, 0, 4096], 32, 2, 128, 16, dt, q8)
    decode_case(prims, [9001], 5, 1, 64, 128, dt, q8)


@pytest.mark.parametrize("dt,q8", FORMS)
def test_decode_many_parts(prims, dt, q8):
    """requests of hundreds of partial results: alone, next to few short ones, next to many"""
    decode_case(prims, [40000], 8, 1, 128, 16, dt, q8)
    decode_case(prims, [100000], 2, 1, 64, 64, dt, q8, out="same")
    decode_case(prims, [30000, 5, 0], 4, 1, 128, 32, dt, q8)
    decode_case(prims, [9] * 40 + [30000] + [7] * 60, 3, 1, 64, 16, dt, q8)


def test_decode_many_short(prims):
    """more requests than work-groups, all short"""
    rng = np.random.default_rng(8)
    decode_case(prims, rng.integers(0, 40, 1500).tolist(), 2, 1, 64, 8)
    decode_case(prims, [1] * 700, 8, 8, 64, 1)
    decode_case(prims, [0] * 33, 8, 2, 64, 16)


@pytest.mark.parametrize("dt,q8", FORMS)
def test_decode_peaked(prims, dt, q8):
    """scaling 1: scores over tens of units, late maxima"""
    decode_case(prims, [700, 65, 2000], 10, 2, 128, 16, dt, q8, scaling=1.0)


@pytest.mark.parametrize("dt,q8", FORMS)
def test_decode_bad_pages(prims, dt, q8):
    """pages outside the pool are left out, a request of only such pages gives zeros"""
    bad = [(0, 0, -1), (1, 3, 10**6), (2, 0, -2**31), (2, 1, 2**31 - 1), (3, 2, -1)]
    got = decode_case(prims, [40, 200, 32, 48, 0], 4, 2, 64, 16, dt, q8, bad=bad)
    assert not got[2].any()


@pytest.mark.parametrize("q8", (False, True))
def test_decode_nan_and_inf_keys(prims, q8):
    """a NaN key reaches its request's heads of that kv head and no other; a key of score -inf weighs nothing"""
    import torch
    R, n, nkv, D, ps = 3, 300, 2, 128, 16
    q = torch.rand((R, 4, D), device=DEV).add_(0.25).bfloat16()
    table = i32(np.arange(R * 19).reshape(R, 19))
    lens = i32([n] * R)
    kf = torch.randn((R * 19, ps, nkv, D), device=DEV)
    if q8:
        kc, vc = (torch.randint(-127, 128, kf.shape, device=DEV, dtype=torch.int8) for _ in range(2))
        kd, vd = (torch.full((*kf.shape[:3], 4), 0.01, dtype=torch.float16, device=DEV) for _ in range(2))
    else:
        kc, vc, kd, vd = kf.bfloat16(), torch.randn_like(kf).bfloat16(), None, None
    run = lambda: prims.attn_decode_paged(q, kc, vc, table, lens, 0.088, 0, kd, vd)
    base = run()
    assert torch.isfinite(base).all()
    page, off = 19 + (n - 1) // ps, (n - 1) % ps  # request 1's newest key
    (kd if q8 else kc)[page, off, 1, 2] = float("nan")
    got = run()
    assert torch.isnan(got[1, 2:]).all()
    got[1, 2:] = base[1, 2:]
    assert torch.equal(got, base)
    if not q8:
        kc[page, off, 1, 2] = -float("inf")  # q > 0: score -inf
        got = run()
        m = lens.clone()
        m[1] = n - 1
        assert torch.allclose(got[1, 2:], prims.attn_decode_paged(q, kc, vc, table, m, 0.088)[1, 2:], rtol=0, atol=1e-4)


def test_decode_far_pages(prims):
    """a pool of more than 2^31 elements a cache: offsets past 32 bits, lengths in its last pages"""
    import torch
    nkv, D, ps = 8, 128, 64
    N = (2**31 // (nkv * D * ps)) + 70
    kc, vc = (torch.empty((N, ps, nkv, D), dtype=torch.bfloat16, device=DEV) for _ in range(2))
    g = torch.Generator(device=DEV).manual_seed(5)
    for c in (kc, vc):
        c[-60:] = torch.randn((60, ps, nkv, D), generator=g, device=DEV).bfloat16()
    table = np.stack([np.arange(N - 60, N - 30), np.arange(N - 1, N - 31, -1)]).astype(np.int32)
    lens = [1900, 1777]
    q = torch.randn((2, 16, D), generator=g, device=DEV).bfloat16()
    got = prims.attn_decode_paged(q, kc, vc, i32(table), i32(lens), 0.088).double().cpu().numpy()
    K, V = (c[-60:].double().cpu().numpy() for c in (kc, vc))
    ref, bound = PO.attn_decode(q.double().cpu().numpy(), K, V, table - (N - 60), lens, ps, 0, 0.088)
    assert np.all(np.abs(got - ref) <= bound)
    # the append writes there too
    k = torch.randn((1, nkv, D), generator=g, device=DEV).bfloat16()
    slot = N * ps - 1
    prims.qk_norm_rope_paged(q[:1], k, k.clone(), 1e-6, 1.0, None, None, i64([0]), i64([slot]), kc, vc)
    assert torch.equal(kc[-1, -1], k[0])


def test_decode_empty_call_and_errors(prims):
    import torch
    q = torch.zeros((2, 8, 128), dtype=torch.bfloat16, device=DEV)
    kc = torch.zeros((4, 16, 2, 128), dtype=torch.bfloat16, device=DEV)
    t, n = i32([[0, 1]] * 2), i32([3, 4])
    args = lambda **kw: {**dict(q=q, k_cache=kc, v_cache=kc, page_table=t, lens=n, scaling=0.1), **kw}
    prims.attn_decode_paged(**args())
    assert prims.attn_decode_paged(q[:0], kc, kc, t[:0], n[:0], 0.1).shape == (0, 8, 128)
    sc = torch.zeros((4, 16, 2, 4), dtype=torch.float16, device=DEV)
    for bad, match in ((dict(q=q[:, :7]), "multiple"), (dict(q=q.half()), "needed"), (dict(q=q.float()), "needed"),
                       (dict(lens=i32([1])), "int32"), (dict(lens=i64([1, 1])), "int32"),
                       (dict(page_table=t[:1]), "page_table"), (dict(page_table=t.t()), "page_table rows"),
                       (dict(k_cache=kc[:, :12].contiguous(), v_cache=kc[:, :12].contiguous()), "power of two"),
                       (dict(v_cache=kc[:2]), "shape"), (dict(k_scale=sc), "both"),
                       (dict(out=torch.zeros((2, 8, 64), device=DEV)), "shape"),
                       (dict(out=torch.zeros((2, 8, 128), dtype=torch.float16, device=DEV)), "dtype_out"),
                       (dict(q=q[:1].expand(2, 8, 128)), "overlap"),
                       (dict(q=torch.zeros(2 * 8 * 128 + 1, dtype=torch.bfloat16, device=DEV)[1:].view(2, 8, 128)), "aligned"),
                       (dict(page_table=t.cpu()), "cpu")):
        with pytest.raises(Exception, match=match):
            prims.attn_decode_paged(**args(**bad))
    small = torch.zeros((2, 8, 32), dtype=torch.bfloat16, device=DEV)
    with pytest.raises(Exception, match="head_dim"):
        prims.attn_decode_paged(small, kc[..., :32].contiguous(), kc[..., :32].contiguous(), t, n, 0.1)


# ------------------------------------------------------- a run of them together
class Engine:
    """a tiny serving loop over the three operators, its state in device memory"""

    def __init__(self, prims, R, W, ps, N, q8, dt, T, nq=10, nkv=2, D=128):
        import torch
        self.p, self.ps, self.dt, self.T = prims, ps, dt, T
        self.table, self.ring = i32(np.full((R, W), -1)), i32(np.arange(N)[::-1].copy())
        self.lens, self.ends, self.new = i32([0] * R), i64([0, N]), i32([0] * R)
        self.starts, self.slots, self.pos = i32([0] * (R + 1)), i64([0] * T), i64([0] * T)
        tdt = {BF16: torch.bfloat16, F16: torch.float16}[dt]
        z = lambda *s, d=tdt: torch.zeros(s, dtype=d, device=DEV)
        self.q, self.k, self.v = z(T, nq, D), z(T, nkv, D), z(T, nkv, D)
        cd = torch.int8 if q8 else tdt
        self.kc, self.vc = z(N, ps, nkv, D, d=cd), z(N, ps, nkv, D, d=cd)
        self.kd, self.vd = (z(N, ps, nkv, D // 32, d=torch.float16) for _ in range(2)) if q8 else (None, None)
        self.co, self.si = rope_tables(W * ps, D, dt)
        self.out = z(R, nq, D, d=torch.float32)

    def step(self):
        """decode: request r's new token is row r of q, k and v"""
        p = self.p
        p.kv_pages(self.table, self.lens, self.new, self.ps, self.ring, self.ends, self.lens, self.ends, self.starts,
                   self.slots, self.pos)
        p.qk_norm_rope_paged(self.q, self.k, self.v, 1e-6, 3.87, self.co, self.si, self.pos, self.slots, self.kc,
                             self.vc, self.kd, self.vd)

    def attend(self):
        self.p.attn_decode_paged(self.q, self.kc, self.vc, self.table, self.lens, 0.088, 0, self.kd, self.vd, self.out)


def feed(e, seed):
    import torch
    g = torch.Generator(device=DEV).manual_seed(seed)
    for t in (e.q, e.k, e.v):
        t.copy_(torch.randn(t.shape, generator=g, device=DEV))


@pytest.mark.parametrize("dt,q8", FORMS)
def test_prompts_then_decode(prims, dt, q8):
    """prompts of ragged lengths appended in one call, then decode steps: each step's attention
    equals 64-bit attention over the keys that the ring form of the sequence gives"""
    import torch
    R, ps = 6, 16
    prompt = [5, 0, 33, 16, 70, 1]
    T = sum(prompt)
    e = Engine(prims, R, 8, ps, 60, q8, dt, T)
    keys = [[] for _ in range(R)]  # (k, v) rows as stored, per request

    def record(owner_of_token):
        k, v = (x.float().cpu().numpy() for x in (e.k, e.v))
        for t, r in enumerate(owner_of_token):
            rows_ = (k[t], v[t])
            if q8:
                rows_ = tuple((lambda qs, d: qs.astype(np.float64).reshape(2, -1, 32) * d.astype(np.float64)[..., None])(
                    *q8_rule(x)).reshape(2, 128) for x in rows_)
            keys[r].append(rows_)

    feed(e, 1)
    e.new.copy_(i32(prompt))
    e.step()
    assert e.lens.tolist() == prompt
    record([r for r in range(R) for _ in range(prompt[r])])
    d = Engine(prims, R, 8, ps, 60, q8, dt, R)
    for name in ("table", "ring", "lens", "ends", "kc", "vc", "kd", "vd"):
        setattr(d, name, getattr(e, name))
    e = d
    for i in range(12):
        feed(e, 10 + i)
        e.new.copy_(e.lens + 1)
        e.step()
        e.attend()
        record(range(R))
        q = e.q.double().cpu().numpy()
        for r in range(R):
            K, V = (np.stack([x[c] for x in keys[r]]).astype(np.float64)[:, None] for c in (0, 1))
            ref, bound = PO.attn_decode(q[r:r + 1], K, V, np.arange(len(keys[r]))[None], [len(keys[r])], 1, 0, 0.088)
            assert np.all(np.abs(e.out[r].double().cpu().numpy() - ref[0]) <= bound[0]), (i, r)


def test_decode_equals_ring_attention(prims):
    """the same keys in a ring: attn_decode and attn_decode_paged agree within both bounds"""
    import torch
    n, nq, nkv, D, ps = 777, 40, 8, 128, 16
    kc, vc = (rows(s, (49 * ps, nkv, D), BF16) for s in (1, 2))
    q = rows(3, (1, nq, D), BF16)
    a = prims.attn_decode(q[0], kc, vc, n - 1, 0.088)
    b = prims.attn_decode_paged(q, kc.view(49, ps, nkv, D), vc.view(49, ps, nkv, D), i32([range(49)]), i32([n]), 0.088)
    K, V = (c.view(49, ps, nkv, D).double().cpu().numpy() for c in (kc, vc))
    _, bound = PO.attn_decode(q.double().cpu().numpy(), K, V, np.arange(49)[None], [n], ps, 0, 0.088)
    assert np.all((a - b[0]).abs().double().cpu().numpy() <= 2 * bound[0])


@pytest.mark.parametrize("q8", (False, True))
def test_captured_decode_loop(prims, q8):
    """a decode step captured once and replayed, with eager work between the replays: every
    replay equals the eager loop, pages and all"""
    import torch
    import mgprims
    R, ps = 7, 16
    side = torch.cuda.Stream()
    p = mgprims.Prims(0, stream=side.cuda_stream)
    e, ref = Engine(p, R, 6, ps, 50, q8, BF16, R), Engine(prims, R, 6, ps, 50, q8, BF16, R)
    for x in (e, ref):
        x.new.copy_(i32([1, 0, 1, 1, 1, 0, 1]))
    torch.cuda.synchronize()

    def step(x):
        x.step()
        x.attend()
        x.new.copy_(x.lens + (x.lens > 0))

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step(e)
    for i in range(40):
        for x in (e, ref):
            feed(x, 100 + i)
        if i == 20:  # a request ends, another begins
            for x in (e, ref):
                x.new[2], x.new[5] = 0, 1
        torch.cuda.synchronize()
        graph.replay()
        step(ref)
        (torch.ones(1000, device=DEV) * 2).sum().item()
        torch.cuda.synchronize()
        for name in ("table", "ring", "lens", "ends", "slots", "pos", "q", "kc", "vc", "out"):
            assert torch.equal(getattr(e, name), getattr(ref, name)), (i, name)
    assert ref.lens.tolist() == [40, 0, 0, 40, 40, 20, 40]
    p.close()


def test_other_stream_and_current_device(prims):
    """a context on a side stream, its tensors made there"""
    import torch
    import mgprims
    side = torch.cuda.Stream()
    p = mgprims.Prims(0, stream=side.cuda_stream)
    with torch.cuda.stream(side):
        a = decode_case(p, [100, 0, 2000], 10, 2, 128, 16)
    b = decode_case(prims, [100, 0, 2000], 10, 2, 128, 16)
    assert np.array_equal(a, b)
    p.close()


# -------------------------------------------------- paths by batch and workspace
@pytest.mark.parametrize("dt,q8", FORMS)
def test_decode_more_than_64_requests(prims, dt, q8):
    """lengths summed by the whole work-group, runs that begin and end inside requests, a join note a team"""
    rng = np.random.default_rng(11)
    lens = rng.integers(0, 900, 100).tolist()
    lens[7] = lens[99] = 0
    decode_case(prims, lens, 16, 8, 64, 16, dt, q8, out="same")


@pytest.mark.parametrize("R", (63, 64, 65, 257))
def test_decode_request_counts(prims, R):
    """at the limits of a wave's and of a work-group's requests, the first and last ones long"""
    lens = [1000] + [3] * (R - 2) + [777]
    decode_case(prims, lens, 4, 2, 64, 16, window=0)


def test_decode_small_workspaces(prims):
    """room for a few teams, for one (nothing is cut), for none of it"""
    import mgprims
    for size in (64, 40000, 200000):
        p = mgprims.Prims(0, workspace_bytes=size)
        decode_case(p, [3000, 5, 0, 900], 10, 2, 128, 16, ws=p)
        decode_case(p, [200] * 90, 10, 2, 64, 16, q8=True, ws=p)
        p.close()


def test_pages_small_workspace(prims):
    """a large step needs no room in the workspace"""
    import mgprims
    rng = np.random.default_rng(12)
    p = mgprims.Prims(0, workspace_bytes=64)
    old = [0] * 90
    new = [int(x) for x in rng.integers(0, 200, 90)]
    table, ring, ends = pages_state(rng, 90, 14, 16, old, 90 * 14)
    assert sum(new) > 4096
    run_pages(p, table, old, new, 16, ring, ends, sum(new) + 3)
    run_pages(prims, table, old, new, 16, ring, ends, sum(new) + 3, in_place=True)
    # too few pages and maps that end early
    run_pages(prims, table, old, new, 16, ring, [ends[0], ends[0] + 200], sum(new))
    run_pages(prims, table, old, new, 16, ring, ends, 5000)
    p.close()


@pytest.mark.parametrize("R", (1, 63, 200, 1024, 1030, 4096))
@pytest.mark.parametrize("tokens", (1024, 1025, 4096, 4097, 9001))
def test_pages_step_sizes(prims, R, tokens):
    """around the sizes where a step takes more work-groups or, in place, two launches: maps with room to spare,
    maps that end early (requests behind the end only shrink) and too few pages"""
    rng = np.random.default_rng(R + tokens)
    ps, most = 16, 2 * tokens // R + 2
    W = (most + 40) // ps + 2
    old = [int(x) for x in rng.integers(0, 40, R)]
    new = [o + int(x) if rng.random() < 0.8 else int(x) // 4 for o, x in zip(old, rng.integers(0, most, R))]
    takes = sum(max(0, PO.pages_of(n, ps) - PO.pages_of(o, ps)) for o, n in zip(old, new))
    table, ring, ends = pages_state(rng, R, W, ps, old, takes + 3, head=7)
    for in_place in (False, True):
        for t, e in ((max(tokens, sum(max(0, n - o) for o, n in zip(old, new))), ends), (tokens, ends),
                     (tokens, [ends[0], ends[0] + takes // 2])):
            run_pages(prims, table, old, new, ps, ring, e, t, in_place=in_place)


@pytest.mark.parametrize("tokens", (700, 6000))
@pytest.mark.parametrize("lens_is,ends_in_place", (("new", False), ("new", True), ("apart", True), ("old", False)))
def test_pages_what_is_in_place(prims, tokens, lens_is, ends_in_place):
    """each of the outputs that may replace its input, alone and together"""
    rng = np.random.default_rng(tokens)
    R, ps = 60, 16
    old = [int(x) for x in rng.integers(0, 40, R)]
    new = [o + tokens // R if i % 5 else 0 for i, o in enumerate(old)]
    W = max(new) // ps + 2
    table, ring, ends = pages_state(rng, R, W, ps, old, R * W, head=3)
    t, dold, dnew, dring, dends = i32(table), i32(old), i32(new), i32(ring), i64(ends)
    lens = {"new": dnew, "old": dold, "apart": i32([-5] * R)}[lens_is]
    eout = dends if ends_in_place else i64([-5, -5])
    starts, slots, pos = i32([-5] * (R + 1)), i64([-5] * tokens), i64([-5] * tokens)
    prims.kv_pages(t, dold, dnew, ps, dring, dends, lens, eout, starts, slots, pos)
    want = PO.kv_pages(table.tolist(), old, new, ps, ring.tolist(), ends, tokens)
    for g, w in zip((t, dring, lens, eout, starts, slots, pos), want):
        assert np.array_equal(g.cpu().numpy(), np.asarray(w).reshape(tuple(g.shape)))


@pytest.mark.parametrize("q8", (False, True))
def test_append_many_tokens(prims, q8):
    """many work-groups, q's rows and k's, a wave of both kinds"""
    run_append(prims, BF16, 701, 5, 3, 128, 16, q8, pad=3)
    run_append(prims, F16, 701, 40, 8, 64, 64, q8, pad=3)


def test_two_contexts_at_once(prims):
    """two contexts on two streams, their calls interleaved"""
    import torch
    import mgprims
    streams = [torch.cuda.Stream() for _ in range(2)]
    ps = [mgprims.Prims(0, stream=s.cuda_stream) for s in streams]
    g = torch.Generator(device=DEV).manual_seed(9)
    kc, vc = (torch.randn((400, 16, 2, 128), generator=g, device=DEV).bfloat16() for _ in range(2))
    sets = []
    for i, lens in enumerate(([3000, 40, 0, 900], [17] * 20 + [2500])):
        R = len(lens)
        q = torch.randn((R, 32, 128), generator=g, device=DEV).bfloat16()
        t = torch.randint(0, 400, (R, 200), generator=g, device=DEV).int()
        sets.append((q, kc, vc, t, i32(lens), 0.088))
    want = [prims.attn_decode_paged(*x) for x in sets]
    torch.cuda.synchronize()
    out = [torch.empty_like(w) for w in want]
    for _ in range(20):
        for p, x, o in zip(ps, sets, out):
            p.attn_decode_paged(*x, out=o)
    torch.cuda.synchronize()
    for o, w in zip(out, want):
        assert torch.equal(o, w)
    for p in ps:
        p.close()


def test_refused_request_attends_its_old_keys(prims):
    """a request without a free page keeps its length, appends nothing, and attends what it has"""
    import torch
    e = Engine(prims, 3, 4, 16, 4, False, BF16, 3)
    e.new.copy_(i32([16, 16, 16]))
    e.slots, e.pos = i64([0] * 48), i64([0] * 48)
    q, k, v = e.q, e.k, e.v
    e.q, e.k, e.v = (torch.zeros((48, *t.shape[1:]), dtype=t.dtype, device=DEV) for t in (q, k, v))
    feed(e, 3)
    e.step()
    assert e.lens.tolist() == [16] * 3
    e.slots, e.pos, e.q, e.k, e.v = i64([0] * 3), i64([0] * 3), q, k, v
    feed(e, 4)
    e.new.copy_(i32([17, 17, 16]))  # one page is left
    before = e.kc.clone()
    e.step()
    assert e.lens.tolist() == [17, 16, 16] and e.ends.tolist() == [4, 4]
    assert e.slots.tolist() == [int(e.table[0, 1]) * 16, -1, -1]
    changed = (e.kc != before).view(-1, 2 * 128).any(1).nonzero().flatten().tolist()
    assert changed == [e.slots[0].item()]
    e.attend()
    K, V = (c.double().cpu().numpy() for c in (e.kc, e.vc))
    ref, bound = PO.attn_decode(e.q.double().cpu().numpy(), K, V, e.table.cpu().numpy(), [17, 16, 16], 16, 0, 0.088)
    assert np.all(np.abs(e.out.double().cpu().numpy() - ref) <= bound)
