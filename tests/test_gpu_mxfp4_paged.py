"""GPU: the paged KV cache in MXFP4 pages against plain forms (tests/paged_oracle.py
for attention, tests/mxfp4_oracle.py for the format). The append is bit for bit
qk_norm_rope with its rows quantized by the format's rule; attention is gated on
the bound counted in paged_oracle.attn_decode, plus half a step of a 16-bit
output."""
import math

import numpy as np
import pytest

import mxfp4_oracle as MO
import oracle as O
import paged_oracle as PO
from test_gpu_paged import i32, i64, rope_tables, rows
from util import BF16, F16, to_dev

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
U = 2.0**-24  # half a step of f32, relative


def u8(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a, np.uint8)).to(DEV)


# ------------------------------------------------------------------- append
def run_append(prims, dt, T, qh, kh, D, ps, pad=0, use_rope=True, offset=0, seed=7):
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
    base = [rows(seed + i, (T, (qh if i == 0 else kh) + 1, D), dt) for i in range(3)]  # rows in wider ones
    q, k, v = base[0][:, offset:offset + qh], base[1][:, offset:offset + kh], base[2][:, :kh]
    eq, ek = q.clone(), k.clone()
    co, si = rope_tables(500, D, dt) if use_rope else (None, None)
    dpos, dslot = i64(pos), i64(slot)
    prims.qk_norm_rope(eq, ek, 1e-6, 3.87, co, si, dpos)
    kc, vc = (torch.full((pages, ps, kh, D // 2), 77, dtype=torch.uint8, device=DEV) for _ in range(2))
    kd, vd = (torch.full((pages, ps, kh, D // 32), 99, dtype=torch.uint8, device=DEV) for _ in range(2))
    want = [t.clone().view(-1, kh, t.shape[-1]) for t in (kc, vc, kd, vd)]
    prims.qk_norm_rope_paged(q, k, v, 1e-6, 3.87, co, si, dpos, dslot, kc, vc, kd, vd)
    assert torch.equal(q.contiguous().view(torch.int16), eq.view(torch.int16))
    assert torch.equal(k.contiguous().view(torch.int16), ek.view(torch.int16))
    live = torch.from_numpy((slot >= 0) & (slot < pages * ps)).to(DEV)
    for c, d, x in ((0, 2, ek), (1, 3, v)):
        qs, sc = MO.quantize(x.double().cpu().numpy())
        want[c][dslot[live]] = u8(qs)[live]
        want[d][dslot[live]] = u8(sc)[live]
    for g, w in zip((kc, vc, kd, vd), want):
        assert torch.equal(g.view(-1, kh, g.shape[-1]), w)


@pytest.mark.parametrize("dt", (BF16, F16))
@pytest.mark.parametrize("T,qh,kh,D,ps", ((1, 40, 8, 128, 16), (61, 32, 2, 128, 16), (130, 4, 1, 64, 32), (33, 3, 3, 256, 1),
                                          (701, 5, 3, 128, 16), (9, 0, 2, 64, 8)))
def test_append(prims, dt, T, qh, kh, D, ps):
    run_append(prims, dt, T, qh, kh, D, ps, pad=2 if T > 40 else 0)


def test_append_without_rope_and_from_wider_rows(prims):
    run_append(prims, BF16, 21, 4, 2, 128, 8, use_rope=False)
    run_append(prims, F16, 21, 4, 2, 64, 8, offset=1)


@pytest.mark.parametrize("dt", (BF16, F16))
def test_append_specials(prims, dt):
    """NaN, infinities, zeros, ties and the type's ends in v: the quantizer's rule, block by block"""
    import torch
    kind = {BF16: torch.bfloat16, F16: torch.float16}[dt]
    v = torch.randn((3, 1, 128), generator=torch.Generator().manual_seed(3)).to(kind)
    v[0, 0, 3], v[0, 0, 40] = float("nan"), float("inf")
    v[0, 0, 64:96] = 0.0
    v[0, 0, 96:] = torch.arange(32).to(kind) / 4
    v[1] = torch.finfo(kind).max
    v[2] = torch.finfo(kind).smallest_normal / 8
    q, k = (torch.ones((3, 1, 128), dtype=kind, device=DEV) for _ in range(2))
    kc, vc = (torch.zeros((1, 4, 1, 64), dtype=torch.uint8, device=DEV) for _ in range(2))
    kd, vd = (torch.zeros((1, 4, 1, 4), dtype=torch.uint8, device=DEV) for _ in range(2))
    prims.qk_norm_rope_paged(q, k, v.to(DEV), 1e-6, 1.0, None, None, i64([0, 1, 2]), i64([1, 0, 2]), kc, vc, kd, vd)
    qs, s = MO.quantize(v.double().numpy())
    got = [t[0, [1, 0, 2]].cpu().numpy() for t in (vc, vd)]
    assert np.array_equal(got[1], s)
    assert np.array_equal(MO.values(*got), MO.values(qs, s), equal_nan=True)


def test_append_errors(prims):
    import torch
    q, k = (torch.zeros((2, h, 128), dtype=torch.bfloat16, device=DEV) for h in (4, 2))
    kc, kd = (torch.zeros((3, 16, 2, n), dtype=torch.uint8, device=DEV) for n in (64, 4))
    p = i64([0, 1])
    args = lambda **kw: {**dict(q=q, k=k, v=k.clone(), eps=1e-6, qk_scale=1.0, cos=None, sin=None, positions=p, slot_map=p,
                                k_cache=kc, v_cache=kc.clone(), k_scale=kd, v_scale=kd.clone()), **kw}
    prims.qk_norm_rope_paged(**args())
    for bad, match in ((dict(k_scale=None), "both"), (dict(k_scale=None, v_scale=None), "need k_scale"),
                       (dict(k_scale=kd.half(), v_scale=kd.half()), "scales"), (dict(v_cache=kc.to(torch.int8)), "needed"),
                       (dict(k_scale=kd[..., :2].contiguous()), "scales"), (dict(k_cache=kc[:, :, :1].contiguous()), "caches must be"),
                       (dict(v_cache=kc[:2]), "shape"), (dict(slot_map=i32([0, 1])), "int64"),
                       (dict(k_cache=torch.zeros((3, 16, 2, 128), dtype=torch.uint8, device=DEV)), "caches must be")):
        with pytest.raises(Exception, match=match):
            prims.qk_norm_rope_paged(**args(**bad))
    z = lambda h, d: torch.zeros((2, h, d), dtype=torch.bfloat16, device=DEV)
    c = lambda d: torch.zeros((1, 16, 2, d), dtype=torch.uint8, device=DEV)
    with pytest.raises(Exception, match="head_dim 64, 128 or 256"):
        prims.qk_norm_rope_paged(z(4, 32), z(2, 32), z(2, 32), 1e-6, 1.0, None, None, p, p, c(16), c(16), c(1), c(1))
    with pytest.raises(Exception, match="32s"):
        prims.qk_norm_rope_paged(z(4, 80), z(2, 80), z(2, 80), 1e-6, 1.0, None, None, p, p, c(40), c(40), c(2), c(2))


# ---------------------------------------------------------------- attention
def decode_case(prims, lens, nq, nkv, D, ps, dt=BF16, out=None, window=0, seed=61, scaling=None, gap=0, bad=None, ws=None,
                scales=None):
    """a pool whose unused slots hold NaN scales: only the requests' own keys may count"""
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
    for r, i, page in bad or ():
        table[r, i] = page
    qb = O.normal(seed, (R, nq, D), 0.0, 1.0, dt)
    pools = []
    for _ in range(2):
        qs, s = MO.quantize(rng.standard_normal((N, ps, nkv, D)))
        if scales is not None:
            s = rng.integers(*scales, s.shape).astype(np.uint8)
        vals = MO.values(qs, s)
        s = s.copy()
        s[~used] = 255
        pools.append((u8(qs), u8(s), vals))
    (kc, kd, K), (vc, vd, V) = pools
    scaling = 1.0 / math.sqrt(D) if scaling is None else scaling
    dq = to_dev(qb, dt)
    od = {None: torch.float32, "same": dq.dtype}[out]
    wide = torch.full((R + 1, nq + gap, D), 7.5, dtype=od, device=DEV)
    o = wide[:R, :nq]
    wt = torch.full((R, W + gap), 5, dtype=torch.int32, device=DEV)
    wt[:, :W] = i32(table)
    (ws or prims).attn_decode_paged(dq, kc, vc, wt[:, :W], i32(lens), scaling, window, kd, vd, o)
    assert (wide[R:] == 7.5).all() and (wide[:, nq:] == 7.5).all()
    # (the bound counts roundings of q.k by sum |q k| scaling, which has to be a magnitude: a negative scaling is the
    # same scores from -q and its magnitude, every product and rounding alike but for the sign)
    sign = -1.0 if scaling < 0 else 1.0
    ref, bound = PO.attn_decode(sign * O.to_f64(qb, dt), K, V, table, lens, ps, window, sign * scaling)
    got = o.double().cpu().numpy()
    if out == "same":
        bound = bound + np.abs(ref) * (2.0**-8 if dt == BF16 else 2.0**-11) + 2.0**-24
    err = np.abs(got - ref)
    assert np.all(err <= bound * 1.0000001 + 1e-30), (float(err.max()), np.argwhere(~(err <= bound))[:4].tolist())
    return got


DTS = (BF16, F16)


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("D", (64, 128))
@pytest.mark.parametrize("ps", (1, 16, 32, 64))
def test_decode_ragged(prims, dt, D, ps):
    """lengths from none to many, at the edges of pages, of the tiles and of a work-group's units"""
    decode_case(prims, [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 500, 0, 1025], 10, 2, D, ps, dt)


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("nq,nkv", ((1, 1), (7, 7), (40, 8), (32, 2), (9, 1), (20, 1), (64, 2), (46, 2)))
def test_decode_heads(prims, dt, nq, nkv):
    """group sizes of 1 to 32 heads, in strided tensors, the output at q's dtype"""
    decode_case(prims, [70, 0, 333], nq, nkv, 128, 16, dt, out="same", gap=2, seed=nq)


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("window", (1, 20, 64, 65, 1000, 2**40))
def test_decode_window(prims, dt, window):
    decode_case(prims, [0, 1, 19, 20, 21, 300, 1500, 999, 1000, 1001], 10, 2, 64, 16, dt, window=window)


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("out", (None, "same"))
def test_decode_long(prims, dt, out):
    """one long request, split over many work-groups, next to short ones; one alone; many parts among many short"""
    decode_case(prims, [20011, 3, 0, 4096], 32, 2, 128, 16, dt, out=out)
    decode_case(prims, [9001], 5, 1, 64, 128, dt, out=out)
    decode_case(prims, [100000], 2, 1, 64, 64, dt, out=out)
    decode_case(prims, [9] * 40 + [30000] + [7] * 60, 3, 1, 64, 16, dt, out=out)


def test_decode_many_short(prims):
    """more requests than work-groups, all short; nothing at all"""
    rng = np.random.default_rng(8)
    decode_case(prims, rng.integers(0, 40, 1500).tolist(), 2, 1, 64, 8)
    decode_case(prims, [1] * 700, 8, 8, 64, 1)
    decode_case(prims, [0] * 33, 8, 2, 64, 16)


@pytest.mark.parametrize("R", (63, 64, 65, 257))
def test_decode_request_counts(prims, R):
    decode_case(prims, [1000] + [3] * (R - 2) + [777], 4, 2, 64, 16)


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("scaling", (1.0, -0.088, 0.0))
def test_decode_peaked(prims, dt, scaling):
    """scores over tens of units, late maxima; a negative scaling; none"""
    decode_case(prims, [700, 65, 2000], 10, 2, 128, 16, dt, scaling=scaling)


@pytest.mark.parametrize("dt", DTS)
def test_decode_bad_pages(prims, dt):
    """pages outside the pool are left out, a request of only such pages gives zeros"""
    bad = [(0, 0, -1), (1, 3, 10**6), (2, 0, -2**31), (2, 1, 2**31 - 1), (3, 2, -1)]
    got = decode_case(prims, [40, 200, 32, 48, 0], 4, 2, 64, 16, dt, bad=bad)
    assert not got[2].any()


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("scales", ((115, 131), (60, 64), (180, 184)))
def test_decode_scales(prims, dt, scales):
    """block scales of every size beside each other, and far from 1 on both sides (scores stay in range through q's
    scaling)"""
    mid = 2.0**(127 - scales[0] - 2)
    decode_case(prims, [300, 64, 5, 1100], 10, 2, 128, 16, dt, scales=scales, scaling=0.05 * min(mid, 1.0) if scales[0] > 127 else 0.05 * mid)


def test_decode_small_workspaces(prims):
    """room for a few teams, for one (nothing is cut), for none of it"""
    import mgprims
    for size in (64, 40000, 200000):
        p = mgprims.Prims(0, workspace_bytes=size)
        decode_case(p, [3000, 5, 0, 900], 10, 2, 128, 16, ws=p)
        decode_case(p, [200] * 90, 10, 2, 64, 16, ws=p)
        p.close()


def attend(prims, q, K, V, table, lens, scaling, **kw):
    """K, V: (codes, scales) on the device"""
    return prims.attn_decode_paged(q, K[0], V[0], table, lens, scaling, 0, K[1], V[1], **kw)


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("D,n,at", ((128, 40, 0), (64, 900, 0), (128, 900, 555)))
@pytest.mark.parametrize("same", (False, True))
def test_small_weights_behind_one_key(prims, dt, D, n, at, same):
    """one key (at `at`) takes nearly everything, and its value is zero in half of the blocks: there an output is made
    of the other keys' weights alone, 2^-13 to 2^-100 of its own. q and k are zero but for one dim of exact products;
    the large key's score is 0, so a score s (in units of log 2) is off by the roundings of the scaling and of their
    product, 2 U |s|, relative 2 U |s| log 2 of its weight; exponential and quotient 8 U; the weight's parts 2^-16;
    its sum (n / 32 + 128) U; half a step of a 16-bit output."""
    import torch
    rng = np.random.default_rng(D + n + at)
    gaps = np.array([13, 16, 19, 21, 24, 26, 30, 34, 37, 40, 50, 64, 80, 96])
    R, ps = len(gaps), 16
    W = -(-n // ps)
    N = R * W
    table = rng.permutation(N).reshape(R, W)
    k = np.zeros((R, W * ps, 1, D))
    k[:, :, 0, 0] = 1.0 + rng.integers(0, 2, (R, W * ps)) / 2  # 1 or 1.5
    k[:, at] = 0.0
    q = np.zeros((R, 1, D))
    q[:, 0, 0] = -gaps * 2.0**-4
    scaling = float(np.float32(16 * math.log(2)))
    vq, vs = MO.quantize(rng.standard_normal((R, W * ps, 1, D)))
    vq[:, at, 0, :D // 4] = 0
    pk = [np.zeros((N, ps, 1, w), np.uint8) for w in (D // 2, D // 32)] + [np.zeros((N, ps, 1, w), np.uint8) for w in (D // 2, D // 32)]
    for dst, src in zip(pk, (*MO.quantize(k), vq, vs)):
        dst[table] = src.reshape(R, W, ps, 1, -1)
    dq = to_dev(O.from_f64(q, dt), dt)
    out = torch.full((R, 1, D), 7.0, dtype=dq.dtype if same else torch.float32, device=DEV)
    attend(prims, dq, (u8(pk[0]), u8(pk[1])), (u8(pk[2]), u8(pk[3])), i32(table), i32([n] * R), scaling, out=out)
    got = out.double().cpu().numpy()
    V = MO.values(vq, vs)
    half = (2.0**-8 if dt == BF16 else 2.0**-11) if same else 0.0
    least = 2.0**-24 if same and dt == F16 else 0.0  # (f16 outputs end there)
    for r in range(R):
        s = q[r, 0, 0] * k[r, :n, 0, 0] * scaling
        p = np.exp(s - s.max())
        p /= p.sum()
        ref, mag = p @ V[r, :n, 0], p @ np.abs(V[r, :n, 0])
        rel = 4 * U * 1.5 * gaps[r] * math.log(2) + 16 * U + 2.0**-16 + (n / 32 + 128) * U
        assert np.all(np.abs(got[r, 0] - ref) <= rel * mag + half * np.abs(ref) * 1.01 + least), (r, got[r, 0, :3], ref[:3])


@pytest.mark.parametrize("dt", DTS)
def test_nan_scales(prims, dt):
    """a key's NaN block reaches its request's heads of that kv head, a value's the block's dims of them, nothing else;
    a masked one (behind the length, in a page of another request) reaches nobody"""
    import torch
    R, n, nkv, D, ps = 3, 300, 2, 128, 16
    rng = np.random.default_rng(2)
    kind = {BF16: torch.bfloat16, F16: torch.float16}[dt]
    q = torch.randn((R, 4, D), generator=torch.Generator().manual_seed(1)).to(kind).to(DEV)
    table, lens = i32(np.arange(R * 19).reshape(R, 19)), i32([n] * R)
    pools = [[u8(x) for x in MO.quantize(rng.standard_normal((R * 19, ps, nkv, D)))] for _ in range(2)]
    base = attend(prims, q, *pools, table, lens, 0.088)
    assert torch.isfinite(base).all()
    page, off = 19 + (n - 1) // ps, (n - 1) % ps  # request 1's newest key
    for which in range(2):
        keep = pools[which][1].clone()
        pools[which][1][page, off, 1, 2] = 255
        got = attend(prims, q, *pools, table, lens, 0.088)
        hit = got[1, 2:] if which == 0 else got[1, 2:, 64:96]
        assert torch.isnan(hit).all()
        hit.copy_(base[1, 2:] if which == 0 else base[1, 2:, 64:96])
        assert torch.equal(got, base)
        pools[which][1][page, off + 1:, :, :] = 255
        pools[which][1][page, off, 1, 2] = keep[page, off, 1, 2]
        assert torch.equal(attend(prims, q, *pools, table, lens, 0.088), base)
        pools[which][1].copy_(keep)


def test_infinite_scores(prims):
    """a key of score -inf weighs nothing beside another; such keys alone give NaN; no key gives zeros"""
    import torch
    D, ps = 64, 16
    rng = np.random.default_rng(3)
    kq, ks = MO.quantize(rng.standard_normal((8, ps, 1, D)))
    vq, vs = MO.quantize(rng.standard_normal((8, ps, 1, D)))
    kq[2, 3], ks[2, 3] = 0xff, 254  # -6 2^127 in every dim: products with q > 0 are -inf
    kq[4], ks[4] = 0xff, 254
    q = torch.rand((3, 2, D), generator=torch.Generator().manual_seed(4)).add_(4.0).bfloat16().to(DEV)
    pools = ((u8(kq), u8(ks)), (u8(vq), u8(vs)))
    table = i32([[0, 1, 2, 3], [4, 4, 4, 4], [5, 6, 7, 0]])
    got = attend(prims, q, *pools, table, i32([64, 40, 0]), 0.1)
    assert torch.isnan(got[1]).all() and not got[2].any()
    live = np.ones(64, bool)
    live[35] = False
    K, V = (MO.values(a, b).reshape(-1, D)[:64] for a, b in ((kq, ks), (vq, vs)))
    ref, bound = PO.attn_decode(q[:1].double().cpu().numpy(), K[live][:, None, None], V[live][:, None, None],
                                np.arange(63)[None], [63], 1, 0, 0.1)
    assert np.all(np.abs(got[0].double().cpu().numpy() - ref[0]) <= bound[0])


def test_decode_far_pages(prims):
    """a pool of more than 2^32 bytes a cache: offsets past 32 bits, lengths in its last pages"""
    import torch
    nkv, D, ps = 8, 128, 64
    N = (2**32 // (nkv * D // 2 * ps)) + 70
    pools = [[torch.empty((N, ps, nkv, w), dtype=torch.uint8, device=DEV) for w in (D // 2, D // 32)] for _ in range(2)]
    rng = np.random.default_rng(5)
    vals = []
    for p in pools:
        qs, s = MO.quantize(rng.standard_normal((60, ps, nkv, D)))
        p[0][-60:], p[1][-60:] = u8(qs), u8(s)
        vals.append(MO.values(qs, s))
    table = np.stack([np.arange(N - 60, N - 30), np.arange(N - 1, N - 31, -1)]).astype(np.int32)
    lens = [1900, 1777]
    q = torch.randn((2, 16, D), generator=torch.Generator().manual_seed(5)).bfloat16().to(DEV)
    got = attend(prims, q, *pools, i32(table), i32(lens), 0.088).double().cpu().numpy()
    ref, bound = PO.attn_decode(q.double().cpu().numpy(), *vals, table - (N - 60), lens, ps, 0, 0.088)
    assert np.all(np.abs(got - ref) <= bound)
    # the append writes there too
    k = torch.randn((1, nkv, D), generator=torch.Generator().manual_seed(6)).bfloat16().to(DEV)
    (kc, kd), (vc, vd) = pools
    prims.qk_norm_rope_paged(q[:1], k, k.clone(), 1e-6, 1.0, None, None, i64([0]), i64([N * ps - 1]), kc, vc, kd, vd)
    qs, s = MO.quantize(k.double().cpu().numpy())
    assert np.array_equal(kc[-1, -1].cpu().numpy(), qs[0]) and np.array_equal(kd[-1, -1].cpu().numpy(), s[0])


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("window", (1, 63, 100, 1000))
@pytest.mark.parametrize("freed", (-1, 0))
def test_nothing_before_a_window_is_used(prims, dt, window, freed):
    """pages before a window freed (bad entries) or holding another request's NaN blocks: the same bits"""
    import torch
    rng = np.random.default_rng(window)
    kind = {BF16: torch.bfloat16, F16: torch.float16}[dt]
    lens, ps, W = [700, 64, 65, 1300], 16, 90
    pools = [[u8(x) for x in MO.quantize(rng.standard_normal((4 * W + 1, ps, 2, 64)))] for _ in range(2)]
    for p in pools:
        p[1][0] = 255
    table = 1 + np.arange(4 * W).reshape(4, W)
    q = torch.randn((4, 6, 64), generator=torch.Generator().manual_seed(2)).to(kind).to(DEV)
    run = lambda t: prims.attn_decode_paged(q, pools[0][0], pools[1][0], i32(t), i32(lens), 0.125, window, pools[0][1], pools[1][1])
    base = run(table)
    gone = table.copy()
    for r, n in enumerate(lens):
        gone[r, :max(0, n - window) // ps] = freed
    assert torch.isfinite(base).all() and torch.equal(run(gone), base)


def test_empty_call_and_errors(prims):
    import torch
    q = torch.zeros((2, 8, 128), dtype=torch.bfloat16, device=DEV)
    kc, kd = (torch.zeros((4, 16, 2, n), dtype=torch.uint8, device=DEV) for n in (64, 4))
    t, n = i32([[0, 1]] * 2), i32([3, 4])
    args = lambda **kw: {**dict(q=q, k_cache=kc, v_cache=kc, page_table=t, lens=n, scaling=0.1, k_scale=kd, v_scale=kd), **kw}
    prims.attn_decode_paged(**args())
    assert prims.attn_decode_paged(**args(q=q[:0], page_table=t[:0], lens=n[:0])).shape == (0, 8, 128)
    for bad, match in ((dict(k_scale=None, v_scale=None), "need k_scale"), (dict(v_scale=None), "both"),
                       (dict(k_scale=kd.half()), "scales"), (dict(v_scale=kd[:2]), "scales"), (dict(q=q[:, :7]), "multiple"),
                       (dict(q=q.float()), "bf16 or f16"), (dict(v_cache=kc.to(torch.int8)), "needed"),
                       (dict(k_cache=torch.zeros(4 * 16 * 2 * 64 + 1, dtype=torch.uint8, device=DEV)[1:].view(4, 16, 2, 64)), "aligned"),
                       (dict(k_scale=torch.zeros(4 * 16 * 2 * 4 + 1, dtype=torch.uint8, device=DEV)[1:].view(4, 16, 2, 4)), "aligned"),
                       (dict(out=torch.zeros((2, 8, 128), dtype=torch.float16, device=DEV)), "dtype_out"),
                       (dict(k_cache=kc[:, :12].contiguous(), v_cache=kc[:, :12].contiguous(), k_scale=kd[:, :12].contiguous(),
                             v_scale=kd[:, :12].contiguous()), "power of two")):
        with pytest.raises(Exception, match=match):
            prims.attn_decode_paged(**args(**bad))
    c = lambda d: torch.zeros((4, 16, 2, d), dtype=torch.uint8, device=DEV)
    with pytest.raises(Exception, match="head_dim"):
        prims.attn_decode_paged(torch.zeros((2, 8, 256), dtype=torch.bfloat16, device=DEV), c(128), c(128), t, n, 0.1, 0, c(8), c(8))


# ------------------------------------------------------- a run of them together
class Engine:
    """a small layer served from 4 bits: projections, cache and output product in MXFP4, state in device memory"""

    def __init__(self, prims, R, W, ps, N, dt, T, nq=10, nkv=2, D=128, hidden=416):
        import torch
        kind = {BF16: torch.bfloat16, F16: torch.float16}[dt]
        self.p, self.ps, self.nq, self.nkv, self.D = prims, ps, nq, nkv, D
        self.table, self.ring = i32(np.full((R, W), -1)), i32(np.arange(N)[::-1].copy())
        self.lens, self.ends, self.new = i32([0] * R), i64([0, N]), i32([0] * R)
        self.starts, self.slots, self.pos = i32([0] * (R + 1)), i64([0] * T), i64([0] * T)
        z = lambda *s, d=kind: torch.zeros(s, dtype=d, device=DEV)
        g = torch.Generator(device=DEV).manual_seed(4)
        out = (nq + 2 * nkv) * D
        self.w = [self.weight(torch.randn(s, generator=g, device=DEV).to(kind) / math.sqrt(s[1])) for s in ((out, hidden), (hidden, nq * D))]
        self.x, self.xq, self.xs = z(T, hidden), z(T, hidden // 2, d=torch.uint8), z(T, hidden // 32, d=torch.uint8)
        self.qkv = z(T, out)
        self.q, self.k, self.v = (t.view(T, -1, D) for t in self.qkv.split([nq * D, nkv * D, nkv * D], 1))
        self.kc, self.vc = z(N, ps, nkv, D // 2, d=torch.uint8), z(N, ps, nkv, D // 2, d=torch.uint8)
        self.kd, self.vd = (z(N, ps, nkv, D // 32, d=torch.uint8) for _ in range(2))
        self.co, self.si = rope_tables(W * ps, D, dt)
        self.out, self.y = z(R, nq, D), z(R, hidden, d=torch.float32)

    def weight(self, w):
        import torch
        q, s = (torch.empty((w.shape[0], w.shape[1] // n), dtype=torch.uint8, device=DEV) for n in (2, 32))
        self.p.quantize_mxfp4(w, q, s)
        return q, s

    def project(self, small):
        """16-bit activations for a step, MXFP4 ones for a prompt"""
        if small:
            self.p.gemv_mxfp4(*self.w[0], self.x, self.qkv)
        else:
            self.p.quantize_mxfp4(self.x, self.xq, self.xs)
            self.p.gemm_mxfp4(self.xq, self.xs, *self.w[0], self.qkv)

    def step(self, small=True):
        p = self.p
        self.project(small)
        p.kv_pages(self.table, self.lens, self.new, self.ps, self.ring, self.ends, self.lens, self.ends, self.starts,
                   self.slots, self.pos)
        p.qk_norm_rope_paged(self.q, self.k, self.v, 1e-6, 3.87, self.co, self.si, self.pos, self.slots, self.kc,
                             self.vc, self.kd, self.vd)

    def attend(self):
        p = self.p
        p.attn_decode_paged(self.q, self.kc, self.vc, self.table, self.lens, 0.088, 0, self.kd, self.vd, self.out)
        p.gemv_mxfp4(*self.w[1], self.out.view(self.out.shape[0], -1), self.y)


def feed(e, seed):
    import torch
    e.x.copy_(torch.randn(e.x.shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV))


@pytest.mark.parametrize("dt", DTS)
def test_prompts_then_decode(prims, dt):
    """prompts of ragged lengths in one pass, then decode steps: every stage is its 64-bit form of what entered it"""
    import torch
    R, ps = 6, 16
    prompt = [5, 0, 33, 16, 70, 1]
    T = sum(prompt)
    half = 2.0**-8 if dt == BF16 else 2.0**-11
    e = Engine(prims, R, 8, ps, 60, dt, T)
    W = [MO.values(*(t.cpu().numpy() for t in w)) for w in e.w]
    keys = [[] for _ in range(R)]

    def f64(t):
        return t.double().cpu().numpy()

    def projected(x):
        ref, bound = MO.product(W[0], x)
        e.project_check = np.all(np.abs(f64(e.qkv) - ref) <= bound + half * (np.abs(ref) + bound) + 2.0**-24)
        assert e.project_check

    def record(owner):
        for t, r in enumerate(owner):
            keys[r].append([MO.values(*MO.quantize(f64(x[t]))) for x in (e.k, e.v)])

    feed(e, 1)
    e.new.copy_(i32(prompt))
    e.project(False)
    projected(MO.values(*MO.quantize(f64(e.x))))
    e.step(False)
    assert e.lens.tolist() == prompt
    record([r for r in range(R) for _ in range(prompt[r])])
    d = Engine(prims, R, 8, ps, 60, dt, R)
    for name in ("table", "ring", "lens", "ends", "kc", "vc", "kd", "vd"):
        setattr(d, name, getattr(e, name))
    e = d
    for i in range(8):
        feed(e, 10 + i)
        e.new.copy_(e.lens + 1)
        e.project(True)
        projected(f64(e.x))
        e.step()
        e.attend()
        record(range(R))
        q = f64(e.q)
        for r in range(R):
            K, V = (np.stack([x[c] for x in keys[r]])[:, None] for c in (0, 1))
            ref, bound = PO.attn_decode(q[r:r + 1], K, V, np.arange(len(keys[r]))[None], [len(keys[r])], 1, 0, 0.088)
            assert np.all(np.abs(f64(e.out[r]) - ref[0]) <= bound[0] + half * (np.abs(ref[0]) + bound[0]) + 2.0**-24), (i, r)
        ref, bound = MO.product(W[1], f64(e.out).reshape(R, -1))
        assert np.all(np.abs(f64(e.y) - ref) <= bound)


def test_captured_decode_loop(prims):
    """a decode step captured once and replayed, with eager work between the replays: every replay equals the eager
    loop, pages and all"""
    import torch
    import mgprims
    R, ps = 7, 16
    side = torch.cuda.Stream()
    p = mgprims.Prims(0, stream=side.cuda_stream)
    e, ref = Engine(p, R, 6, ps, 50, BF16, R), Engine(prims, R, 6, ps, 50, BF16, R)
    for x in (e, ref):
        x.new.copy_(i32([1, 0, 1, 1, 1, 0, 1]))
    torch.cuda.synchronize()

    def step(x):
        x.step()
        x.attend()
        p_ = x.p
        p_.quantize_mxfp4(x.x, x.xq, x.xs)
        p_.gemm_mxfp4(x.xq, x.xs, *x.w[0], x.qkv)
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
        for name in ("table", "ring", "lens", "ends", "slots", "pos", "kc", "vc", "kd", "vd", "out", "y", "qkv"):
            assert torch.equal(getattr(e, name), getattr(ref, name)), (i, name)
    assert ref.lens.tolist() == [40, 0, 0, 40, 40, 20, 40]
    p.close()


def test_two_contexts_at_once(prims):
    """two contexts on two streams, their calls interleaved"""
    import torch
    import mgprims
    streams = [torch.cuda.Stream() for _ in range(2)]
    ps = [mgprims.Prims(0, stream=s.cuda_stream) for s in streams]
    rng = np.random.default_rng(9)
    pools = [[u8(x) for x in MO.quantize(rng.standard_normal((400, 16, 2, 128)))] for _ in range(2)]
    g = torch.Generator(device=DEV).manual_seed(9)
    sets = []
    for lens in ([3000, 40, 0, 900], [17] * 20 + [2500]):
        q = torch.randn((len(lens), 32, 128), generator=g, device=DEV).bfloat16()
        sets.append((q, *pools, torch.randint(0, 400, (len(lens), 200), generator=g, device=DEV).int(), i32(lens), 0.088))
    want = [attend(prims, *x) for x in sets]
    torch.cuda.synchronize()
    out = [torch.empty_like(w) for w in want]
    for _ in range(20):
        for p, x, o in zip(ps, sets, out):
            attend(p, *x, out=o)
    torch.cuda.synchronize()
    for o, w in zip(out, want):
        assert torch.equal(o, w)
    for p in ps:
        p.close()
