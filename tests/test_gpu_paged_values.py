"""GPU: paged decode attention where scores and weights reach the ends of their
range, against 64 bits. The inputs make every score exact (or nearly so), so that
a bound counts the weights and sums alone.
"""
import numpy as np
import pytest

import oracle as O
import paged_oracle as PO
from test_gpu_paged import DEV, FORMS, i32
from util import BF16, to_dev

pytestmark = pytest.mark.gpu

U = 2.0**-24  # half a step of f32, relative


def pool(x, dt, q8, quants=None):
    """x [pages, ps, heads, D] f64 of values that the storage type holds, or Q8_0: quants of that shape, x their
    scales [.., D / 32] -> (cache, scales, values in f64)"""
    import torch
    if not q8:
        b = O.from_f64(x, dt)
        return to_dev(b, dt), None, O.to_f64(b, dt)
    d = x.astype(np.float16)
    vals = quants.astype(np.float64).reshape(*d.shape, 32) * d.astype(np.float64)[..., None]
    return torch.from_numpy(quants.astype(np.int8)).to(DEV), torch.from_numpy(d).to(DEV), vals.reshape(quants.shape)


def random_values(rng, shape, dt, q8):
    if not q8:
        return pool(rng.standard_normal(shape), dt, False)
    return pool(rng.uniform(0.001, 0.03, (*shape[:3], shape[3] // 32)), dt, True, rng.integers(-127, 128, shape))


def softmax_rows(s, V):
    """softmax(s) V and softmax(s) |V| in f64: s [heads, keys], V [keys, D]"""
    with np.errstate(invalid="ignore"):
        p = np.exp(s - s.max(1, keepdims=True))
    p /= p.sum(1, keepdims=True)
    return p @ V, p @ np.abs(V)


@pytest.mark.parametrize("dt,q8", FORMS)
@pytest.mark.parametrize("D,n", ((128, 50), (64, 700)))
@pytest.mark.parametrize("same", (False, True))
def test_finite_scores_of_any_magnitude(prims, dt, q8, D, n, same):
    """scores of 2^24 to 2^30 of either sign. A request's keys are of two kinds, t in every dim and t / 2, and q
    holds a power of two: every product and partial sum of a score is a whole multiple of 2^-2 below 2^24 of its
    last bit, so scores are exact, equal within a kind, and far enough apart between the kinds that one kind
    weighs nothing. Weights are then 0 and 1: an output is its kind's mean, off by its sum of n terms (n / 32 + 128
    additions meet one), the quotient and the scaling (4) and half a step of a 16-bit output."""
    import torch
    rng = np.random.default_rng(D + n)
    R, ps = 24, 16
    W = -(-n // ps)
    N = R * W
    table = rng.permutation(N).reshape(R, W)
    t = 2048.0 + 85 * np.arange(R)
    t = np.floor(t / 16) * 16 if dt == BF16 else np.floor(t / 2) * 2  # 8 and 11 bits
    kind = rng.integers(0, 2, (R, W * ps))
    kind[:, 0], kind[:, 1] = 0, 1
    k = np.zeros((N, ps, 1, D))
    k[table] = (t[:, None] / (1 + kind)).reshape(R, W, ps, 1, 1)
    if q8:  # quants 64 and 32 of scales t / 64
        quants = np.zeros((N, ps, 1, D))
        quants[table] = (64 // (1 + kind)).reshape(R, W, ps, 1, 1)
        d = np.zeros((N, ps, 1, D // 32))
        d[table] = (t / 64)[:, None, None, None, None]
        kc, kd, K = pool(d, dt, True, quants)
    else:
        kc, kd, K = pool(k, dt, False)
    assert np.array_equal(K, k)
    vc, vd, V = random_values(rng, (N, ps, 1, D), dt, q8)
    gains = np.array([2048.0, -2048.0, 4096.0, -1024.0, 16384.0, -512.0])
    q = np.broadcast_to(gains[None, :, None], (R, len(gains), D))
    dq = to_dev(O.from_f64(np.ascontiguousarray(q), dt), dt)
    scaling = D**-0.5
    out = torch.full(q.shape, 7.0, dtype=dq.dtype if same else torch.float32, device=DEV)
    prims.attn_decode_paged(dq, kc, vc, i32(table), i32([n] * R), scaling, 0, kd, vd, out)
    got = out.double().cpu().numpy()
    half = (2.0**-8 if dt == BF16 else 2.0**-11) if same else 0.0
    for r in range(R):
        key = np.arange(n)
        rows = [x[table[r, key // ps], key % ps, 0] for x in (K, V)]
        ref, mag = softmax_rows(q[r] @ rows[0].T * scaling, rows[1])
        bound = (n / 32 + 132) * U * mag + half * np.abs(ref) + (2.0**-24 if same else 0.0)
        assert np.all(np.abs(got[r] - ref) <= bound), (r, t[r], got[r, :, 0].tolist(), ref[:, 0].tolist())


@pytest.mark.parametrize("dt,q8", FORMS)
@pytest.mark.parametrize("D,n,at", ((128, 40, 0), (64, 900, 0), (128, 900, 555)))
@pytest.mark.parametrize("same", (False, True))
def test_small_weights_behind_one_key(prims, dt, q8, D, n, at, same):
    """one key (at `at`) takes nearly everything, and its value is zero in half of the dims: there an output is made
    of the other keys' weights alone, 2^-13 to 2^-100 of its own. q and k are zero but for one dim, q is a power of
    two and the large key's score is 0, so a score s (in units of log 2) is off by the roundings of the scaling and
    of their product, 2 U |s|, and enters the weight once: relative 2 U |s| log 2; exponential and quotient 8 U; the
    weight's parts 2^-16; its sum (n / 32 + 128) U; half a step of a 16-bit output."""
    import torch
    rng = np.random.default_rng(D + n + at)
    gaps = np.array([13, 16, 19, 21, 24, 26, 30, 34, 37, 40, 50, 64, 80, 99])  # of each request
    R, ps = len(gaps), 16
    W = -(-n // ps)
    N = R * W
    table = rng.permutation(N).reshape(R, W)
    # the others' scores: from the gap to one unit above it, in 64 steps, over log 2 and the gain
    key = np.arange(W * ps)
    k0 = (gaps[:, None] - (key * 37 % 64) / 64) * 0.7
    k0[:, at] = 0.0
    k = np.zeros((N, ps, 1, D))
    if q8:
        quants = np.zeros((N, ps, 1, D))
        d = np.zeros((N, ps, 1, D // 32))
        quants[table, :, 0, 0] = np.where(k0 > 0, 100, 0).reshape(R, W, ps)
        d[table, :, 0, 0] = (k0 / 100).reshape(R, W, ps)
        kc, kd, K = pool(d, dt, True, quants)
    else:
        k[table, :, 0, 0] = k0.reshape(R, W, ps)
        kc, kd, K = pool(k, dt, False)
    if q8:
        vq = rng.integers(-127, 128, (N, ps, 1, D))
        vd_ = rng.uniform(0.001, 0.03, (N, ps, 1, D // 32))
        vq[table[:, at // ps], at % ps, 0, :D // 2] = 0
        vc, vd, V = pool(vd_, dt, True, vq)
    else:
        v = rng.standard_normal((N, ps, 1, D))
        v[table[:, at // ps], at % ps, 0, :D // 2] = 0.0
        vc, vd, V = pool(v, dt, False)
    q = np.zeros((R, 3, D))
    q[:, :, 0] = -1.0
    dq = to_dev(O.from_f64(q, dt), dt)
    out = torch.full(q.shape, 7.0, dtype=dq.dtype if same else torch.float32, device=DEV)
    prims.attn_decode_paged(dq, kc, vc, i32(table), i32([n] * R), 1.0, 0, kd, vd, out)
    got = out.double().cpu().numpy()
    half = (2.0**-8 if dt == BF16 else 2.0**-11) if same else 0.0
    tiny = 2.0**-25 if same and dt != BF16 else 0.0  # half of f16's smallest step
    worst = []
    for r in range(R):
        j = np.arange(n)
        kr, vr = (x[table[r, j // ps], j % ps, 0] for x in (K, V))
        s = q[r] @ kr.T
        ref, mag = softmax_rows(s, vr)
        err = 2 * U * np.abs(s).max() + (8 + n / 32 + 128) * U + 2.0**-16
        bound = err * mag + half * np.abs(ref) + tiny
        assert np.abs(ref[:, :D // 2]).max() < 2.0**(-gaps[r] * 0.99 + 14)  # (these dims do hold small weights only)
        worst.append((int(gaps[r]), float((np.abs(got[r] - ref) / np.maximum(bound, 1e-300)).max())))
    assert all(w <= 1 for _, w in worst), worst


def infinite_keys(D, dt, q8, pages, ps, nkv, seed):
    """a pool of ordinary keys and values, and a function that gives key (page, place) of head 1 the score -inf"""
    import torch
    g = torch.Generator(device=DEV).manual_seed(seed)
    shape = (pages, ps, nkv, D)
    if not q8:
        t = torch.bfloat16 if dt == BF16 else torch.float16
        kc, vc = (torch.randn(shape, generator=g, device=DEV).to(t) for _ in range(2))

        def spoil(page, place):
            kc[page, place, 1, 3] = -float("inf")
        return kc, vc, None, None, spoil
    kc, vc = (torch.randint(-127, 128, shape, generator=g, device=DEV, dtype=torch.int8) for _ in range(2))
    kd, vd = (torch.full((*shape[:3], D // 32), 0.01, dtype=torch.float16, device=DEV) for _ in range(2))

    def spoil(page, place):
        kc[page, place, 1, :32] = -5
        kd[page, place, 1, 0] = float("inf")
    return kc, vc, kd, vd, spoil


@pytest.mark.parametrize("dt,q8", FORMS)
@pytest.mark.parametrize("D,lens,teams", ((128, [40, 5, 300], None), (64, [9000, 33, 700], None), (128, [30000], None),
                                          (64, [200] * 80, 64), (64, [3000] * 3, 64)))
def test_scores_of_minus_infinity(prims, dt, q8, D, lens, teams):
    """a softmax over scores of -inf alone is NaN, for that request and kv head only and however its keys are split;
    with one finite score among them that key takes all; keys left out (bad pages) do not count, and a request with
    such keys only gives zeros"""
    import mgprims
    import torch
    ps, nkv, R = 16, 2, len(lens)
    W = -(-max(lens) // ps)
    kc, vc, kd, vd, spoil = infinite_keys(D, dt, q8, R * W, ps, nkv, D + R)
    table = torch.arange(R * W, device=DEV).int().view(R, W)
    q = torch.rand((R, 6, D), device=DEV).add_(0.25).to(torch.bfloat16 if dt == BF16 else torch.float16)
    n = i32(lens)
    p = mgprims.Prims(0, workspace_bytes=teams) if teams else prims  # (no room for partial results: nothing is cut)
    run = lambda t=table, w=0: p.attn_decode_paged(q, kc, vc, t, n, 0.1, w, kd, vd)
    base = run()
    assert torch.isfinite(base).all()
    r = R - 1
    rows = slice(r * W, (r + 1) * W)
    spoil(rows, slice(None))
    got = run()
    assert torch.isnan(got[r, 3:]).all()
    got[r, 3:] = base[r, 3:]
    assert torch.equal(got, base)
    assert torch.isnan(run(w=3)[r, 3:]).all()
    out_of_pool = table.clone()
    out_of_pool[r, 0] = -1  # some left out: still NaN where others are left
    assert torch.isnan(run(out_of_pool)[r, 3:]).all() == (lens[r] > ps)
    out_of_pool[r] = R * W
    assert not run(out_of_pool)[r].any()
    # one finite key
    at = lens[r] // 2
    page, place = r * W + at // ps, at % ps
    if q8:
        kd[page, place, 1, 0] = 0.01
        value = vc[page, place, 1].float() * vd[page, place, 1, 0].float()
    else:
        kc[page, place, 1, 3] = 1.0
        value = vc[page, place, 1].float()
    # (its weight is 1: quotient and products exact, but for a Q8_0 value's scale in two or three parts)
    assert torch.allclose(run()[r, 3:], value.expand(3, D), rtol=2.0**-16, atol=0)
    if teams:
        p.close()


@pytest.mark.parametrize("dt,q8", FORMS)
@pytest.mark.parametrize("D,ps", ((64, 16), (128, 64), (128, 1)))
@pytest.mark.parametrize("window", (1, 31, 100, 1000))
@pytest.mark.parametrize("freed", ("bad", "foreign"))
def test_nothing_before_a_window_is_used(prims, dt, q8, D, ps, window, freed):
    """pages behind a sliding window have gone: what the window's first page holds before it is NaN, table entries
    before it are outside the pool or pages of NaN; every request equals one of the window's own keys alone"""
    import torch
    rng = np.random.default_rng(D + ps + window)
    lens = [0, 1, window, window + 1, window + 17, 333, 2077]
    R, W = len(lens), 2077 // ps + 2
    kept = [(max(0, n - window), n) for n in lens]
    pages = [list(range(lo // ps, -(-n // ps))) for lo, n in kept]
    N = sum(map(len, pages)) + 1  # the last one is nobody's
    perm = rng.permutation(N - 1)
    table = rng.integers(N, 2 * N, (R, W)) if freed == "bad" else np.full((R, W), N - 1)
    used = np.zeros((N, ps), bool)
    at = 0
    for r, (lo, n) in enumerate(kept):
        for pg in pages[r]:
            table[r, pg] = perm[at]
            j = np.arange(pg * ps, (pg + 1) * ps)
            used[perm[at]] = (j >= lo) & (j < n)
            at += 1
    caches, plain = [], []
    for _ in range(2):
        c, d, x = random_values(rng, (N, ps, 1, D), dt, q8)
        (d if q8 else c)[torch.from_numpy(~used).to(DEV)] = float("nan")
        caches.append((c, d))
        plain.append(x)
    q = rng.standard_normal((R, 3, D))
    dq = to_dev(O.from_f64(q, dt), dt)
    (kc, kd), (vc, vd) = caches
    got = prims.attn_decode_paged(dq, kc, vc, i32(table), i32(lens), 0.1, window, kd, vd).double().cpu().numpy()
    qf = dq.double().cpu().numpy()
    for r, (lo, n) in enumerate(kept):
        j = np.arange(lo, n)
        K, V = (x[table[r, j // ps], j % ps] for x in plain)  # [keys, 1, D]
        ref, bound = PO.attn_decode(qf[r:r + 1], K[:, None], V[:, None], np.arange(len(j))[None], [len(j)], 1, 0, 0.1)
        assert np.all(np.abs(got[r] - ref[0]) <= bound[0]), r


@pytest.mark.parametrize("q8", (False, True))
@pytest.mark.parametrize("T", (1, 5, 70))
def test_append_without_query_heads(prims, q8, T):
    """k and v alone: as with q heads beside them"""
    import torch
    g = torch.Generator(device=DEV).manual_seed(T)
    k, v = (torch.randn((T, 3, 128), generator=g, device=DEV).bfloat16() for _ in range(2))
    slots = torch.randperm(80, generator=g, device=DEV)[:T]
    res = []
    for heads in (0, 2):
        q, kk = torch.ones((T, heads, 128), dtype=torch.bfloat16, device=DEV), k.clone()
        kc, vc = (torch.zeros((10, 8, 3, 128), dtype=torch.int8 if q8 else torch.bfloat16, device=DEV) for _ in range(2))
        kd, vd = (torch.zeros((10, 8, 3, 4), dtype=torch.float16, device=DEV) if q8 else None for _ in range(2))
        prims.qk_norm_rope_paged(q, kk, v, 1e-6, 1.0, None, None, slots, slots, kc, vc, kd, vd)
        res.append([t for t in (kk, kc, vc, kd, vd) if t is not None])
    assert all(torch.equal(a, b) for a, b in zip(*res)) and res[0][1].any()


@pytest.mark.parametrize("dt,q8", FORMS)
@pytest.mark.parametrize("nq,nkv,ps,window,scaling", ((17, 1, 16, 0, 0.088), (46, 2, 16, 2**40, -0.088), (4, 2, 1 << 20, 70, 0.0)))
def test_decode_corners(prims, dt, q8, nq, nkv, ps, window, scaling):
    """groups of 17 and 23 query heads, scalings of zero and below, windows past 32 bits, the largest pages"""
    rng = np.random.default_rng(nq)
    lens, D = [0, 130, 33, 1], 64
    N, W = (4, 1) if ps > 1000 else (40, 9)
    if ps > 1000:  # (the first 160 keys of each page are filled, and are all that the oracle sees)
        import torch
        shape = (N, ps, nkv, D)
        c = [torch.zeros(shape, dtype=torch.int8 if q8 else torch.bfloat16 if dt == BF16 else torch.float16, device=DEV)
             for _ in range(2)]
        d = [torch.zeros((*shape[:3], D // 32), dtype=torch.float16, device=DEV) if q8 else None for _ in range(2)]
        plain = []
        for cc, dd in zip(c, d):
            x, s, vals = random_values(rng, (N, 160, nkv, D), dt, q8)
            cc[:, :160] = x
            if q8:
                dd[:, :160] = s
            plain.append(vals)
        (kc, vc), (kd, vd), (K, V) = c, d, plain
    else:
        (kc, kd, K), (vc, vd, V) = (random_values(rng, (N, ps, nkv, D), dt, q8) for _ in range(2))
    table = np.stack([rng.permutation(N)[:W] for _ in lens])
    q = rng.standard_normal((len(lens), nq, D))
    dq = to_dev(O.from_f64(q, dt), dt)
    got = prims.attn_decode_paged(dq, kc, vc, i32(table), i32(lens), scaling, window, kd, vd).double().cpu().numpy()
    # (the oracle's bound takes a scaling's magnitude: the sign goes into q)
    qf = dq.double().cpu().numpy() * (-1.0 if scaling < 0 else 1.0)
    ref, bound = PO.attn_decode(qf, K, V, table, lens, min(ps, 160), window, abs(scaling))
    assert np.all(np.abs(got - ref) <= bound)
