"""GPU: decode attention over MXFP4 pages where its kernel takes another way: two
kv heads a wave or one, pages below a load's keys and above, references that lag
behind rising scores beside V scales past 127, NaN blocks of every head. Gated as
in test_gpu_mxfp4_paged.py."""
import numpy as np
import pytest

import mxfp4_oracle as MO
import paged_oracle as PO
from test_gpu_mxfp4_paged import DTS, attend, decode_case, i32, u8
from util import BF16, F16

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


# pairs of heads with one to eight queries each; odd numbers of heads; more than eight queries; groups in two
@pytest.mark.parametrize("nq,nkv", ((6, 6), (16, 2), (14, 2), (18, 2), (9, 3), (24, 1), (64, 2), (36, 4)))
@pytest.mark.parametrize("D", (64, 128))
@pytest.mark.parametrize("ps", (2, 4, 8, 16, 128))
def test_ways(prims, nq, nkv, D, ps):
    rng = np.random.default_rng(nq + ps)
    lens = [700, 0, 31, 32, 33, 127, 128, 129, 1, *rng.integers(0, 600, 20).tolist()]
    decode_case(prims, lens, nq, nkv, D, ps, seed=nq + D)
    decode_case(prims, lens, nq, nkv, D, ps, F16, out="same", window=97, seed=nq + D)


@pytest.mark.parametrize("nq,nkv", ((40, 8), (32, 2)))
def test_runs_over_many_requests(prims, nq, nkv):
    """runs that cross several requests, whose waves end in turn: more work than a work-group a CU"""
    rng = np.random.default_rng(1)
    decode_case(prims, rng.integers(0, 1200, 300).tolist(), nq, nkv, 64, 16)


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("nq,nkv", ((4, 2), (12, 1)))
@pytest.mark.parametrize("step", (0.01, 0.11, 3.0, -0.11))
def test_rising_scores_and_large_values(prims, dt, nq, nkv, step):
    """a score a key of step * its place (in log 2 units), so that references move at every step, now and then, or once;
    V scales below 128 in some stretches of keys, past it in others, up to 2^110 of 6. q and k are zero but for two
    dims of exact products (a place's 16s and its rest), so a score s is off by the roundings of the scaling and of
    its product, 2 U |s|, and the reference's, up to 2^-23 |s| more, each relative log 2 of its weight; exponential and
    quotient 8 U; a weight's parts 2^-16; its sum (n / 32 + 128) U."""
    import torch
    U, D, ps, n = 2.0**-24, 128, 16, 1500
    rng = np.random.default_rng(5)
    W = -(-n // ps)
    table = rng.permutation(W).reshape(1, W)
    # places up to 1535 = 96 * 16 + rest, as sums of what a code holds
    place = np.arange(W * ps)
    k = np.zeros((W * ps, nkv, D))
    k[:, :, 0] = (place // 256)[:, None] % 8      # 0 .. 5 (5 as 4 + 1 below)
    k[:, :, 32] = (place // 64 % 4)[:, None]
    k[:, :, 64] = (place // 16 % 4)[:, None]
    k[:, :, 96] = (place // 4 % 4)[:, None]
    k[:, :, 97] = (place % 4)[:, None]
    k[:, :, 1] = np.where(k[:, :, 0] == 5, 1, 0)
    k[:, :, 0] = np.where(k[:, :, 0] == 5, 4, k[:, :, 0])
    kq, ks = MO.quantize(k)
    assert np.array_equal(MO.values(kq, ks), k)
    q = np.zeros((1, nq, D))
    q[:, :, [0, 1]], q[:, :, 32], q[:, :, 64], q[:, :, 96], q[:, :, 97] = 256, 64, 16, 4, 1
    scaling = float(np.float32(step * np.log(2)))
    vq = rng.integers(0, 256, (W * ps, nkv, D // 2), dtype=np.uint8)
    vs = rng.integers(100, 120, (W * ps, nkv, D // 32), dtype=np.uint8)
    vs[300:420] = rng.integers(120, 238, vs[300:420].shape)
    vs[1100:1101, :, 1:] = 237
    pools = []
    for codes, s in ((kq, ks), (vq, vs)):
        dst = [np.zeros((W, ps, nkv, x.shape[-1]), np.uint8) for x in (codes, s)]
        for d, x in zip(dst, (codes, s)):
            d[table[0]] = x.reshape(W, ps, nkv, -1)
        pools.append(tuple(u8(d) for d in dst))
    kind = {BF16: torch.bfloat16, F16: torch.float16}[dt]
    out = torch.empty((1, nq, D), dtype=torch.float32, device=DEV)
    attend(prims, torch.from_numpy(q).to(kind).to(DEV), *pools, i32(table), i32([n]), scaling, out=out)
    got = out.double().cpu().numpy()[0]
    V = MO.values(vq, vs)[:n]
    s = scaling * place[:n]
    p = np.exp(s - s.max())
    p /= p.sum()
    for h in range(nq):
        v = V[:, h // (nq // nkv)]
        # a weight's error goes by its own score and by that of the reference, at most the largest in magnitude
        rel = 6 * U * np.abs(s).max() + 16 * U + 2.0**-16 + (n / 32 + 128) * U
        lim = rel * (p @ np.abs(v)) + 2.0**-126 * n * 8
        # (weights times scales below 2^-118 of the largest weight keep less of themselves: 2^-110 of a code at least)
        lim += 6 * n * 2.0**-110
        assert np.all(np.abs(got[h] - p @ v) <= lim), (h, np.abs(got[h] - p @ v).max())


@pytest.mark.parametrize("nq,nkv,D", ((6, 2, 64), (16, 2, 128), (5, 1, 64), (24, 1, 128), (6, 3, 64)))
def test_nan_blocks(prims, nq, nkv, D):
    """a V block's NaN reaches its 32 dims of its head's queries, whichever head and block, and a K block's all of them"""
    import torch
    n, ps = 150, 16
    rng = np.random.default_rng(D + nq)
    q = torch.randn((1, nq, D), generator=torch.Generator().manual_seed(1)).bfloat16().to(DEV)
    table, lens = i32(np.arange(10).reshape(1, 10)), i32([n])
    pools = [[u8(x) for x in MO.quantize(rng.standard_normal((10, ps, nkv, D)))] for _ in range(2)]
    base = attend(prims, q, *pools, table, lens, 0.1)
    per = nq // nkv
    for g in range(nkv):
        for b in range(D // 32):
            for which, at in ((0, 77), (1, 0), (1, 149)):
                keep = pools[which][1].clone()
                pools[which][1][at // ps, at % ps, g, b] = 255
                got = attend(prims, q, *pools, table, lens, 0.1)
                pools[which][1].copy_(keep)
                want = base.clone()
                want[:, per * g:per * (g + 1), slice(None) if which == 0 else slice(32 * b, 32 * b + 32)] = float("nan")
                assert torch.equal(torch.isnan(got), torch.isnan(want))
                assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(want))


@pytest.mark.parametrize("nq,nkv", ((8, 2), (16, 1)))
def test_queries_that_are_not_finite(prims, nq, nkv):
    """a head whose query holds an infinity or a NaN gives NaN (also at a scaling of zero), the others what they gave"""
    import torch
    rng = np.random.default_rng(7)
    pools = [[u8(x) for x in MO.quantize(rng.standard_normal((8, 16, nkv, 64)))] for _ in range(2)]
    table, lens = i32([[0, 1, 2, 3], [4, 5, 6, 7]]), i32([60, 64])
    q = torch.randn((2, nq, 64), generator=torch.Generator().manual_seed(3)).bfloat16().to(DEV)
    for scaling in (0.1, 0.0, -0.3):
        base = attend(prims, q, *pools, table, lens, scaling)
        assert torch.isfinite(base).all()
        for value in (float("inf"), float("nan")):
            r = q.clone()
            r[1, 3, 40] = value
            got = attend(prims, r, *pools, table, lens, scaling)
            assert torch.isnan(got[1, 3]).all()
            got[1, 3] = base[1, 3]
            assert torch.equal(got, base)
