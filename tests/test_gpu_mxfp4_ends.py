"""GPU: MXFP4 products and decode attention at the ends of the format's scales,
where a code's value is a subnormal of bf16 (0 to 3) or passes it (253 and 254:
2^128 and above), against 64-bit forms (tests/mxfp4_oracle.py): values as any other."""
import numpy as np
import pytest

import mxfp4_oracle as MO
import paged_oracle as PO
from test_gpu_mxfp4 import DEV, dtypes, gemm, gemv, u8, weight
from test_gpu_mxfp4_paged import attend, i32

pytestmark = pytest.mark.gpu


def normal(seed, shape, scale, dtype):
    """values of the storage type, none below 2^-3 of scale in magnitude (their products stay f32 normals)"""
    import torch
    x = np.random.default_rng(seed).standard_normal(shape)
    x = np.where(np.abs(x) < 0.125, np.copysign(0.125, x), x) * scale
    return torch.from_numpy(x.astype(np.float32)).to(dtypes()[dtype])


@pytest.mark.parametrize("dtype", ("bf16", "f16"))
@pytest.mark.parametrize("B", (1, 3, 9, 40, 64))
@pytest.mark.parametrize("n", (64, 1024))
def test_gemv_smallest_scales(prims, dtype, B, n):
    """Weights of 2^-128 to 6 2^-124 count in full. Products with bf16 activations of 2^57 and more are normal numbers of
    f32; f16's reach 2^15, whose second parts' products are subnormals, off by half a step, 2^-150, each."""
    qs, s = weight(n, 40, n, (0, 4))
    x = normal(B, (B, n), 2.0**60 if dtype == "bf16" else 2.0**12, dtype)
    got = gemv(prims, qs, s, x, "f32")
    ref, bound = MO.product(MO.values(qs, s), x.double().numpy())
    slack = 0.0 if dtype == "bf16" else n * 2.0**-149
    assert slack <= 2.0**-16 * np.abs(ref).max()
    assert np.all(np.abs(got - ref) <= bound + slack), np.abs(got - ref).max() / np.abs(ref).max()


@pytest.mark.parametrize("dtype", ("bf16", "f16"))
@pytest.mark.parametrize("B", (1, 3, 9, 40, 64))
@pytest.mark.parametrize("n,lo,hi", ((64, 254, 255), (416, 253, 255), (1056, 250, 255), (2208, 188, 255), (9984, 251, 255)))
@pytest.mark.parametrize("mixed", (False, True))
def test_gemv_largest_scales(prims, dtype, B, n, lo, hi, mixed):
    """weights up to 6 2^127 and activations small enough that sums are finite; mixed: ordinary, smallest and zero blocks
    beside"""
    qs, s = weight(n + B, 70, n, (lo, hi))
    if mixed:
        s[:, 1::3] = 120
        s[::2, 0] = np.arange(35) % 3
        qs[3, :16] = 0x80
    x = normal(B, (B, n), 2.0**-15, dtype)
    got = gemv(prims, qs, s, x, "f32")
    ref, bound = MO.product(MO.values(qs, s), x.double().numpy())
    assert np.isfinite(ref).all() and np.all(np.abs(got - ref) <= bound), np.argwhere(~(np.abs(got - ref) <= bound))[:4].tolist()


@pytest.mark.parametrize("dtype", ("bf16", "f16"))
@pytest.mark.parametrize("B", (1, 4, 20))
def test_gemv_largest_scales_and_sums(prims, dtype, B):
    """sums past f32 are infinite with their sign, whatever the activations' second parts; an infinite activation makes its
    own outputs infinite, or NaN beside a zero; a NaN block its row"""
    import torch
    n = 640
    qs, s = np.full((50, n // 2), 0x77, np.uint8), np.full((50, n // 32), 252, np.uint8)  # 6 2^125
    s[::3] = 254
    s[7, 4] = 255
    qs[9] = 0xff  # negative
    x = torch.full((B, n), 60096.0, dtype=torch.float32).to(dtypes()[dtype])  # (f16: bf16's next value less 64)
    got = gemv(prims, qs, s, x, "f32")
    want = np.where(np.arange(50) == 9, -np.inf, np.inf) * np.ones((B, 1))
    want[:, 7] = np.nan
    assert np.array_equal(got, want, equal_nan=True)
    qs[20, :16] = 0  # 32 zeros
    x = normal(1, (B, n), 2.0**-15, dtype)
    x[B - 1, 5] = float("-inf")
    got = gemv(prims, qs, s, x, "f32")[B - 1]
    want = -want[0]
    want[20] = np.nan
    assert np.array_equal(got, want, equal_nan=True)


@pytest.mark.parametrize("T", (3, 40, 300))
def test_gemm_largest_scales(prims, T):
    """MXFP4 activations, down to 2^-128, beside weights up to 6 2^127"""
    aq, as_ = weight(T, T, 1056, (0, 110))
    qs, s = weight(7, 90, 1056, (250, 255))
    got = gemm(prims, aq, as_, qs, s, "f32")
    ref, bound = MO.product(MO.values(qs, s), MO.values(aq, as_))
    assert np.isfinite(ref).all() and np.all(np.abs(got - ref) <= bound)


@pytest.mark.parametrize("dtype", ("bf16", "f16"))
@pytest.mark.parametrize("nq,nkv,D", ((4, 2, 64), (10, 2, 128), (12, 1, 128), (3, 1, 64)))
@pytest.mark.parametrize("lo,hi", ((253, 255), (249, 255), (190, 194)))
def test_scores_of_largest_scales(prims, dtype, nq, nkv, D, lo, hi):
    """keys up to 6 2^127 beside ordinary, smallest and zero ones, queries and scaling such that scores stay within tens"""
    R, ps, W = 3, 16, 20
    lens = [300, 64, 1]
    rng = np.random.default_rng(lo + nq)
    kq = rng.integers(0, 256, (R * W, ps, nkv, D // 2), dtype=np.uint8)
    ks = rng.integers(lo, hi, (R * W, ps, nkv, D // 32)).astype(np.uint8)
    ks[::3, ::2] = rng.integers(100, 130, ks[::3, ::2].shape)
    ks[1::4, 3, :, 0] = rng.integers(0, 3, ks[1::4, 3, :, 0].shape)
    kq[2, 5] = 0x88
    vq, vs = MO.quantize(rng.standard_normal((R * W, ps, nkv, D)))
    q = normal(nq, (R, nq, D), 2.0**-15, dtype)
    scaling = 2.0**(127 - hi + 15 - 3)
    table = rng.permutation(R * W).reshape(R, W)
    got = attend(prims, q.to(DEV), (u8(kq), u8(ks)), (u8(vq), u8(vs)), i32(table), i32(lens), scaling).double().cpu().numpy()
    ref, bound = PO.attn_decode(q.double().numpy(), MO.values(kq, ks), MO.values(vq, vs), table, lens, ps, 0, scaling)
    assert np.isfinite(ref).all() and np.all(np.abs(got - ref) <= bound), np.argwhere(~(np.abs(got - ref) <= bound))[:4].tolist()


@pytest.mark.parametrize("dtype", ("bf16", "f16"))
@pytest.mark.parametrize("nq,nkv", ((2, 1), (4, 2), (12, 1)))
@pytest.mark.parametrize("size", (4.0, 60000.0))
@pytest.mark.parametrize("s", (252, 254))
def test_infinite_scores_of_either_type(prims, dtype, nq, nkv, size, s):
    """a key of score -inf weighs nothing beside another, also where the queries' second parts have the other sign; such
    keys alone give NaN; no key gives zeros"""
    import torch
    D, ps = 64, 16
    rng = np.random.default_rng(3)
    kq, ks = MO.quantize(rng.standard_normal((8, ps, nkv, D)) / size)
    vq, vs = MO.quantize(rng.standard_normal((8, ps, nkv, D)))
    kq[2, 3], ks[2, 3] = 0xff, s  # -6 2^(s - 127) in every dim: products' sums with q > 0 are past f32
    kq[4], ks[4] = 0xff, s
    q = (torch.rand((3, nq, D), generator=torch.Generator().manual_seed(4)) / 16 + 1).mul_(size).to(dtypes()[dtype])
    pools = ((u8(kq), u8(ks)), (u8(vq), u8(vs)))
    got = attend(prims, q.to(DEV), *pools, i32([[0, 1, 2, 3], [4, 4, 4, 4], [5, 6, 7, 0]]), i32([64, 40, 0]), 0.1)
    assert torch.isnan(got[1]).all() and not got[2].any()
    live = np.arange(64) != 35
    K, V = (MO.values(a, b)[:4].reshape(64, 1, nkv, D)[live] for a, b in ((kq, ks), (vq, vs)))
    ref, bound = PO.attn_decode(q[:1].double().numpy(), K, V, np.arange(63)[None], [63], 1, 0, 0.1)
    assert np.all(np.abs(got[:1].double().cpu().numpy() - ref) <= bound)


def test_more_than_a_launch_takes(prims):
    """threads past 2^32 along an axis are refused by name, before anything is launched"""
    import torch
    t = torch.zeros(4096, dtype=torch.uint8, device=DEV)
    p, L, h, bf = t.data_ptr(), prims.lib, prims.h, 1

    def refused(rc):
        return rc == -1 and (b"too large" in L.mg_last_error() or b"too many" in L.mg_last_error())

    for rows, n in ((2**31, 32), (2**26, 1024), (1, 2**36), (2**26 - 4, 1024 + 32)):
        assert refused(L.mg_quantize_mxfp4(h, p, 0, rows, n, bf, p, p)), (rows, n)
    for rows, n in ((2**30, 32), (2**25, 1024), (1, 2**35), (2**35 // 96 + 1, 96)):
        assert refused(L.mg_dequant_mxfp4(h, p, p, p, rows, n, bf)), (rows, n)
    for batch in (1, 3):
        assert refused(L.mg_gemv_mxfp4(h, p, p, p, batch, 2**28, 32, 0, p, 0, bf, bf))
    assert refused(L.mg_gemv_mxfp4(h, p, p, p, 64, 2**30, 32, 0, p, 0, bf, bf))
    assert refused(L.mg_gemm_mxfp4(h, p, p, 5, p, p, 2**28, 32, p, 0, bf))
    torch.cuda.synchronize()
    assert not t.any()
