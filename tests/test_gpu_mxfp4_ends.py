"""GPU: MXFP4 products at the ends of the format's scales, where a code's value is
a subnormal of bf16 (0 to 3) or passes it (253 and 254: 2^128 and above), against
64-bit forms (tests/mxfp4_oracle.py)."""
import numpy as np
import pytest

import mxfp4_oracle as MO
from test_gpu_mxfp4 import dtypes, gemm, gemv, weight

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
