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


@pytest.mark.parametrize("T", (3, 40, 300))
def test_gemm_largest_scales(prims, T):
    """MXFP4 activations, down to 2^-128, beside weights up to 6 2^127"""
    aq, as_ = weight(T, T, 1056, (0, 110))
    qs, s = weight(7, 90, 1056, (250, 255))
    got = gemm(prims, aq, as_, qs, s, "f32")
    ref, bound = MO.product(MO.values(qs, s), MO.values(aq, as_))
    assert np.isfinite(ref).all() and np.all(np.abs(got - ref) <= bound)
