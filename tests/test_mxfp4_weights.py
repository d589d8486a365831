"""Decode attention over MXFP4 pages holds a weight in bf16 parts, three for f32
outputs: what that keeps of it. Two keys, the first with score 0 and value 0, the
second with the weight r = exp(-m scaling), m = 1 .. 256: an output is v r / (1 +
r). On the CPU: two parts miss the bound, three do not."""
import numpy as np
import pytest

import mxfp4_oracle as MO

U = 2.0**-24  # half a step of f32, relative
SCALING = float(np.float32(0.0054321))  # m scaling log2(e) < 2.01
# q k = -m is exact. log2 r: the scaling's and the product's rounding, 2 U of up to 2.01 each way, log 2 of it in r: 2.8 U;
# the exponential 2 U; the sum U, and at most half of r's errors through it; quotient and product U each; three products
# added in f32, 2 U each where an addition may truncate: 2.8 + 2 + 1 + 2.4 + 2 + 6 < 20. (A value's scale is a power of two.)
LIMIT = 20 * U


def in_parts(p, parts):
    """the sum of bf16 parts of p (f32), all but the last by truncation"""
    left, total = p.copy(), np.zeros(p.shape)
    for i in range(parts):
        b = left.view(np.uint32).astype(np.uint64)
        if i + 1 == parts:
            b = b + 0x7fff + (b >> 16 & 1)
        part = (b & 0xffff0000).astype(np.uint32).view(np.float32)
        total += part
        left = (left - part).astype(np.float32)
    return total


@pytest.mark.parametrize("parts,kept", ((2, False), (3, True)))
def test_what_parts_keep(parts, kept):
    r = np.exp(-np.arange(1, 257) * SCALING)
    err = np.abs(in_parts(r.astype(np.float32), parts) / r - 1)
    assert (err.max() <= U) if kept else (err.max() > 4 * LIMIT)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ("bfloat16", "float16"))
@pytest.mark.parametrize("nq,nkv,D", ((8, 2, 128), (8, 2, 64), (16, 1, 128), (4, 1, 64)))
@pytest.mark.parametrize("lo,hi", ((110, 128), (100, 150), (245, 253)))
def test_f32_outputs(prims, dtype, nq, nkv, D, lo, hi):
    """(V scales past 127 take the weights' other way)"""
    import torch
    from test_gpu_mxfp4_paged import attend, i32, u8
    R, ps = 256 // nq, 16
    rng = np.random.default_rng(D + nq)
    m = rng.permutation(256).reshape(R, nq) + 1
    q = np.zeros((R, nq, D))
    q[:, :, 5] = -m
    k = np.zeros((R, ps, nkv, D))
    k[:, 1, :, 5] = 1.0
    vq = rng.integers(0, 256, (R, ps, nkv, D // 2), dtype=np.uint8)
    vq[:, 0] = 0
    vs = rng.integers(lo, hi, (R, ps, nkv, D // 32)).astype(np.uint8)
    got = attend(prims, torch.from_numpy(q).to(getattr(torch, dtype)).to("cuda:0"), tuple(u8(x) for x in MO.quantize(k)),
                 (u8(vq), u8(vs)), i32(np.arange(R).reshape(R, 1)), i32([2] * R), SCALING).double().cpu().numpy()
    r = np.exp(-m * SCALING)[..., None]
    ref = np.repeat(MO.values(vq, vs)[:, 1], nq // nkv, 1) * r / (1 + r)
    assert np.all(np.abs(got - ref) <= LIMIT * np.abs(ref)), float(np.max(np.abs(got - ref) / np.maximum(np.abs(ref), 1e-300)) / U)
