"""GPU: MXFP4 products at the sizes where they are divided otherwise: large and
small tiles, rows' sums in parts, little or no workspace, scales at odd
addresses, captured, on another stream, and beside another context's. Operands
are whole numbers whose sums f32 holds in any order, so every output is exact;
the bounded ones are gated as tests/mxfp4_oracle.py counts."""
import numpy as np
import pytest

import mxfp4_oracle as MO

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def whole(seed, rows, n, unit=128):
    """codes of 0, 1, .. 12 at scale 2 (in units of a half, their values are whole), some blocks of scale 1, and their
    values in f64"""
    import torch
    g = torch.Generator(device=DEV).manual_seed(seed)
    qs = torch.randint(0, 256, (rows, n // 2), generator=g, device=DEV, dtype=torch.uint8)
    s = torch.randint(unit, unit + 2, (rows, n // 32), generator=g, device=DEV, dtype=torch.uint8)
    return qs, s, values(qs, s)


def values(qs, s):
    import torch
    grid = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, -0., -.5, -1, -1.5, -2, -3, -4, -6], dtype=torch.float64, device=DEV)
    v = grid[torch.stack((qs & 15, qs >> 4), -1).flatten(1).int()]
    return v * torch.exp2(s.double() - 127).repeat_interleave(32, 1)


def padded(rows, cols, dtype, pad=0):
    import torch
    return torch.full((rows, cols + pad), 7.0, dtype=dtype, device=DEV)


# (sums of at most 144 * 4 * 19968 < 2^24 are whole numbers that f32 holds, exact in any order)
TILES = ((300, 25600, 512), (257, 20000, 1056),     # large tiles, one part; a row's last piece ragged
         (513, 5120, 19968), (1024, 5120, 19968),   # .. in parts
         (600, 9000, 4000),
         (130, 300, 19968), (65, 1000, 19936),      # small tiles in up to eight parts, the last one shorter
         (500, 5120, 5120), (129, 129, 1024))


@pytest.mark.parametrize("T,rows,n", TILES)
def test_tiles(prims, T, rows, n):
    import torch
    aq, as_, A = whole(1, T, n)
    qs, s, W = whole(2, rows, n)
    ref = A @ W.t().contiguous()
    y = padded(T, rows, torch.float32, 3)
    prims.gemm_mxfp4(aq, as_, qs, s, y[:, :rows])
    assert torch.equal(y[:, :rows].double(), ref) and bool((y[:, rows:] == 7).all())
    z = padded(T, rows, torch.bfloat16, 8)
    prims.gemm_mxfp4(aq, as_, qs, s, z[:, :rows])
    assert torch.equal(z[:, :rows], ref.float().bfloat16()) and bool((z[:, rows:] == 7).all())


@pytest.mark.parametrize("T", (32, 100, 128))
@pytest.mark.parametrize("rows,n", ((512, 19968), (1000, 2048), (5120, 4000)))
def test_waves_of_more_tokens(prims, T, rows, n):
    """small weights: passes of 16 tokens over them, and the tiles past that"""
    import torch
    aq, as_, A = whole(3, T, n)
    qs, s, W = whole(4, rows, n)
    y = padded(T, rows, torch.float32)
    prims.gemm_mxfp4(aq, as_, qs, s, y)
    assert torch.equal(y.double(), A @ W.t().contiguous())


@pytest.mark.parametrize("dtype", ("bfloat16", "float16"))
@pytest.mark.parametrize("B", (1, 4, 5, 17, 40, 64))
@pytest.mark.parametrize("rows,n", ((6656, 19968), (300, 19936), (33000, 96), (1000, 2560)))
def test_gemv_parts(prims, dtype, B, rows, n):
    """rows' sums in parts and in one, the last part shorter, and of fewer steps than parts"""
    import torch
    g = torch.Generator(device=DEV).manual_seed(B)
    qs, s, W = whole(5, rows, n, 127)  # (halves up to 12)
    x = torch.randint(-5, 6, (B, n), generator=g, device=DEV).to(getattr(torch, dtype))
    ref = x.double() @ W.t().contiguous()
    y = padded(B, rows, torch.float32, 1)
    prims.gemv_mxfp4(qs, s, x, y[:, :rows])
    assert torch.equal(y[:, :rows].double(), ref) and bool((y[:, rows:] == 7).all())
    z = padded(B, rows, x.dtype, 3)
    prims.gemv_mxfp4(qs, s, x, z[:, :rows])
    assert torch.equal(z[:, :rows], ref.float().to(x.dtype)) and bool((z[:, rows:] == 7).all())


def at_odd(t):
    """the same bytes, three bytes past a 16-byte boundary"""
    import torch
    flat = torch.empty(t.numel() + 16, dtype=torch.uint8, device=DEV)
    v = flat[3:3 + t.numel()].view(t.shape)
    v.copy_(t)
    return v


@pytest.mark.parametrize("T,rows,n", ((5, 700, 4096), (300, 25600, 512), (513, 5120, 4096), (200, 300, 19968)))
def test_scales_anywhere(prims, T, rows, n):
    """scales are bytes: they may lie at any address; the same bits come out"""
    import torch
    aq, as_, A = whole(6, T, n)
    qs, s, W = whole(7, rows, n)
    y, z = padded(T, rows, torch.float32), padded(T, rows, torch.float32)
    prims.gemm_mxfp4(aq, as_, qs, s, y)
    prims.gemm_mxfp4(aq, at_odd(as_), qs, at_odd(s), z)
    assert torch.equal(y.double(), A @ W.t().contiguous()) and torch.equal(y, z)
    x = A[:min(T, 64)].bfloat16()  # (whole numbers below 2^8)
    u, v = padded(len(x), rows, torch.float32), padded(len(x), rows, torch.float32)
    prims.gemv_mxfp4(qs, s, x, u)
    prims.gemv_mxfp4(qs, at_odd(s), x, v)
    assert torch.equal(u, y[:len(x)]) and torch.equal(u, v)


@pytest.mark.parametrize("room", (64, 100 << 10, 3 << 20))
def test_little_workspace(prims, room):
    """parts and laid-out scales take what workspace there is, and none if it holds none of it"""
    import torch
    import mgprims
    p = mgprims.Prims(0, workspace_bytes=room)
    try:
        for T, rows, n in ((130, 300, 19968), (200, 700, 1056), (600, 3000, 8224)):
            aq, as_, A = whole(8, T, n)
            qs, s, W = whole(9, rows, n)
            y = padded(T, rows, torch.float32)
            p.gemm_mxfp4(aq, as_, qs, s, y)
            assert torch.equal(y.double(), A @ W.t().contiguous()), (T, rows, n)
            x = A[:40].half()
            z = padded(40, rows, torch.float32)
            p.gemv_mxfp4(qs, s, x, z)
            assert torch.equal(z, y[:40]), (T, rows, n)
        torch.cuda.synchronize()
    finally:
        p.close()


def test_more_tokens_than_a_launch_takes():
    """without room for laid-out scales, past 65535 passes of 16 tokens"""
    import torch
    import mgprims
    T, rows, n = 65535 * 16 + 37, 3, 32
    aq, as_, A = whole(13, T, n)
    qs, s, W = whole(14, rows, n)
    y = padded(T, rows, torch.float32)
    p = mgprims.Prims(0, workspace_bytes=64)
    try:
        p.gemm_mxfp4(aq, as_, qs, s, y)
        assert torch.equal(y.double(), A @ W.t().contiguous())
    finally:
        p.close()


def test_values_of_all_sizes(prims):
    """real activations and weights against their kept values, in large tiles, in parts, and of 16 bits"""
    import torch
    g = torch.Generator(device=DEV).manual_seed(3)
    for T, rows, n in ((333, 5120, 12800), (700, 8192, 2048)):
        w = torch.randn((rows, n), generator=g, device=DEV) * torch.rand((rows, 1), generator=g, device=DEV)
        x = torch.randn((T, n), generator=g, device=DEV)
        out = []
        for t in (w, x):
            qs, s = (torch.empty((t.shape[0], n // k), dtype=torch.uint8, device=DEV) for k in (2, 32))
            prims.quantize_mxfp4(t, qs, s)
            out += [qs, s]
        W, A = values(*out[:2]), values(*out[2:])
        y = padded(T, rows, torch.float32)
        prims.gemm_mxfp4(out[2], out[3], out[0], out[1], y)
        mag = A.abs() @ W.abs().t().contiguous()
        bound = (n / 64 + 25) * 2.0**-23
        assert bool(((y.double() - A @ W.t().contiguous()).abs() <= bound * mag).all())
        for x16 in (x[:48].bfloat16(), x[:64].half(), x[:3].half()):
            z = padded(len(x16), rows, torch.float32)
            prims.gemv_mxfp4(out[0], out[1], x16, z)
            ref, mag = x16.double() @ W.t().contiguous(), x16.double().abs() @ W.abs().t().contiguous()
            assert bool(((z.double() - ref).abs() <= bound * mag).all())


def test_captured_and_beside_others():
    """a captured graph of a quantizer and products in parts, replayed between eager calls of other sizes on the same
    context and while another context works on its own stream"""
    import torch
    import mgprims
    T, rows, n = 200, 1000, 19936  # (laid-out scales and parts in the workspace)
    W, V, B = whole(10, rows, n), whole(11, 700, 19968), whole(12, 300, 19968)
    x = torch.zeros((T, n), dtype=torch.bfloat16, device=DEV)
    xq, xs = torch.empty((T, n // 2), dtype=torch.uint8, device=DEV), torch.empty((T, n // 32), dtype=torch.uint8, device=DEV)
    y, z, v, eager = (padded(*size, torch.float32) for size in ((T, rows), (40, rows), (300, 700), (300, 700)))
    want = B[2] @ V[2].t().contiguous()
    main, side = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    p, other = (mgprims.Prims(0, stream=t.cuda_stream) for t in (main, side))

    def step():
        p.quantize_mxfp4(x, xq, xs)
        p.gemm_mxfp4(xq, xs, W[0], W[1], y)
        p.gemv_mxfp4(W[0], W[1], x[:40], z)

    try:
        with torch.cuda.stream(main):
            step()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=main):
            step()
        for i in range(4):
            X = torch.randint(-4, 5, (T, n), device=DEV, dtype=torch.int32).bfloat16()
            x.copy_(X)
            for t in (y, z, v, eager):
                t.zero_()
            torch.cuda.synchronize()
            other.gemm_mxfp4(B[0], B[1], V[0], V[1], v)
            with torch.cuda.stream(main):
                g.replay()
            p.gemm_mxfp4(B[0], B[1], V[0], V[1], eager)
            other.gemm_mxfp4(B[0], B[1], V[0], V[1], v)
            torch.cuda.synchronize()
            ref = X.double() @ W[2].t().contiguous()  # (values the format holds)
            assert torch.equal(y.double(), ref) and torch.equal(z.double(), ref[:40]), i
            assert torch.equal(v.double(), want) and torch.equal(eager.double(), want), i
    finally:
        p.close(), other.close()
