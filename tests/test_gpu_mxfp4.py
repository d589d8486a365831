"""GPU: MXFP4 quantizer, dequantizer and products against 64-bit forms
(tests/mxfp4_oracle.py). Codes, scales and values are exact; products are gated
on the bound counted there, plus half a step of a 16-bit output, and are exact
where every partial sum is a whole number that f32 holds."""
import numpy as np
import pytest

import mxfp4_oracle as MO

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def dtypes():
    import torch
    return {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def u8(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a, np.uint8)).to(DEV)


def new(*shape, dtype=None, fill=0):
    import torch
    return torch.full(shape, fill, dtype=dtype or torch.uint8, device=DEV)


def half_step(dtype):
    """half a step of a stored value, relative (f32 sums are counted by the bound)"""
    return {"bf16": 2.0**-8, "f16": 2.0**-11, "f32": 0.0}[dtype]


def rows_of(seed, shape, dtype, spread=3.0):
    """rows of many sizes, blocks of zeros, ties and the format's ends, as stored values"""
    import torch
    r = np.random.default_rng(seed)
    x = r.standard_normal(shape) * np.exp(spread * r.standard_normal((shape[0], 1)))
    x[0, :32] = 0
    x[-1, -32:] = np.array([4, .25, .75, 1.25, 1.75, 2.5, 3.5, 5, 6, 7, -.25, -.75, -1.25, -1.75, -2.5, -3.5, -5, -7, 7.5,
                            3.99, 0.2, 0.3, -0.0, 0, 1, 2, 3, .5, -.5, -1, -2, 1.5])
    if shape[0] > 3:
        x[1, :32] = 1e-6 * np.arange(32)  # f16 subnormals
        x[2, -32:] = 3e38 if dtype != "f16" else 65504
    return torch.from_numpy(x.astype(np.float32)).to(dtypes()[dtype])


def same_codes(qs, s, x):
    """scales are equal, and codes wherever the block is not NaN (there they stand for nothing)"""
    wq, ws = MO.quantize(x.double().numpy())
    assert np.array_equal(s.cpu().numpy(), ws)
    live = np.repeat(ws != 255, 16, -1)
    assert np.array_equal(qs.cpu().numpy()[live], wq[live])


# -------------------------------------------------------------------- format
@pytest.mark.parametrize("dtype", ("bf16", "f16", "f32"))
@pytest.mark.parametrize("shape", ((1, 32), (5, 96), (33, 160), (7, 2048), (61, 19968), (1000, 32), (300, 4096)))
def test_quantize(prims, dtype, shape):
    x = rows_of(sum(shape), shape, dtype)
    qs, s = new(shape[0], shape[1] // 2, fill=0x77), new(shape[0], shape[1] // 32, fill=9)
    prims.quantize_mxfp4(x.to(DEV), qs, s)
    same_codes(qs, s, x)


@pytest.mark.parametrize("dtype", ("bf16", "f16", "f32"))
def test_quantize_strided_rows(prims, dtype):
    """rows of a wider buffer; what lies beside them changes nothing"""
    import torch
    x = rows_of(4, (19, 416), dtype)
    wide = torch.full((19, 480), float("nan"), dtype=x.dtype, device=DEV)
    wide[:, 32:448] = x.to(DEV)
    qs, s = new(19, 208), new(19, 13)
    prims.quantize_mxfp4(wide[:, 32:448], qs, s)
    same_codes(qs, s, x)


@pytest.mark.parametrize("dtype", ("bf16", "f16"))
def test_every_stored_value(prims, dtype):
    """every 16-bit pattern, as the largest of its block beside a grid of smaller ones"""
    import torch
    bits = np.arange(65536, dtype=np.uint16)
    x = torch.from_numpy(bits.view(np.int16)).view(dtypes()[dtype])
    big = x.double().numpy()
    fine = np.where(np.isfinite(big), big, 0.0)
    rel = np.concatenate(([1.0], np.linspace(-1.0, 1.0, 31)))
    rest = torch.from_numpy((fine[:, None] * rel).astype(np.float32)).to(dtypes()[dtype])
    rest[:, 0] = x
    qs, s = new(65536, 16), new(65536, 1)
    prims.quantize_mxfp4(rest.to(DEV), qs, s)
    same_codes(qs, s, rest)
    out = torch.empty((65536, 32), dtype=torch.float32, device=DEV)
    prims.dequant_mxfp4(qs, s, out)
    assert torch.equal(torch.isnan(out).all(1).cpu(), ~torch.isfinite(x))


@pytest.mark.parametrize("dtype", ("bf16", "f16", "f32"))
def test_dequantize_every_byte(prims, dtype):
    """every pair of codes at every scale: one rounding to the output's type, infinities and zeros where it
    ends, NaN at scale 255, the sign of zero kept"""
    import torch
    qs = np.tile(np.arange(256, dtype=np.uint8).reshape(1, 256), (256, 1))
    s = np.repeat(np.arange(256, dtype=np.uint8)[:, None], 16, 1)
    out = torch.full((256, 512), 7.0, dtype=dtypes()[dtype], device=DEV)
    prims.dequant_mxfp4(u8(qs), u8(s), out)
    want = torch.from_numpy(MO.values(qs, s)).to(torch.float32).to(dtypes()[dtype])
    got = out.cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    same = (got == want) & (torch.signbit(got) == torch.signbit(want))
    assert bool((same | torch.isnan(want)).all())


@pytest.mark.parametrize("dtype", ("bf16", "f16", "f32"))
@pytest.mark.parametrize("shape", ((1, 32), (3, 96), (17, 480), (128, 4096), (301, 2080)))
def test_dequantize(prims, dtype, shape):
    import torch
    r = np.random.default_rng(shape[1])
    qs = r.integers(0, 256, (shape[0], shape[1] // 2), dtype=np.uint8)
    s = r.integers(100, 150, (shape[0], shape[1] // 32), dtype=np.uint8)
    flat = torch.full((shape[0] * shape[1] + 64,), 7.0, dtype=dtypes()[dtype], device=DEV)
    out = flat[:shape[0] * shape[1]].view(shape)
    prims.dequant_mxfp4(u8(qs), u8(s), out)
    want = torch.from_numpy(MO.values(qs, s)).to(torch.float32).to(dtypes()[dtype])
    assert torch.equal(out.cpu(), want)
    assert bool((flat[shape[0] * shape[1]:] == 7).all())


def test_no_rows(prims):
    import torch
    for dtype in (torch.bfloat16, torch.float32):
        x = torch.empty((0, 64), dtype=dtype, device=DEV)
        prims.quantize_mxfp4(x, new(0, 32), new(0, 2))
        prims.dequant_mxfp4(new(0, 32), new(0, 2), x)
        prims.quantize_mxfp4(torch.empty((3, 0), dtype=dtype, device=DEV), new(3, 0), new(3, 0))


# ------------------------------------------------------------------ products
def weight(seed, rows, n, scales=(110, 130)):
    r = np.random.default_rng(seed)
    return (r.integers(0, 256, (rows, n // 2), dtype=np.uint8),
            r.integers(*scales, (rows, n // 32), dtype=np.uint8))


def gemv(prims, qs, s, x, out, pad=0):
    """x a CPU tensor; returns y of rows pad wider, and its padding"""
    import torch
    y = torch.full((x.shape[0], qs.shape[0] + pad), 7.0, dtype=dtypes()[out], device=DEV)
    prims.gemv_mxfp4(u8(qs), u8(s), x.to(DEV), y[:, :qs.shape[0]])
    assert bool((y[:, qs.shape[0]:] == 7).all())
    return y[:, :qs.shape[0]].double().cpu().numpy()


def check_product(got, w, x, out):
    ref, bound = MO.product(w, x)
    err = np.abs(got - ref)
    lim = bound + half_step(out) * (np.abs(ref) + bound) + (2.0**-25 if out == "f16" else 0.0)
    assert np.all(err <= lim), (float((err / np.maximum(lim, 1e-300)).max()), np.argwhere(err > lim)[:4].tolist())


@pytest.mark.parametrize("dtype", ("bf16", "f16"))
@pytest.mark.parametrize("B", (1, 2, 7, 16, 17, 32, 33, 48, 63, 64))
@pytest.mark.parametrize("rows,n", ((1, 32), (15, 96), (17, 128), (100, 672), (259, 2208), (1024, 5120)))
def test_gemv(prims, dtype, B, rows, n):
    import torch
    qs, s = weight(rows + n, rows, n)
    x = torch.from_numpy(np.random.default_rng(B).standard_normal((B, n)).astype(np.float32)).to(dtypes()[dtype])
    for out in ("f32", dtype):
        check_product(gemv(prims, qs, s, x, out, pad=3), MO.values(qs, s), x.double().numpy(), out)


@pytest.mark.parametrize("dtype", ("bf16", "f16"))
@pytest.mark.parametrize("rows,n,B", ((20000, 512, 1), (6656, 19968, 2), (25600, 1056, 5), (5120, 4096, 40)))
def test_gemv_large(prims, dtype, rows, n, B):
    import torch
    qs, s = weight(5, rows, n)
    x = torch.from_numpy(np.random.default_rng(6).standard_normal((B, n)).astype(np.float32)).to(dtypes()[dtype])
    check_product(gemv(prims, qs, s, x, "f32"), MO.values(qs, s), x.double().numpy(), "f32")


@pytest.mark.parametrize("dtype", ("bf16", "f16"))
@pytest.mark.parametrize("B", (1, 5, 20, 64))
@pytest.mark.parametrize("n", (32, 416, 4096))
def test_gemv_whole_numbers(prims, dtype, B, n):
    """codes and activations whose sums f32 holds in any order: every output exact"""
    import torch
    r = np.random.default_rng(n + B)
    qs, _ = weight(n, 70, n)
    s = np.full((70, n // 32), 128, np.uint8)  # values 0, 1, .. 12
    x = torch.from_numpy(r.integers(-9, 10, (B, n)).astype(np.float32)).to(dtypes()[dtype])
    assert np.array_equal(gemv(prims, qs, s, x, "f32"), x.double().numpy() @ MO.values(qs, s).T)


@pytest.mark.parametrize("dtype", ("bf16", "f16"))
@pytest.mark.parametrize("lo,hi", ((0, 1), (20, 30), (90, 106), (138, 146), (180, 190)))
def test_gemv_far_scales(prims, dtype, lo, hi):
    """weights past what 16 bits of either type hold, alone and beside ordinary ones; blocks of zeros at scale 0"""
    import torch
    for mixed in (False, True):
        qs, s = weight(lo, 40, 1024, (lo, hi))
        if mixed:
            s[:, 1::2] = 120
        qs[3, :16] = 0x80
        s[3, 0] = 0
        x = torch.from_numpy(np.random.default_rng(8).standard_normal((9, 1024)).astype(np.float32)).to(dtypes()[dtype])
        got = gemv(prims, qs, s, x, "f32")
        ref, bound = MO.product(MO.values(qs, s), x.double().numpy())
        # (a weight, a product or a sum below f32's smallest normal value loses bits or vanishes, 1024 of them)
        assert np.all(np.abs(got - ref) <= bound + 1024 * 2.0**-126 * (1 + float(x.abs().max())))


def test_gemv_f16_subnormals(prims):
    """f16 activations and weights below 2^-14 are not flushed"""
    import torch
    r = np.random.default_rng(2)
    qs, s = weight(9, 33, 256, (105, 112))
    x = torch.from_numpy((r.integers(-40, 41, (3, 256)) * 2.0**-24).astype(np.float32)).half()
    w = MO.values(qs, s)
    got = gemv(prims, qs, s, x, "f32")
    ref, bound = MO.product(w, x.double().numpy())
    assert np.all(np.abs(got - ref) <= bound) and np.abs(ref).max() > 0


@pytest.mark.parametrize("dtype", ("bf16", "f16"))
def test_gemv_not_finite(prims, dtype):
    """a NaN block makes its row NaN and no other; an infinite activation its own outputs; rows beside are as before"""
    import torch
    qs, s = weight(3, 50, 640)
    x = torch.from_numpy(np.random.default_rng(1).standard_normal((6, 640)).astype(np.float32)).to(dtypes()[dtype])
    base = gemv(prims, qs, s, x, "f32")
    s2 = s.copy()
    s2[7, 11] = 255
    got = gemv(prims, qs, s2, x, "f32")
    assert np.isnan(got[:, 7]).all()
    got[:, 7] = base[:, 7]
    assert np.array_equal(got, base)
    x2 = x.clone()
    x2[4, 100] = float("inf")
    got = gemv(prims, qs, s, x2, "f32")
    ref = np.where(MO.values(qs, s)[:, 100] == 0, np.nan, np.sign(MO.values(qs, s)[:, 100]) * np.inf)
    assert np.array_equal(got[4], ref, equal_nan=True)
    got[4] = base[4]
    assert np.array_equal(got, base)


def test_gemv_strides(prims):
    import torch
    qs, s = weight(3, 50, 640)
    x = torch.from_numpy(np.random.default_rng(1).standard_normal((20, 640)).astype(np.float32)).bfloat16().to(DEV)
    wide = torch.full((20, 704), float("nan"), dtype=x.dtype, device=DEV)
    wide[:, 8:648] = x
    y, z = (torch.empty((20, 50), device=DEV) for _ in range(2))
    prims.gemv_mxfp4(u8(qs), u8(s), x, y)
    prims.gemv_mxfp4(u8(qs), u8(s), wide[:, 8:648], z)
    assert torch.equal(y, z)


def gemm(prims, aq, as_, qs, s, out, pad=0):
    import torch
    y = torch.full((aq.shape[0], qs.shape[0] + pad), 7.0, dtype=dtypes()[out], device=DEV)
    prims.gemm_mxfp4(u8(aq), u8(as_), u8(qs), u8(s), y[:, :qs.shape[0]])
    assert bool((y[:, qs.shape[0]:] == 7).all())
    return y[:, :qs.shape[0]].double().cpu().numpy()


@pytest.mark.parametrize("T", (1, 7, 16, 17, 33, 64, 65, 127, 128, 129, 200, 333))
@pytest.mark.parametrize("rows,n", ((1, 32), (15, 96), (17, 128), (100, 672), (259, 2208), (513, 4096)))
def test_gemm(prims, T, rows, n):
    aq, as_ = weight(T, T, n, (118, 130))
    qs, s = weight(rows + n, rows, n)
    w, a = MO.values(qs, s), MO.values(aq, as_)
    for out in ("f32", "bf16"):
        check_product(gemm(prims, aq, as_, qs, s, out, pad=5), w, a, out)


@pytest.mark.parametrize("T,rows,n", ((1000, 1024, 1056), (513, 5120, 544), (300, 700, 19968), (4096, 259, 512)))
def test_gemm_large(prims, T, rows, n):
    aq, as_ = weight(T, T, n, (118, 126))
    qs, s = weight(rows + n, rows, n, (118, 124))
    for out in ("f32", "f16"):
        check_product(gemm(prims, aq, as_, qs, s, out), MO.values(qs, s), MO.values(aq, as_), out)


@pytest.mark.parametrize("T", (1, 20, 100, 300))
@pytest.mark.parametrize("n", (32, 416, 4096))
def test_gemm_whole_numbers(prims, T, n):
    """every output exact, each element of the operands in its place"""
    aq, _ = weight(T + 1, T, n)
    qs, _ = weight(n, 270, n)
    as_, s = np.full((T, n // 32), 128, np.uint8), np.full((270, n // 32), 128, np.uint8)
    assert np.array_equal(gemm(prims, aq, as_, qs, s, "f32"), MO.values(aq, as_) @ MO.values(qs, s).T)


@pytest.mark.parametrize("T", (3, 150))
def test_gemm_scales_and_nan(prims, T):
    """scales from end to end (their product in range), and NaN blocks of either operand"""
    n = 512
    aq, as_ = weight(1, T, n, (0, 20))
    qs, s = weight(2, 90, n, (235, 255))
    w, a = MO.values(qs, s), MO.values(aq, as_)
    check_product(gemm(prims, aq, as_, qs, s, "f32"), w, a, "f32")
    aq, as_ = weight(1, T, n)
    base = gemm(prims, aq, as_, qs * 0 + 0x22, s * 0 + 127, "f32")
    as2, s2 = as_.copy(), s * 0 + 127
    as2[2, 5] = 255
    s2[77, 15] = 255
    got = gemm(prims, aq, as2, qs * 0 + 0x22, s2, "f32")
    assert np.isnan(got[2]).all() and np.isnan(got[:, 77]).all()
    got[2], got[:, 77] = base[2], base[:, 77]
    assert np.array_equal(got, base)


def test_weights_activations_product(prims):
    """a weight and a prompt's activations quantized on the device, multiplied: the product of what was kept; the
    same rows one by one and through the 16-bit form of the kept activations agree with it"""
    import torch
    g = torch.Generator(device=DEV).manual_seed(1)
    w = (torch.randn((300, 1024), generator=g, device=DEV) / 32).bfloat16()
    x = torch.randn((70, 1024), generator=g, device=DEV).bfloat16()
    wq, ws, xq, xs = new(300, 512), new(300, 32), new(70, 512), new(70, 32)
    prims.quantize_mxfp4(w, wq, ws)
    prims.quantize_mxfp4(x, xq, xs)
    kept = torch.empty_like(x)
    prims.dequant_mxfp4(xq, xs, kept)
    y, one, z = (torch.empty((70, 300), device=DEV) for _ in range(3))
    prims.gemm_mxfp4(xq, xs, wq, ws, y)
    for t in range(70):
        prims.gemm_mxfp4(xq[t:t + 1], xs[t:t + 1], wq, ws, one[t:t + 1])
    for t in range(0, 70, 35):
        prims.gemv_mxfp4(wq, ws, kept[t:t + 35], z[t:t + 35])
    W, A = (MO.values(q.cpu().numpy(), s.cpu().numpy()) for q, s in ((wq, ws), (xq, xs)))
    for got in (y, one, z):
        check_product(got.double().cpu().numpy(), W, A, "f32")


def test_products_of_nothing(prims):
    import torch
    y = torch.full((2, 3), 7.0, device=DEV)
    prims.gemm_mxfp4(new(2, 0), new(2, 0), new(3, 0), new(3, 0), y)
    assert bool((y == 0).all())
    prims.gemm_mxfp4(new(0, 32), new(0, 2), new(3, 32), new(3, 2), y[:0])
    prims.gemm_mxfp4(new(2, 32), new(2, 2), new(0, 32), new(0, 2), y[:, :0])
    prims.gemv_mxfp4(new(0, 32), new(0, 2), torch.zeros((2, 64), dtype=torch.half, device=DEV), y[:, :0])
    y.fill_(7)
    prims.gemv_mxfp4(new(3, 0), new(3, 0), torch.zeros((2, 0), dtype=torch.half, device=DEV), y)
    assert bool((y == 0).all())


def test_errors(prims):
    import torch
    bf = torch.bfloat16
    x = torch.zeros((4, 64), dtype=bf, device=DEV)
    qs, s, y = new(6, 32), new(6, 2), torch.zeros((4, 6), device=DEV)
    for call, match in (
            (lambda: prims.quantize_mxfp4(x, new(4, 32), new(4, 1)), "scales"),
            (lambda: prims.quantize_mxfp4(x, new(4, 16), new(4, 1)), "expected"),
            (lambda: prims.quantize_mxfp4(x.double(), new(4, 32), new(4, 2)), "expected"),
            (lambda: prims.quantize_mxfp4(x.t(), new(64, 2), new(64, 1)), "32s"),
            (lambda: prims.quantize_mxfp4(torch.zeros((4, 72), dtype=bf, device=DEV)[:, 1:65], new(4, 32), new(4, 2)), "aligned"),
            (lambda: prims.quantize_mxfp4(torch.zeros((4, 66), dtype=bf, device=DEV)[:, :64], new(4, 32), new(4, 2)), "aligned"),
            (lambda: prims.dequant_mxfp4(qs, s, torch.zeros((6, 128), dtype=bf, device=DEV)[:, :64]), "contiguous"),
            (lambda: prims.dequant_mxfp4(qs.cpu(), s, y), "cpu"),
            (lambda: prims.gemv_mxfp4(qs, s, torch.zeros((65, 64), dtype=bf, device=DEV), torch.zeros((65, 6), device=DEV)), "64"),
            (lambda: prims.gemv_mxfp4(qs, s, x[:0], y[:0]), "64"),
            (lambda: prims.gemv_mxfp4(qs, s, x.float(), y), "bf16 or f16"),
            (lambda: prims.gemv_mxfp4(qs, s, x, y.half()), "dtype_out"),
            (lambda: prims.gemv_mxfp4(qs, s, x[:, :32], y), "expected"),
            (lambda: prims.gemv_mxfp4(qs, s, x[:1].expand(4, 64), y), "overlap"),
            (lambda: prims.gemv_mxfp4(qs, s, x, torch.zeros((6, 4), device=DEV).t()), "stride"),
            (lambda: prims.gemv_mxfp4(new(12, 32)[::2], s, x, y), "contiguous"),
            (lambda: prims.gemv_mxfp4(new(6 * 32 + 1)[1:].view(6, 32), s, x, y), "aligned"),
            (lambda: prims.gemm_mxfp4(new(4, 16), new(4, 1), qs, s, y), "differ"),
            (lambda: prims.gemm_mxfp4(new(4, 32), new(4, 2), qs, s, y[:3]), "expected"),
            (lambda: prims.gemm_mxfp4(new(4, 32).to(torch.int8), new(4, 2), qs, s, y), "uint8")):
        with pytest.raises(Exception, match=match):
            call()
