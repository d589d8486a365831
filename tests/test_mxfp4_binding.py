"""CPU: what the binding refuses of the MXFP4 calls before the library is asked,
what it passes on, and the C ABI's refusals without a context."""
import ctypes

import pytest
import torch

import mgprims as M
from test_paged_binding import BF, Calls, Untouched, i32, i64

U8, F16 = torch.uint8, torch.float16


@pytest.fixture()
def P():
    p = M.Prims.__new__(M.Prims)
    p.h, p.device, p.lib = None, -1, Untouched()  # (get_device() of a CPU tensor is -1)
    p._i32, p._i64, p._i8, p._f16, p._u8 = torch.int32, torch.int64, torch.int8, F16, U8
    p._codes = {BF: M.BF16, F16: M.F16, torch.float32: M.F32}
    return p


def z(*s, d=U8):
    return torch.zeros(s, dtype=d)


# codes [6, 32], scales [6, 2] of rows of 64
CODES = (dict(qs=z(6, 32, d=torch.int8)), dict(s=z(6, 2, d=torch.int8)), dict(s=z(6, 2, d=F16)), dict(qs=z(6, 2, 16)),
         dict(qs=z(6, 24)), dict(s=z(6, 1)), dict(s=z(5, 2)), dict(s=z(12)), dict(qs=z(6, 64)[:, ::2]), dict(qs=z(12, 32)[::2]),
         dict(s=z(6, 4)[:, :2]), dict(qs=z(32, 6).t()), dict(s=z(2, 6).t()))


@pytest.mark.parametrize("bad", CODES + (
    dict(x=z(6, 64, d=torch.float64)), dict(x=z(6, 64, d=torch.int16)), dict(x=z(5, 64, d=BF)), dict(x=z(6, 32, d=BF)),
    dict(x=z(64, 6, d=BF).t()), dict(x=z(1, 64, d=BF).expand(6, 64)), dict(x=z(6, 1, 64, d=BF))))
def test_quantize_refusals(P, bad):
    a = {**dict(x=z(6, 64, d=BF), qs=z(6, 32), s=z(6, 2)), **bad}
    with pytest.raises(M.MgError):
        P.quantize_mxfp4(**a)


@pytest.mark.parametrize("bad", CODES + (dict(out=z(6, 96, d=BF)[:, :64]), dict(out=z(6, 64)), dict(out=z(6, 128, d=BF))))
def test_dequantize_refusals(P, bad):
    with pytest.raises(M.MgError):
        P.dequant_mxfp4(**{**dict(qs=z(6, 32), s=z(6, 2), out=z(6, 64, d=BF)), **bad})


@pytest.mark.parametrize("bad", CODES + (
    dict(x=z(3, 32, d=BF)), dict(x=z(64, d=BF)), dict(x=z(3, 64)), dict(x=z(1, 64, d=BF).expand(3, 64)), dict(x=z(64, 3, d=BF).t()),
    dict(y=z(3, 5, d=BF)), dict(y=z(2, 6, d=BF)), dict(y=z(6, 3, d=BF).t()), dict(y=z(3, 6, d=torch.float64)),
    dict(y=z(1, 6, d=BF).expand(3, 6))))
def test_gemv_refusals(P, bad):
    with pytest.raises(M.MgError):
        P.gemv_mxfp4(**{**dict(qs=z(6, 32), s=z(6, 2), x=z(3, 64, d=BF), y=z(3, 6, d=BF)), **bad})


@pytest.mark.parametrize("bad", CODES + (
    dict(a_qs=z(3, 16), a_s=z(3, 1)), dict(a_qs=z(3, 32, d=torch.int8)), dict(a_s=z(4, 2)), dict(a_qs=z(6, 32)[::2]),
    dict(y=z(6, 3, d=BF)), dict(y=z(3, 6)), dict(y=z(3, 12, d=BF)[:, ::2])))
def test_gemm_refusals(P, bad):
    with pytest.raises(M.MgError):
        P.gemm_mxfp4(**{**dict(a_qs=z(3, 32), a_s=z(3, 2), qs=z(6, 32), s=z(6, 2), y=z(3, 6, d=BF)), **bad})


POOLS = (dict(k_scale=None), dict(v_scale=None), dict(k_scale=None, v_scale=None), dict(k_scale=z(4, 8, 2, 2, d=F16)),
         dict(v_scale=z(4, 8, 2, 1)), dict(v_scale=z(4, 8, 2, 4)[..., :2]), dict(k_cache=z(4, 8, 2, 64)), dict(v_cache=z(3, 8, 2, 32)),
         dict(v_cache=z(4, 8, 2, 32, d=torch.int8)), dict(k_cache=z(4, 8, 2, 32, d=torch.int8)), dict(k_cache=z(4, 16, 32)),
         dict(k_cache=z(4, 2, 8, 32).transpose(1, 2), v_cache=z(4, 2, 8, 32).transpose(1, 2)))


def pool(**k):
    return {**dict(k_cache=z(4, 8, 2, 32), v_cache=z(4, 8, 2, 32), k_scale=z(4, 8, 2, 2), v_scale=z(4, 8, 2, 2)), **k}


@pytest.mark.parametrize("bad", POOLS + (dict(k=z(3, 3, 64, d=BF), v=z(3, 3, 64, d=BF)),
                                         dict(q=z(3, 4, 48, d=BF), k=z(3, 2, 48, d=BF), v=z(3, 2, 48, d=BF))))
def test_append_refusals(P, bad):
    a = dict(q=z(3, 4, 64, d=BF), k=z(3, 2, 64, d=BF), v=z(3, 2, 64, d=BF), eps=1e-6, qk_scale=1.0, cos=None, sin=None,
             positions=i64(0, 1, 2), slot_map=i64(0, 1, 2), **pool())
    with pytest.raises(M.MgError):
        P.qk_norm_rope_paged(**{**a, **bad})


@pytest.mark.parametrize("bad", POOLS + (dict(q=z(2, 4, 128, d=BF)), dict(lens=i32(1)), dict(out=z(2, 4, 64))))
def test_decode_refusals(P, bad):
    a = dict(q=z(2, 4, 64, d=BF), page_table=z(2, 3, d=torch.int32), lens=i32(1, 2), scaling=0.1, out=z(2, 4, 64, d=BF), **pool())
    with pytest.raises(M.MgError):
        P.attn_decode_paged(**{**a, **bad})


def test_what_is_taken(P):
    """row strides, types, and uint8 pools to their own entry points"""
    P.lib = Calls()
    P.quantize_mxfp4(z(6, 96, d=F16)[:, :64], z(6, 32), z(6, 2))
    name, a = P.lib.args
    assert name == "mg_quantize_mxfp4" and a[2:6] == (96, 6, 64, M.F16)
    P.quantize_mxfp4(z(1, 64, d=BF).expand(1, 64), z(1, 32), z(1, 2))
    assert P.lib.args[1][2] == 64
    P.dequant_mxfp4(z(6, 32), z(6, 2), z(6, 64, d=torch.float32))
    assert P.lib.args[1][4:] == (6, 64, M.F32)
    P.gemv_mxfp4(z(6, 32), z(6, 2), z(3, 72, d=BF)[:, :64], z(3, 9, d=torch.float32)[:, :6])
    name, a = P.lib.args
    assert name == "mg_gemv_mxfp4" and a[4:8] == (3, 6, 64, 72) and a[9:] == (9, M.BF16, M.F32)
    P.gemm_mxfp4(z(3, 32), z(3, 2), z(6, 32), z(6, 2), z(3, 8, d=F16)[:, :6])
    name, a = P.lib.args
    assert name == "mg_gemm_mxfp4" and a[3] == 3 and a[6:8] == (6, 64) and a[9:] == (8, M.F16)
    P.attn_decode_paged(q=z(2, 4, 64, d=BF), page_table=z(2, 3, d=torch.int32), lens=i32(1, 2), scaling=0.1, **pool())
    assert P.lib.args[0] == "mg_attn_decode_paged_mxfp4"
    P.qk_norm_rope_paged(q=z(3, 4, 64, d=BF), k=z(3, 2, 64, d=BF), v=z(3, 2, 64, d=BF), eps=1e-6, qk_scale=1.0, cos=None,
                         sin=None, positions=i64(0, 1, 2), slot_map=i64(0, 1, 2), **pool())
    assert P.lib.args[0] == "mg_qk_norm_rope_paged_mxfp4" and P.lib.args[1][-2] == 32


def test_abi_without_a_context():
    L = M.load_library()
    for name in M._SIGS:
        if "mxfp4" in name:
            args = [0.0 if t is ctypes.c_double else None if t is ctypes.c_void_p else 0 for t in M._SIGS[name][0]]
            assert getattr(L, name)(*args) == -1
            assert b"NULL context" in L.mg_last_error()
