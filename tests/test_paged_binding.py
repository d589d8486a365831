"""CPU: what the binding refuses of the paged KV cache's calls, before the
library is asked: a stand-in library fails the test when it is called, CPU
tensors stand in for a device's. And the C ABI without a context."""
import ctypes

import pytest
import torch

import mgprims as M


class Untouched:
    def __getattr__(self, name):
        def call(*_):
            pytest.fail(f"{name} was called")
        return call


class Calls:
    """takes every call and remembers its arguments"""

    def __init__(self):
        self.args = None

    def __getattr__(self, name):
        def call(*a):
            self.args = (name, a)
            return 0
        return call


@pytest.fixture()
def P():
    p = M.Prims.__new__(M.Prims)
    p.h, p.device, p.lib = None, -1, Untouched()  # (get_device() of a CPU tensor is -1)
    p._i32, p._i64, p._i8, p._f16 = torch.int32, torch.int64, torch.int8, torch.float16
    p._codes = {torch.bfloat16: M.BF16, torch.float16: M.F16, torch.float32: M.F32}
    return p


def i32(*v):
    return torch.tensor(v, dtype=torch.int32)


def i64(*v):
    return torch.tensor(v, dtype=torch.int64)


BF = torch.bfloat16


def pages_args(**k):
    return {**dict(page_table=torch.zeros((2, 3), dtype=torch.int32), old_lens=i32(0, 0), new_lens=i32(1, 1), page_size=16,
                   free_ring=i32(0, 1, 2), ends=i64(0, 3), lens=i32(0, 0), ends_out=i64(0, 0), starts=i32(0, 0, 0),
                   slot_map=i64(0, 0, 0), positions=i64(0, 0, 0)), **k}


@pytest.mark.parametrize("bad", (
    dict(page_table=torch.zeros((2, 3), dtype=torch.int64)), dict(page_table=torch.zeros((3, 3), dtype=torch.int32)),
    dict(page_table=torch.zeros(6, dtype=torch.int32)), dict(page_table=torch.zeros((1, 3), dtype=torch.int32).expand(2, 3)),
    dict(page_table=torch.zeros((3, 2), dtype=torch.int32).t()), dict(old_lens=i64(0, 0)), dict(new_lens=i32(1)),
    dict(new_lens=i32(1, 1, 1, 1)[::2]), dict(lens=i32(0)), dict(ends=i64(0, 3, 4)), dict(ends_out=i32(0, 0)),
    dict(free_ring=i64(0, 1)), dict(starts=i32(0, 0)), dict(slot_map=i64(0, 0)), dict(positions=i32(0, 0, 0))))
def test_kv_pages_refusals(P, bad):
    with pytest.raises(M.MgError):
        P.kv_pages(**pages_args(**bad))


def append_args(**k):
    z = lambda *s, d=BF: torch.zeros(s, dtype=d)
    return {**dict(q=z(3, 4, 64), k=z(3, 2, 64), v=z(3, 2, 64), eps=1e-6, qk_scale=1.0, cos=z(9, 32), sin=z(9, 32),
                   positions=i64(0, 1, 2), slot_map=i64(0, 1, 2), k_cache=z(4, 8, 2, 64), v_cache=z(4, 8, 2, 64)), **k}


@pytest.mark.parametrize("bad", (
    dict(q=torch.zeros(3, 4, 64, dtype=torch.int16)), dict(q=torch.zeros(3, 256, dtype=BF)),
    dict(q=torch.zeros(1, 4, 64, dtype=BF).expand(3, 4, 64)), dict(q=torch.zeros(3, 4, 128, dtype=BF)[..., ::2]),
    dict(k=torch.zeros(3, 3, 64, dtype=BF)), dict(v=torch.zeros(2, 2, 64, dtype=BF)),
    dict(v=torch.zeros(3, 2, 64, dtype=torch.float16)), dict(cos=None), dict(cos=torch.zeros(9, 64, dtype=BF)),
    dict(cos=torch.zeros(9, 32), sin=torch.zeros(9, 32)), dict(sin=torch.zeros(8, 32, dtype=BF)),
    dict(positions=i64(0, 1)), dict(slot_map=i32(0, 1, 2)), dict(positions=i64(0, 1, 2, 3, 4, 5)[::2]),
    dict(k_cache=torch.zeros(4, 8, 2, 32, dtype=BF)), dict(v_cache=torch.zeros(3, 8, 2, 64, dtype=BF)),
    dict(k_cache=torch.zeros(4, 8, 2, 64, dtype=torch.int8)), dict(k_scale=torch.zeros(4, 8, 2, 2, dtype=torch.float16)),
    dict(k_cache=torch.zeros(4, 2, 8, 64, dtype=BF).transpose(1, 2), v_cache=torch.zeros(4, 2, 8, 64, dtype=BF).transpose(1, 2)),
    dict(k_cache=torch.zeros(4, 8, 2, 64, dtype=torch.int8), v_cache=torch.zeros(4, 8, 2, 64, dtype=torch.int8),
         k_scale=torch.zeros(4, 8, 2, 2), v_scale=torch.zeros(4, 8, 2, 2))))
def test_append_refusals(P, bad):
    with pytest.raises(M.MgError):
        P.qk_norm_rope_paged(**append_args(**bad))


def decode_args(**k):
    z = lambda *s, d=BF: torch.zeros(s, dtype=d)
    return {**dict(q=z(2, 4, 64), k_cache=z(4, 8, 2, 64), v_cache=z(4, 8, 2, 64), page_table=torch.zeros((2, 3), dtype=torch.int32),
                   lens=i32(1, 2), scaling=0.1, out=z(2, 4, 64)), **k}


@pytest.mark.parametrize("bad", (
    dict(q=torch.zeros(2, 4, 64, dtype=torch.float64)), dict(q=torch.zeros(2, 4, 64, dtype=torch.float16)),
    dict(q=torch.zeros(4, 2, 64, dtype=BF).transpose(0, 1)), dict(out=torch.zeros(2, 4, 32, dtype=BF)),
    dict(out=torch.zeros(1, 4, 64, dtype=BF).expand(2, 4, 64)), dict(out=torch.zeros(2, 4, 64, dtype=torch.int32)),
    dict(lens=i32(1)), dict(lens=i64(1, 2)), dict(page_table=torch.zeros((1, 3), dtype=torch.int32)),
    dict(k_cache=torch.zeros(4, 8, 2, 32, dtype=BF), v_cache=torch.zeros(4, 8, 2, 32, dtype=BF)),
    dict(k_cache=torch.zeros(32, 2, 64, dtype=BF)), dict(v_scale=torch.zeros(4, 8, 2, 2, dtype=torch.float16))))
def test_decode_refusals(P, bad):
    with pytest.raises(M.MgError):
        P.attn_decode_paged(**decode_args(**bad))


def test_what_is_taken(P):
    """views that the library can read: padded rows, one request's odd strides, no maps"""
    P.lib = Calls()
    wide = torch.zeros((2, 7), dtype=torch.int32)
    P.kv_pages(**pages_args(page_table=wide[:, :3], slot_map=None, starts=None))
    name, a = P.lib.args
    assert name == "mg_kv_pages" and a[2:5] == (7, 2, 3) and a[-1] == 3 and a[-3] is None and a[-4] is None
    P.kv_pages(**pages_args(slot_map=None, positions=None))
    assert P.lib.args[1][-1] == 0
    q = torch.zeros(2, 6, 64, dtype=BF)[:, 1:5]
    P.attn_decode_paged(**decode_args(q=q))
    assert P.lib.args[1][2] == 6 * 64
    P.attn_decode_paged(**decode_args(q=q[:1].expand(1, 4, 64), out=None, lens=i32(1), page_table=wide[:1, :3]))
    assert P.lib.args[1][2] == 4 * 64 and P.lib.args[1][-1] == M.F32
    P.qk_norm_rope_paged(**append_args(cos=None, sin=None))
    assert P.lib.args[1][13:16] == (None, None, 0)


def test_abi_without_a_context():
    L = M.load_library()
    n = {name: [0.0 if t is ctypes.c_double else None if t is ctypes.c_void_p else 0 for t in M._SIGS[name][0]]
         for name in ("mg_kv_pages", "mg_qk_norm_rope_paged", "mg_attn_decode_paged")}
    for name, args in n.items():
        assert getattr(L, name)(*args) == -1
        assert b"NULL context" in L.mg_last_error()
