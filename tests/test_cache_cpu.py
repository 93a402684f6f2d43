"""The cache and the norm and rotation without a GPU: where a position lies, refusals, sizes that hosts ask for."""
import ctypes as C

import numpy as np
import pytest
import torch

import flashmask_b200 as fm
from flashmask_b200 import _lib
import _cache_util as ref


def cache(pages=5, page=16, H=2, d=64, dv=64, dtype=0):
    c = _lib.KvCache()
    c.k = c.v = c.k_scale = c.v_scale = 256
    c.num_pages, c.page_size, c.Hkv, c.d, c.dv, c.dtype = pages, page, H, d, dv, dtype
    return c


def args(table=None, B=1, S=1, Hq=4):
    a = _lib.KvArgs()
    a.B, a.S, a.Hq, a.causal, a.softmax_scale = B, S, Hq, 1, 0.1
    if table is not None:
        a.max_pages, a.table_stride, a.page_table = table.shape[1], table.shape[1], table.ctypes.data
    a.seqlens = a.start = a.q = a.k = a.v = a.o = a.lse = a.k_out = a.v_out = a.workspace = 256
    return a


def test_every_position_lies_inside_the_payload_or_nowhere():
    lib = _lib.load()
    table = np.array([[3, -1, 5, 0, 2 ** 31 - 1, -2 ** 31, 4], [0, 1, 2, 3, 4, 5, 6]], dtype=np.int32)
    c, a = cache(d=64, dv=128), args(table, B=2)
    for value, w in ((0, 64), (1, 128)):
        for b in range(2):
            for pos in list(range(-20, 7 * 16 + 20)) + [2 ** 31 - 1, 2 ** 31, -2 ** 31, -2 ** 31 - 1, 2 ** 40]:
                for h in range(2):
                    at = lib.fm_kv_locate(C.byref(c), C.byref(a), b, h, pos, value)
                    page = int(table[b, pos // 16]) if 0 <= pos < 7 * 16 else -1
                    if 0 <= page < 5:
                        assert at == ((page * 2 + h) * 16 + pos % 16) * w and at + w <= 5 * 2 * 16 * w
                    else:
                        assert at == -1, (pos, at)
    assert lib.fm_kv_locate(C.byref(c), C.byref(a), 2, 0, 0, 0) == -1
    assert lib.fm_kv_locate(C.byref(c), C.byref(a), 0, 2, 0, 0) == -1


def test_offsets_beyond_32_bits():
    lib = _lib.load()
    table = np.array([[1 << 20]], dtype=np.int32)
    c, a = cache(pages=(1 << 20) + 1, page=128, H=8, d=128, dv=128), args(table)
    assert lib.fm_kv_locate(C.byref(c), C.byref(a), 0, 7, 127, 0) == (((1 << 20) * 8 + 7) * 128 + 127) * 128 > 2 ** 32


def test_refusals_come_before_any_launch():
    lib = _lib.load()
    table = np.zeros((1, 3), dtype=np.int32)
    calls = {"write": lambda c, a: lib.fm_kv_write(C.byref(c), C.byref(a), None), "read": lambda c, a: lib.fm_kv_read(C.byref(c), C.byref(a), None),
             "attention": lambda c, a: lib.fm_kv_attention(C.byref(c), C.byref(a), None)}
    for name, call in calls.items():
        for change, status in ((dict(page_size=24), 2), (dict(page_size=256), 2), (dict(d=72), 2), (dict(d=192), 2), (dict(dv=256), 2), (dict(num_pages=0), 1),
                               (dict(Hkv=0), 1), (dict(dtype=2), 1), (dict(k=None), 1), (dict(v_scale=None), 1), (dict(k=264), 1)):
            c = cache()
            for key, value in change.items():
                setattr(c, key, value)
            assert call(c, args(table)) == status, (name, change)
        for change, status in ((dict(B=-1), 1), (dict(S=-1), 1), (dict(dtype=7), 1), (dict(page_table=None), 1), (dict(max_pages=2 ** 28), 2)):
            a = args(table)
            for key, value in change.items():
                setattr(a, key, value)
            assert call(cache(), a) == status, (name, change)
    for change, status in ((dict(Hq=3), 1), (dict(window=-1), 1), (dict(window=4, causal=0), 1), (dict(q=None), 1), (dict(q=264), 1), (dict(B=9000), 2)):
        a = args(np.zeros((9000, 3), dtype=np.int32))
        a.workspace_bytes = 1 << 40
        for key, value in change.items():
            setattr(a, key, value)
        assert calls["attention"](cache(), a) == status, change
    a = args(table)
    a.workspace_bytes = 16
    assert calls["attention"](cache(), a) == 4 and b"workspace" in lib.fm_last_error()
    for which in ("k_stride", "v_stride"):
        a = args(table)
        setattr(a, which, _lib.I64x3(64, 4, 64))
        assert calls["write"](cache(), a) == 1


def test_nothing_to_do_is_no_error():
    lib = _lib.load()
    for B, S in ((0, 1), (1, 0)):
        a = args(np.zeros((1, 1), dtype=np.int32), B=B, S=S)
        a.workspace_bytes = 1 << 40
        assert lib.fm_kv_write(C.byref(cache()), C.byref(a), None) == 0
        assert lib.fm_kv_attention(C.byref(cache()), C.byref(a), None) == 0
        if S == 0 or B == 0:
            assert lib.fm_kv_read(C.byref(cache()), C.byref(a), None) == 0


def test_size_queries_survive_arguments_that_a_call_would_refuse():
    lib = _lib.load()
    for B, S, Hq, Hkv in ((1, 1, 4, 0), (1, 1, 3, 2), (-1, 1, 4, 2), (1, -1, 4, 2), (1, 1, 0, 2), (1, 1, 4, -2)):
        assert lib.fm_kv_attention_workspace_bytes(C.byref(cache(H=Hkv)), C.byref(args(B=B, S=S, Hq=Hq))) == 0
    assert lib.fm_kv_attention_workspace_bytes(C.byref(cache()), C.byref(args())) > 0
    n = _lib.NormRotaryArgs()
    assert lib.fm_norm_rotary_bwd_workspace_bytes(C.byref(n)) == 0
    n.B, n.S, n.Hq, n.Hk, n.d = 2, 100, 8, 2, 128
    assert lib.fm_norm_rotary_bwd_workspace_bytes(C.byref(n)) > 0


def test_norm_rotary_refusals():
    lib = _lib.load()

    def make(**change):
        n = _lib.NormRotaryArgs()
        n.B, n.S, n.Hq, n.Hk, n.d, n.rot, n.table = 1, 4, 2, 1, 64, 64, 8
        n.q = n.k = n.q_out = n.k_out = n.cos = n.sin = 256
        for key, value in change.items():
            setattr(n, key, value)
        return n
    for change, status in ((dict(d=60), 2), (dict(d=528), 2), (dict(rot=24), 2), (dict(rot=80), 2), (dict(cos=None), 1), (dict(q=264), 1), (dict(q=None), 1),
                           (dict(dtype=5), 1), (dict(eps=-1.0), 1), (dict(S=9), 1), (dict(q_stride=_lib.I64x3(1, 2, 3)), 1), (dict(B=-1), 1)):
        assert lib.fm_norm_rotary_fwd(C.byref(make(**change)), None) == status, change
    assert lib.fm_norm_rotary_fwd(C.byref(make(B=0)), None) == 0
    assert lib.fm_norm_rotary_bwd(C.byref(make(d_q=256, d_k=256, dq_weight=256)), None) == 4


def test_tensors_on_the_cpu_are_refused():
    c = fm.QuantizedKVCache.empty(2, 1, 32, page_size=16, device="cpu")
    assert c.page_size == 16 and c.k.dtype == torch.float8_e4m3fn
    x, t, n = torch.zeros(1, 1, 1, 32, dtype=torch.bfloat16), torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(RuntimeError):
        fm.kv_cache_write(c, x, x, t, n)
    with pytest.raises(RuntimeError):
        fm.kv_cache_read(c, t, n, n, 1)
    with pytest.raises(RuntimeError):
        fm.kv_cache_attention(x, c, t, n)
    with pytest.raises(RuntimeError):
        fm.qk_norm_rotary(x, x, None, None, torch.zeros(1, 16), torch.zeros(1, 16))
    with pytest.raises(ValueError):
        fm.kv_cache_attention(x, c, t, n, window_size=0)
    with pytest.raises(TypeError):
        fm.kv_cache_read(c, t, n, n, 1, dtype=torch.float32)
    for bad in (dict(head_dim=72), dict(head_dim=192), dict(head_dim=64, page_size=20), dict(head_dim=512)):
        with pytest.raises(NotImplementedError):
            fm.QuantizedKVCache.empty(2, 1, device="cpu", **bad)
    with pytest.raises(TypeError):
        fm.QuantizedKVCache.empty(2, 1, 64, device="cpu", dtype=torch.uint8)


def test_the_oracle_rounds_as_the_type_does():
    """grid() of the oracle against the conversion of torch, which rounds to nearest even as well."""
    x = torch.cat([torch.linspace(-448, 448, 4001), torch.logspace(-12, 2, 3000, base=2.0), torch.arange(-448, 449) / 16.0]).double()
    assert torch.equal(ref.grid(x, torch.float8_e4m3fn), x.float().to(torch.float8_e4m3fn).double())
    assert ref.least_exponent(448.0, torch.float8_e4m3fn) == 0 and ref.least_exponent(448.5, torch.float8_e4m3fn) == 1
    assert ref.least_exponent(127.0, torch.int8) == 0 and ref.least_exponent(1.0, torch.int8) == -6 and ref.least_exponent(0.0, torch.int8) == -64


def test_nan_rows_refusals():
    lib = _lib.load()
    table = np.zeros((1, 3), dtype=np.int32)
    for change, status in ((dict(Hq=3), 1), (dict(window=-1), 1), (dict(window=4, causal=0), 1), (dict(o=None), 1), (dict(lse=None), 1), (dict(seqlens=None), 1),
                           (dict(marks=None), 1), (dict(dtype=7), 1), (dict(B=-1), 1)):
        a = args(table)
        a.marks = 256
        for key, value in change.items():
            setattr(a, key, value)
        assert lib.fm_kv_nan_rows(C.byref(cache()), C.byref(a), None) == status, change
    for B, S in ((0, 1), (1, 0)):
        assert lib.fm_kv_nan_rows(C.byref(cache()), C.byref(args(table, B=B, S=S)), None) == 0


def test_the_most_keys_of_a_dense_forward():
    lib = _lib.load()
    for d, dv, most in ((64, 64, 262144), (80, 48, 262144), (128, 128, 262144), (192, 128, 262144), (256, 256, 2 ** 31 - 1), (576, 512, 2 ** 31 - 1), (192, 192, 0), (72, 640, 0)):
        assert lib.fm_fwd_max_keys(d, dv) == most, (d, dv)
