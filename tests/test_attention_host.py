"""The attention operators without a GPU: refusals of the wrappers and of the C entry points (both before anything is
launched), their registry keys, the workspace function, and the float64 statements against hand-made cases."""

from __future__ import annotations

import ctypes
import math

import numpy as np
import pytest

from hipengine_amd.core.build import load_library
from hipengine_amd.kernels.hip_gfx950.attention import kv_cache_q8 as C
from hipengine_amd.kernels.hip_gfx950.attention import paged_attention_q8 as A
from hipengine_amd.kernels.hip_gfx950.attention import qk_norm_rope as R
from hipengine_amd.kernels.hip_gfx950.sampling import sample_rows as S
from hipengine_amd.kernels.registry import resolve
from oracle import attention_oracle as O


class Never:
    """Stands in for the library: reaching it fails the test."""

    def __getattr__(self, name):
        raise AssertionError(f"{name} was reached")


def cache(**over):
    args = dict(k_ptr=4096, v_ptr=8192, k_scale_ptr=16, v_scale_ptr=16, pages=4, page_size=64, kv_heads=2, head_dim=128)
    return C.KVCacheQ8(**(args | over))


@pytest.mark.parametrize("over", [{"pages": 0}, {"pages": 2**31}, {"page_size": 16}, {"page_size": 96}, {"page_size": 2**21},
                                  {"kv_heads": 0}, {"kv_heads": 65536}, {"head_dim": 96}, {"k_ptr": 0}, {"v_scale_ptr": 0},
                                  {"k_ptr": 4097}, {"v_ptr": 8200}])
def test_cache_refusals(over):
    with pytest.raises(ValueError):
        cache(**over)


def test_cache_sizes():
    assert C.KVCacheQ8.value_bytes(4, 64, 2, 128) == 4 * 64 * 2 * 128 and C.KVCacheQ8.scale_bytes(4, 64, 2) == 4 * 2 * 2 * 4
    assert sorted(C.v_place(t) for t in range(32)) == list(range(32))


NORM = dict(q_ptr=16, k_ptr=32, q_out_ptr=48, k_out_ptr=64, tokens=1, q_heads=4, kv_heads=2, head_dim=128)
ROT = dict(positions_ptr=16, inv_freq_ptr=16, rotary_dim=64)


@pytest.mark.parametrize("over", [
    {"tokens": 0}, {"tokens": 4194304}, {"q_heads": -1}, {"q_heads": 0, "kv_heads": 0}, {"q_heads": 4097}, {"head_dim": 96},
    {"q_ptr": 0}, {"k_out_ptr": None}, {"in_kind": "q8_1"}, {"out_kind": "f16"}, {"eps": -1.0}, {"eps": math.nan},
    {"rotary_dim": 64}, {**ROT, "rotary_dim": 24}, {**ROT, "rotary_dim": 0}, {**ROT, "rotary_dim": 144},
    {**ROT, "positions_ptr": None}, {"q_stride": 511}, {"k_out_stride": 255}, {"q_stride": -1},
    {"q_out_ptr": 16, "out_kind": "f32"}, {"k_out_ptr": 32, "k_stride": 300},
])
def test_qk_norm_rope_refusals(over):
    with pytest.raises(ValueError):
        R.qk_norm_rope(**(NORM | over), library=Never())


APPEND = dict(k_ptr=16, v_ptr=16, page_table_ptr=16, table_stride=2, q_start_ptr=16, kv_lens_ptr=16, tokens=3, batch=2, max_q_len=2)


@pytest.mark.parametrize("over", [
    {"tokens": 0}, {"batch": 0}, {"max_q_len": 0}, {"table_stride": 0}, {"k_ptr": 0}, {"v_ptr": None}, {"page_table_ptr": 0},
    {"q_start_ptr": 0}, {"kv_lens_ptr": 0}, {"in_kind": "int8"}, {"rotary_dim": 16}, {"inv_freq_ptr": 16, "rotary_dim": 8},
    {"inv_freq_ptr": 16, "rotary_dim": 256}, {"k_stride": 100}, {"v_stride": -4}, {"eps": -1e-6}, {"batch": 65536},
])
def test_append_refusals(over):
    with pytest.raises(ValueError):
        C.kv_append_q8(cache(), **(APPEND | over), library=Never())


READ = dict(k_out_ptr=16, v_out_ptr=16, page_table_ptr=16, table_stride=2, row_start_ptr=16, kv_lens_ptr=16, tokens=3, batch=2)


@pytest.mark.parametrize("over", [{"tokens": 0}, {"batch": 0}, {"table_stride": 0}, {"k_out_ptr": None, "v_out_ptr": 0},
                                  {"out_kind": ""}, {"k_out_stride": 255}, {"batch": 65536}, {"row_start_ptr": 0}, {"kv_lens_ptr": None}])
def test_read_refusals(over):
    with pytest.raises(ValueError):
        C.kv_read_q8(cache(), **(READ | over), library=Never())


ATTEND = dict(q_ptr=16, out_ptr=32, page_table_ptr=16, table_stride=2, q_start_ptr=16, kv_lens_ptr=16, tokens=3, batch=2,
              max_q_len=2, max_kv_len=100, q_heads=8)


@pytest.mark.parametrize("over", [
    {"tokens": 0}, {"tokens": 2**26 + 1}, {"batch": 0}, {"batch": 65536}, {"max_q_len": 0}, {"max_kv_len": -1},
    {"max_kv_len": 2**30 + 1}, {"q_heads": 0}, {"q_heads": 7}, {"q_heads": 4098}, {"table_stride": 0}, {"kind": "f32"},
    {"scale": 0.0}, {"scale": -1.0}, {"scale": math.inf}, {"scale": math.nan}, {"window": -1}, {"q_stride": 1023},
    {"out_stride": 5}, {"q_ptr": 0}, {"out_ptr": 0}, {"out_ptr": 16}, {"page_table_ptr": 0}, {"kv_lens_ptr": 0},
])
def test_attention_refusals(over):
    with pytest.raises(ValueError):
        A.paged_attention_q8(cache(), **(ATTEND | over), library=Never())


SAMPLE = dict(logits_ptr=16, uniform_ptr=16, out_ids_ptr=16, rows=2, vocab_size=100, workspace_ptr=16, workspace_bytes=1 << 20)


@pytest.mark.parametrize("over", [{"rows": 0}, {"rows": 65536}, {"vocab_size": 0}, {"vocab_size": 2**22 + 1}, {"logits_stride": 99},
                                  {"logits_stride": -1}, {"logits_ptr": 0}, {"uniform_ptr": None}, {"out_ids_ptr": 0}, {"workspace_ptr": None}])
def test_sample_refusals(over):
    with pytest.raises(ValueError):
        S.sample_f32_rows_i32(**(SAMPLE | over), library=Never())


# ---- the C entry points refuse by themselves -------------------------------------------------------------------------


def _norm(**over):
    a = dict(q=16, k=32, qw=None, kw=None, pos=None, freq=None, qo=48, ko=64, ik=1, ok=1, tokens=1, hq=4, hk=2, dim=128, rot=0,
             qs=0, ks=0, qos=0, kos=0, eps=1e-6, rs=1.0, inter=0, stream=None) | over
    fn = load_library().hipengine_gfx950_qk_norm_rope
    fn.argtypes, fn.restype = R._ARGS, ctypes.c_int
    return fn(*a.values())


@pytest.mark.parametrize("over", [
    {"q": None}, {"k": None}, {"qo": None}, {"ko": None}, {"ik": 3}, {"ik": -1}, {"ok": 3}, {"tokens": 0}, {"tokens": 1 << 31},
    {"hq": -1}, {"hq": 0, "hk": 0}, {"hq": 5000}, {"dim": 80}, {"rot": 16}, {"freq": 16, "rot": 16}, {"freq": 16, "pos": 16, "rot": 20},
    {"freq": 16, "pos": 16, "rot": 256}, {"qs": 100}, {"kos": 255}, {"eps": math.nan}, {"qo": 16, "ok": 0}, {"ko": 32, "ks": 1000}])
def test_c_norm_refuses(over):
    assert _norm(**over) == 1


def _append(**over):
    a = dict(k=16, v=16, kind=1, ks=0, vs=0, w=None, pos=None, freq=None, rot=0, inter=0, eps=1e-6, rs=1.0, kc=4096, vc=8192,
             ksc=16, vsc=16, table=16, ts=2, qs=16, lens=16, tokens=3, batch=2, maxq=2, pages=4, size=64, heads=2, dim=128,
             stream=None) | over
    fn = load_library().hipengine_gfx950_kv_append_q8
    fn.argtypes, fn.restype = C._APPEND_ARGS, ctypes.c_int
    return fn(*a.values())


@pytest.mark.parametrize("over", [
    {"k": None}, {"v": None}, {"kind": 3}, {"ks": 10}, {"vs": -1}, {"rot": 32}, {"freq": 16, "rot": 8}, {"eps": -1.0}, {"kc": None},
    {"vc": 8193}, {"ksc": None}, {"vsc": None}, {"table": None}, {"ts": 0}, {"qs": None}, {"lens": None}, {"tokens": 0}, {"batch": 0},
    {"batch": 65536}, {"batch": 1 << 40}, {"maxq": 0}, {"pages": 0}, {"pages": 1 << 31}, {"size": 48}, {"size": 16}, {"size": 1 << 21}, {"heads": 0},
    {"heads": 65536}, {"dim": 127}, {"tokens": 1 << 31}])
def test_c_append_refuses(over):
    assert _append(**over) == 1


def _read(**over):
    a = dict(kc=4096, vc=8192, ksc=16, vsc=16, table=16, ts=2, rs=16, lens=16, k=16, v=16, kind=1, ks=0, vs=0, tokens=3, batch=2,
             pages=4, size=64, heads=2, dim=128, stream=None) | over
    fn = load_library().hipengine_gfx950_kv_read_q8
    fn.argtypes, fn.restype = C._READ_ARGS, ctypes.c_int
    return fn(*a.values())


@pytest.mark.parametrize("over", [{"k": None, "v": None}, {"kind": 9}, {"ks": 255}, {"vs": 1}, {"tokens": 0}, {"batch": -1}, {"batch": 65536}, {"rs": None},
                                  {"kc": 4104}, {"dim": 32}, {"size": 33}])
def test_c_read_refuses(over):
    assert _read(**over) == 1


def _attend(**over):
    a = dict(q=16, out=32, kind=1, qs=0, os=0, kc=4096, vc=8192, ksc=16, vsc=16, table=16, ts=2, start=16, lens=16, tokens=3, batch=2,
             maxq=2, maxkv=100, hq=8, hk=2, dim=128, pages=4, size=64, scale=0.1, window=0, ws=None, wsb=0, stream=None) | over
    fn = load_library().hipengine_gfx950_paged_attention_q8
    fn.argtypes, fn.restype = A._ARGS, ctypes.c_int
    return fn(*a.values())


@pytest.mark.parametrize("over", [
    {"q": None}, {"out": None}, {"out": 16}, {"kind": 0}, {"kind": 3}, {"qs": 8}, {"os": 8}, {"kc": None}, {"vc": 8200}, {"ksc": None},
    {"table": None}, {"ts": 0}, {"start": None}, {"lens": None}, {"tokens": 0}, {"tokens": 1 << 27}, {"batch": 0}, {"batch": 1 << 16},
    {"maxq": 0}, {"maxkv": -1}, {"maxkv": 1 << 31}, {"hq": 9}, {"hk": 0}, {"dim": 192}, {"pages": 0}, {"size": 8}, {"scale": 0.0},
    {"scale": math.nan}, {"scale": math.inf}, {"window": -5}, {"maxkv": 1 << 20},                      # (this needs a workspace)
    {"maxkv": 1 << 20, "ws": 4096, "wsb": 64}])
def test_c_attention_refuses(over):
    assert _attend(**over) == 1


def _sample(**over):
    a = dict(logits=16, ls=0, u=16, t=None, k=None, p=None, m=None, ids=16, lp=None, rows=2, vocab=100, ws=16, wsb=1 << 20, stream=None) | over
    fn = load_library().hipengine_gfx950_sample_f32_rows_i32
    fn.argtypes, fn.restype = S._ARGS, ctypes.c_int
    return fn(*a.values())


@pytest.mark.parametrize("over", [{"logits": None}, {"ls": 99}, {"u": None}, {"ids": None}, {"rows": 0}, {"rows": 65536}, {"vocab": 0},
                                  {"vocab": 1 << 23}, {"ws": None}, {"ws": 20}, {"wsb": 100}])
def test_c_sample_refuses(over):
    assert _sample(**over) == 1


def test_sample_workspace_function():
    assert 0 < S.sample_workspace_bytes(1, 1) < S.sample_workspace_bytes(1, 1000) < S.sample_workspace_bytes(2, 1000)
    with pytest.raises(ValueError):
        S.sample_workspace_bytes(0, 5)
    fn = load_library().hipengine_gfx950_sample_f32_rows_i32_workspace_bytes
    fn.argtypes = S._WORKSPACE_ARGS
    assert fn(1, 1, None) == 1 and fn(1, 1 << 23, ctypes.byref(ctypes.c_int64())) == 1


def test_workspace_function():
    f = A.paged_attention_q8_workspace_bytes
    assert f(1, 1, 1, 1, 8, 8, 128) == 0
    one = f(1, 1, 1, 32768, 40, 8, 128)
    assert one > 0 and one % (40 * 130 * 4) == 0
    sizes = [f(3, 3, 1, n, 40, 8, 128) for n in range(1, 40000, 97)]
    assert sizes == sorted(sizes)                          # never less for a longer cache
    for bad in ((0, 1, 1, 1, 8, 8, 128), (1, 1, 1, 1, 9, 8, 128), (1, 1, 1, 1, 8, 8, 100)):
        with pytest.raises(ValueError):
            f(*bad)
    fn = load_library().hipengine_gfx950_paged_attention_q8_workspace_bytes
    fn.argtypes = A._WORKSPACE_ARGS
    assert fn(1, 1, 1, 1, 8, 8, 128, None) == 1 and fn(1, 1, 1, 1, 8, 3, 128, ctypes.byref(ctypes.c_int64())) == 1


def test_registry_keys():
    from hipengine_amd.kernels.hip_gfx950 import register_backend_kernels

    register_backend_kernels(replace=True)
    assert resolve(backend="hip_gfx950", layer="qk_norm+rope", quant="f32_weight") is R.qk_norm_rope
    assert resolve(backend="hip_gfx950", layer="kv_cache", quant="q8_block32", variant="append") is C.kv_append_q8
    assert resolve(backend="hip_gfx950", layer="kv_cache", quant="q8_block32", variant="read") is C.kv_read_q8
    assert resolve(backend="hip_gfx950", layer="attention", quant="q8_block32", variant="paged") is A.paged_attention_q8
    assert resolve(backend="hip_gfx950", layer="sample", quant="f32", variant="rows_i32") is S.sample_f32_rows_i32


# ---- the statements the GPU tests compare with -----------------------------------------------------------------------


def test_statement_of_the_layout():
    rng = np.random.default_rng(1)
    k, v = (rng.integers(-127, 128, (2, 3, 64, 64)) for _ in range(2))
    kb, vb = O.pack_cache(k, v)
    assert all(np.array_equal(a, b) for a, b in zip(O.unpack_cache(kb, vb, 64), (k, v)))
    # token 37 is token 5 of block 1; dim 19 is value 3 of the second sixteen
    assert kb[1, 2, 1, (1 * 32 + 5) * 16 + 3] == k[1, 2, 37, 19] + 128
    assert vb[1, 2, 1, 19 * 32 + C.v_place(5)] == v[1, 2, 37, 19] + 128


def test_statement_of_the_rotation():
    x = np.arange(1.0, 65.0).reshape(1, 1, 64)
    freq = np.array([0.5, 0.25] + [0.1] * 6)
    for interleaved in (False, True):
        y, _ = O.norm_rotate(x, None, [3], freq, interleaved=interleaved)
        a, b = (2, 3) if interleaved else (1, 9)
        t = 3 * 0.25
        assert np.isclose(y[0, 0, a], x[0, 0, a] * math.cos(t) - x[0, 0, b] * math.sin(t))
        assert np.isclose(y[0, 0, b], x[0, 0, b] * math.cos(t) + x[0, 0, a] * math.sin(t))
        assert np.array_equal(y[..., 16:], x[..., 16:])


def test_statement_of_append_and_attention():
    rng = np.random.default_rng(2)
    dim, page = 64, 32
    table = np.array([[1, 0]], np.int32)
    ki, vi = (np.zeros((2, 1, page, dim), np.int64) for _ in range(2))
    ks, vs = np.ones((2, 1, 1)), np.ones((2, 1, 1))
    k, v = rng.standard_normal((40, 1, dim)), rng.standard_normal((40, 1, dim))
    O.append(k[:30], v[:30], ki, vi, ks, vs, table, [0, 30], [30])
    O.append(k[30:] * 4, v[30:], ki, vi, ks, vs, table, [0, 10], [40])
    values, there = O.gather(ki, ks, table[0], 40)
    assert there.all()
    full = np.concatenate([k[:30], k[30:] * 4])[:, 0]
    assert np.abs(values[0] - full).max() <= ks.max() * 1.01
    q = rng.standard_normal((2, 2, dim))
    out, *_ = O.attention(q, ki, vi, ks, vs, table, [0, 2], [40], scale=0.1, window=5)
    vv, _ = O.gather(vi, vs, table[0], 40)
    s = q[0, 1] @ values[0, 34:39].T * 0.1                 # the query at place 38 sees 34 .. 38
    p = np.exp(s) / np.exp(s).sum()
    assert np.allclose(out[0, 1], p @ vv[0, 34:39])


def test_statement_of_sampling():
    row = np.log(np.array([1.0, 4.0, 2.0, 4.0, 1.0]))                   # order: 1, 3, 2, 0, 4
    one = lambda *args, **kw: next(iter(O.sample(*args, **kw)))  # noqa: E731
    assert one(row, 0.0) == 0 and one(row, 0.99) == 4
    assert one(row, 0.5, top_k=1) == 1 and one(row, 0.6, top_k=2) == 3
    assert one(row, 0.99, top_p=0.4) == 3                                # 4 of 12 is not 0.4, 8 is
    assert one(row, 0.99, top_p=0.3) == 1
    assert one(row, 0.99, min_p=0.4) == 3 and one(row, 0.45, min_p=0.4) == 2
    assert one(row, 0.99, temperature=0) == 1 and one(np.full(3, -np.inf), 0.5) == -1
    assert np.isclose(O.sample(row, 0.0)[0][0], math.log(1 / 12))
    assert set(O.sample(row, 1 / 12 + 1e-9, accuracy=1e-6)) == {0, 1}    # on the border between the first two tokens


# ---- limits of attention's sizes ---------------------------------------------------------------------------------------


@pytest.mark.parametrize("tokens,max_q,q_heads,kv_heads,dim,fits", [
    (1 << 20, 1 << 20, 7, 1, 128, True),
    (1048560, 1048560, 8, 1, 128, True), (1048561, 1048561, 8, 1, 128, False),     # 65535 * 128 rows, and a token more
    (1 << 20, 1 << 20, 8, 1, 64, False), (1 << 26, 1 << 26, 16, 16, 64, False),
    (1 << 20, 1 << 20, 8, 1, 256, True), (2097120, 2097120, 8, 1, 256, True), (2097121, 2097121, 8, 1, 256, False),
    (1 << 20, 1000, 8, 1, 64, True),                                               # many short sequences
    (5, 1 << 40, 40, 8, 128, True), (1, 2**62, 4096, 1, 64, True),                 # announced for more rows than there are
])
def test_rows_of_a_sequence_that_fit(tokens, max_q, q_heads, kv_heads, dim, fits):
    """The workspace function, the launch and both wrappers agree on what they take."""
    fn = load_library().hipengine_gfx950_paged_attention_q8_workspace_bytes
    fn.argtypes = A._WORKSPACE_ARGS
    sizes = (tokens, 1, max_q, 4096, q_heads, kv_heads, dim)
    assert fn(*sizes, ctypes.byref(ctypes.c_int64())) == (0 if fits else 1)
    call = dict(ATTEND, tokens=tokens, batch=1, max_q_len=max_q, max_kv_len=4096, q_heads=q_heads)
    small = cache(kv_heads=kv_heads, head_dim=dim)
    if fits:
        assert A.paged_attention_q8_workspace_bytes(*sizes) >= 0
        with pytest.raises(AssertionError, match="was reached"):
            A.paged_attention_q8(small, **call, library=Never())
    else:
        assert _attend(tokens=tokens, batch=1, maxq=max_q, maxkv=4096, hq=q_heads, hk=kv_heads, dim=dim, ws=4096, wsb=1 << 62) == 1
        with pytest.raises(ValueError, match="65535"):
            A.paged_attention_q8_workspace_bytes(*sizes)
        with pytest.raises(ValueError, match="65535"):
            A.paged_attention_q8(small, **call, library=Never())
