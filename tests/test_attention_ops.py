"""Masked attention and the 8-bit cache: what the host refuses, without a GPU."""
from __future__ import annotations

import ctypes

import pytest
import torch

from flash_vla_b200 import op_table
from flash_vla_b200.hardware.nvidia.b200.pi0.backends.cuda import _lib
from flash_vla_b200.hardware.nvidia.b200.pi0.buffers import QuantizedCache, allocate_quantized_cache

bf16, f32, i32 = torch.bfloat16, torch.float32, torch.int32
OPS = ("masked_attention", "cache_append", "cache_attention", "cache_evict")


def test_both_tables_hold_the_operators():
    for fused in (True, False):
        assert set(OPS) <= set(vars(op_table(fused)))
    assert op_table(True, plan={"masked_attention": "cuda"}).masked_attention is op_table().masked_attention


def z(*shape, dtype=bf16):
    return torch.zeros(shape, dtype=dtype)


GOOD = dict(Q=(2, 3, 8, 64), K=(2, 5, 2, 64), V=(2, 5, 2, 64), out=(2, 3, 8, 64))


@pytest.mark.parametrize("change,kw,message", [
    ({"K": (2, 5, 3, 64), "V": (2, 5, 3, 64)}, {}, "query heads"), ({"V": (2, 6, 2, 64)}, {}, "do not fit"), ({"out": (2, 3, 8, 32)}, {}, "do not fit"),
    ({n: s[:3] + (60,) for n, s in GOOD.items()}, {}, "16 bytes"), ({n: s[:3] + (264,) for n, s in GOOD.items()}, {}, "head_dim"),
    ({"Q": (2, 3, 258, 64), "out": (2, 3, 258, 64)}, {}, "query heads"), ({"Q": (6, 8, 64)}, {}, "episodes, tokens"),
    ({}, {"prefix": z(2, dtype=i32)}, "causal"), ({}, {"q_docs": z(2, 3, dtype=i32)}, "documents"), ({}, {"cap": -1.0}, "cap"), ({}, {"cap": float("nan")}, "cap"),
    ({}, {"scale": float("inf")}, "scale"), ({}, {"k_lens": z(2, dtype=torch.int64)}, "k_lens"), ({}, {"k_lens": z(3, dtype=i32)}, "k_lens"),
    ({}, {"slopes": z(8)}, "slopes"), ({}, {"lse": z(2, 3, 8, dtype=f32)}, "lse"), ({}, {}, "CUDA")])
def test_masked_attention_refuses(change, kw, message):
    t = {n: z(*s) for n, s in {**GOOD, **change}.items()}
    kw = dict(kw)
    scale = kw.pop("scale", 0.125)
    with pytest.raises(ValueError, match=message):
        op_table().masked_attention(t["Q"], t["K"], t["V"], scale, t["out"], **kw)


def test_masked_attention_refuses_types_and_layouts():
    t = {n: z(*s) for n, s in GOOD.items()}
    call = op_table().masked_attention
    with pytest.raises(ValueError, match="bfloat16"):
        call(t["Q"].half(), t["K"], t["V"], 1.0, t["out"])
    with pytest.raises(ValueError, match="contiguous"):
        call(z(2, 3, 64, 8).mT, t["K"], t["V"], 1.0, t["out"])
    with pytest.raises(ValueError, match="16 bytes"):
        call(z(2, 3, 8, 65)[..., :64], t["K"], t["V"], 1.0, t["out"])
    with pytest.raises(ValueError, match="share memory"):
        call(t["Q"], t["K"], t["V"], 1.0, z(1, 3, 8, 64).expand(2, 3, 8, 64))


def cache(E=2, rows=128, HK=2, D=64, block=64):
    return allocate_quantized_cache(E, rows, HK, D, "cpu", block)


def test_allocate_quantized_cache():
    c = cache(rows=100, block=32)
    assert c.K.shape == (2, 128, 2, 64) and c.K.dtype == torch.float8_e4m3fn and c.K_scale.shape == (2, 4, 2) and (c.V_scale == 1).all()
    with pytest.raises(ValueError, match="blocks"):
        cache(block=48)
    with pytest.raises(ValueError, match="head_dim"):
        cache(D=72)


def test_cache_append_refuses():
    call, starts = op_table().cache_append, z(2, dtype=i32)
    for K, c, match in ((z(2, 3, 1, 64), cache(), "do not fit"), (z(2, 129, 2, 64), cache(), "129 rows"), (z(2, 3, 2, 64, dtype=f32), cache(), "bfloat16"),
                        (z(2, 3, 2, 64), cache()._replace(K_scale=z(2, 2, 2)), "K_scale"), (z(2, 3, 2, 64), cache()._replace(K=z(2, 128, 2, 64)), "float8"),
                        (z(2, 3, 2, 64), QuantizedCache(cache().K, cache().V, z(2, 3, 2, dtype=f32), z(2, 3, 2, dtype=f32)), "blocks"), (z(2, 3, 2, 64), cache(), "CUDA")):
        with pytest.raises(ValueError, match=match):
            call(K, K, c, starts)
    with pytest.raises(ValueError, match="starts"):
        call(z(2, 3, 2, 64), z(2, 3, 2, 64), cache(), z(3, dtype=i32))


def test_cache_attention_refuses():
    call, Q, lengths = op_table().cache_attention, z(2, 1, 4, 64), z(2, dtype=i32)
    with pytest.raises(ValueError, match="do not fit"):
        call(z(2, 1, 4, 128), cache(), lengths, 1.0, z(2, 1, 4, 128))
    with pytest.raises(ValueError, match="weights"):
        call(Q, cache(), lengths, 1.0, Q, weights=z(2, 64, dtype=f32))
    with pytest.raises(ValueError, match="decay"):
        call(Q, cache(), lengths, 1.0, Q, decay=float("nan"))
    with pytest.raises(ValueError, match="k_pos"):
        call(Q, cache(), lengths, 1.0, Q, k_pos=z(2, 128))
    with pytest.raises(ValueError, match="CUDA"):
        call(Q, cache(), lengths, 1.0, Q)


def test_cache_evict_refuses():
    call, lengths, w = op_table().cache_evict, z(2, dtype=i32), z(2, 128, dtype=f32)
    for keep, kw, out, match in ((0, {}, cache(), "0 rows"), (129, {}, cache(), "129 rows"), (10, {"sinks": 6, "recent": 5}, cache(), "first 6"),
                                 (10, {"recent": -1}, cache(), "last -1"), (10, {}, cache(HK=1), "into"), (10, {"out_weights": z(2, 64, dtype=f32)}, cache(), "out_weights"),
                                 (10, {}, cache(), "CUDA")):
        with pytest.raises(ValueError, match=match):
            call(cache(), lengths, w, keep, out, z(2, dtype=i32), **kw)


def attention_struct(**kw):
    a = _lib.Attention()
    P = 1 << 20
    a.q = a.k = a.v = a.out = P
    a.episodes, a.tokens, a.keys, a.heads, a.kv_heads, a.head_dim, a.scale = 1, 4, 16, 8, 1, 64, 1.0
    for n, v in kw.items():
        setattr(a, n, v)
    return ctypes.byref(a)


@pytest.mark.parametrize("kw", [{"episodes": 0}, {"tokens": 0}, {"heads": 0}, {"kv_heads": 0}, {"kv_heads": 3}, {"heads": 129}, {"head_dim": 0}, {"head_dim": 260},
                                {"head_dim": 12}, {"q": None}, {"k": None}, {"q": (1 << 20) + 8}, {"k_scale": 1 << 20}, {"prefix": 1 << 20}, {"q_docs": 1 << 20},
                                {"weights": 1 << 20}, {"cap": -1.0}, {"k_scale": 1 << 20, "v_scale": 1 << 20, "block": 48}, {"keys": -1}])
def test_attention_entry_refuses_before_it_launches(kw):
    lib = _lib.load()
    before = lib.fvla_launch_count()
    assert lib.fvla_attention_run(attention_struct(**kw), None) == -1
    assert b"attention" in lib.fvla_last_error() and lib.fvla_launch_count() == before
    assert lib.fvla_attention_run(None, None) == -1


def test_cache_entries_refuse_before_they_launch():
    lib, P = _lib.load(), 1 << 20
    before = lib.fvla_launch_count()
    assert lib.fvla_cache_append(None, None) == -1 and lib.fvla_cache_evict(None, None) == -1
    for kw in ({"episodes": 0}, {"tokens": 200}, {"block": 48}, {"head_dim": 72}, {"k_held": None}, {"starts": None}, {"v": P + 4}):
        a = _lib.CacheAppend()
        a.k = a.v = a.k_held = a.v_held = a.k_scale = a.v_scale = a.starts = P
        a.episodes, a.tokens, a.rows, a.kv_heads, a.head_dim, a.block = 1, 4, 128, 1, 64, 64
        for n, v in kw.items():
            setattr(a, n, v)
        assert lib.fvla_cache_append(ctypes.byref(a), None) == -1, kw
    for kw, status in (({"keep": 0}, -1), ({"keep": 200}, -1), ({"sinks": 40, "recent": 40}, -1), ({"out_block": 24}, -1), ({"weights": None}, -1), ({"ws": None}, -2),
                       ({"ws_bytes": 8}, -2)):
        a = _lib.CacheEvict()
        for n, _ in _lib.CacheEvict._fields_[:15]:
            setattr(a, n, P)
        a.ws_bytes = 1 << 20
        a.episodes, a.rows, a.out_rows, a.kv_heads, a.head_dim, a.block, a.out_block, a.keep = 1, 128, 64, 1, 64, 64, 64, 64
        for n, v in kw.items():
            setattr(a, n, v)
        assert lib.fvla_cache_evict(ctypes.byref(a), None) == status, kw
    assert lib.fvla_launch_count() == before
    assert lib.fvla_cache_evict_workspace_bytes(2, 100) >= 800 and lib.fvla_cache_evict_workspace_bytes(0, 100) == 0
