"""Masked attention and the 8-bit cache: tables, refusals and plans, without a GPU."""
from __future__ import annotations

import ctypes
import random
from types import SimpleNamespace

import pytest
import torch

from flash_vla_b200 import op_table
from flash_vla_b200.hardware.nvidia.b200.pi0 import backends
from flash_vla_b200.hardware.nvidia.b200.pi0.backends.cuda import _lib, attention_ops
from flash_vla_b200.hardware.nvidia.b200.pi0.buffers import allocate_quantized_cache

bf16, f32, i32 = torch.bfloat16, torch.float32, torch.int32


def z(*shape, dtype=bf16):
    return torch.zeros(shape, dtype=dtype)


def test_a_backend_need_not_offer_the_operators(monkeypatch):
    """The registry's contract is two dicts; what goes beyond it is optional."""
    def f():
        return 1
    monkeypatch.setitem(backends.BACKENDS, "two dicts", SimpleNamespace(ALL_WRAPPERS={"decoder_norm": f}, FUSED_WRAPPERS={}))
    for table in (op_table(False, backend="two dicts"), op_table(True, backend="two dicts"), op_table(False, plan={"decoder_norm": "two dicts"}, backend="two dicts"),
                  op_table(True, plan={"decoder_norm": "two dicts"}, backend="two dicts")):
        assert vars(table) == {"decoder_norm": f}


def test_the_entry_takes_no_tokens_only_with_weights():
    lib, P = _lib.load(), 1 << 20
    a = _lib.Attention()
    a.q = a.k = a.v = a.out = a.k_scale = a.v_scale = P
    a.episodes, a.tokens, a.keys, a.heads, a.kv_heads, a.head_dim, a.block, a.scale = 1, 0, 64, 8, 1, 64, 16, 1.0
    a.q_stride[:] = a.out_stride[:] = a.k_stride[:] = a.v_stride[:] = (512, 512, 64)
    assert lib.fvla_attention_run(ctypes.byref(a), None) == -1 and b"empty" in lib.fvla_last_error()
    a.tokens, a.weights = -1, P
    assert lib.fvla_attention_run(ctypes.byref(a), None) == -1 and b"empty" in lib.fvla_last_error()
    a.tokens, a.q = 1, None
    assert lib.fvla_attention_run(ctypes.byref(a), None) == -1 and b"null" in lib.fvla_last_error()
    a.tokens, a.q, a.lse = 1, P, None
    assert lib.fvla_attention_run(ctypes.byref(a), None) == -1 and b"log-sum-exp" in lib.fvla_last_error()


def test_operands_that_interleave_are_apart_and_others_are_not():
    """Against the bytes themselves."""
    rng = random.Random(3)
    seen = {True: 0, False: 0}
    for _ in range(4000):
        def operand():
            shape = [rng.choice((1, 1, 2, 3)) for _ in range(3)] + [rng.choice((1, 2, 4))]
            order, stride, reach = rng.sample(range(3), 3), [0] * 3 + [1], shape[3]
            for axis in order:
                stride[axis] = reach * rng.choice((1, 2, 3)) if rng.random() < 0.9 else 0
                reach = max(reach, stride[axis] * shape[axis])
            size = rng.choice((1, 2))
            p = rng.randrange(0, 60)
            at = {p + size * (i * stride[0] + j * stride[1] + k * stride[2] + d) + b for i in range(shape[0]) for j in range(shape[1]) for k in range(shape[2])
                  for d in range(shape[3]) for b in range(size)}
            return p, attention_ops._footprint(tuple(shape), tuple(stride), size), at
        (p, a, x), (q, b, y) = operand(), operand()
        assert a[0] == max(x) + 1 - p
        apart = attention_ops._apart(p, a, q, b)
        assert not (apart and x & y) and apart == attention_ops._apart(q, b, p, a)
        seen[apart] += 1
    assert min(seen.values()) > 500
    kv = attention_ops._footprint((2, 5, 3, 8), (2 * 5 * 3 * 8, 2 * 3 * 8, 8, 1), 2)               # rows of (K, V)
    assert attention_ops._apart(0, kv, 3 * 8 * 2, kv) and not attention_ops._apart(0, kv, 3 * 8 * 2 - 2, kv)
    assert attention_ops._footprint((2, 0, 3, 8), (24, 24, 8, 1), 2) == (0, 0, ())


def test_attention_refuses_a_result_over_what_it_reads():
    call = op_table().masked_attention
    store = z(1 << 16)

    def at(first, *shape, strides=None):
        dense = [shape[1] * shape[2] * shape[3], shape[2] * shape[3], shape[3], 1]
        return store.as_strided(shape, strides or dense, first)
    Q, K, V = at(0, 2, 3, 4, 64), at(4096, 2, 5, 2, 64), at(8192, 2, 5, 2, 64)
    for out in (at(64, 2, 3, 4, 64), at(0, 2, 3, 4, 64, strides=[64 * 4 * 3, 64, 64 * 3, 1]), at(4096 + 64, 2, 3, 4, 64), at(8192 - 8, 2, 3, 4, 64)):
        with pytest.raises(ValueError, match="lies over"):
            call(Q, K, V, 0.1, out)
    with pytest.raises(ValueError, match="lies over"):                  # one Q for two episodes, in place of its first
        call(Q[:1].expand(2, 3, 4, 64), K, V, 0.1, Q)
    for out in (Q, at(16384, 2, 3, 4, 64)):                             # (as far as a machine without a GPU goes)
        with pytest.raises(ValueError, match="CUDA"):
            call(Q, K, V, 0.1, out)
    qkv = store[:2 * 3 * 8 * 64].view(2, 3, 8, 64)
    with pytest.raises(ValueError, match="CUDA"):                       # Q, K and V as parts of one projection's rows
        call(qkv[:, :, :4], qkv[:, :, 4:6], qkv[:, :, 6:], 0.1, qkv[:, :, :4])
    held = store.view(torch.uint8).view(torch.float8_e4m3fn)[:128 * 64].view(1, 64, 2, 64)
    c = allocate_quantized_cache(1, 64, 2, 64, "cpu")._replace(V=held)
    with pytest.raises(ValueError, match="lies over"):
        op_table().cache_attention(at(8192, 1, 3, 4, 64), c, z(1, dtype=i32), 0.1, at(2048, 1, 3, 4, 64))


def test_rows_of_a_result_may_not_overlap():
    store, Q, K = z(1 << 14), z(2, 3, 4, 64), z(2, 5, 2, 64)
    for strides in ((768, 256, 32, 1), (768, 128, 64, 1), (512, 256, 64, 1), (64, 256, 128, 1)):
        with pytest.raises(ValueError, match="share memory"):
            op_table().masked_attention(Q, K, K, 0.1, store.as_strided((2, 3, 4, 64), strides))
    for strides in ((768, 64, 192, 1), (64, 1024, 128, 1), (2048, 512, 64, 1)):
        with pytest.raises(ValueError, match="CUDA"):
            op_table().masked_attention(Q, K, K, 0.1, store.as_strided((2, 3, 4, 64), strides))
    with pytest.raises(ValueError, match="CUDA"):                       # keys may: a window that moves by a row
        op_table().masked_attention(Q, z(1 << 12).as_strided((2, 5, 2, 64), (64, 64, 64, 1)), K, 0.1, z(2, 3, 4, 64))


def test_append_refuses_a_cache_that_is_its_own_twin():
    c, starts, new = allocate_quantized_cache(2, 128, 2, 64, "cpu"), z(2, dtype=i32), z(2, 3, 2, 64)
    for twin in (c._replace(V=c.K), c._replace(V_scale=c.K_scale)):
        with pytest.raises(ValueError, match="share memory"):
            op_table().cache_append(new, new, twin, starts)


@pytest.mark.parametrize("kw", [{"scale": 1e39}, {"scale": -1e300}, {"scale": float("nan")}, {"cap": 1e39}, {"cap": 1e-45}, {"cap": 1e-300}, {"scale": 1e10, "cap": 1e-30}, {"decay": 1e39},
                                {"decay": -float("inf")}])
def test_numbers_beyond_fp32_are_refused(kw):
    """They would reach the kernels as infinities, or (a cap that rounds to zero) as another function."""
    Q, c = z(1, 1, 2, 64), allocate_quantized_cache(1, 64, 2, 64, "cpu")
    with pytest.raises(ValueError, match="finite numbers"):
        op_table().cache_attention(Q, c, z(1, dtype=i32), kw.get("scale", 0.1), z(1, 1, 2, 64), cap=kw.get("cap", 0.0), decay=kw.get("decay", 1.0))


@pytest.mark.parametrize("kw", [{"scale": float("inf")}, {"scale": float("nan")}, {"cap": float("inf")}, {"cap": 3e38}, {"scale": 1e10, "cap": 1e-30}, {"decay": float("nan")}])
def test_the_entry_refuses_numbers_that_are_not_finite(kw):
    a = _lib.Attention()
    a.q = a.k = a.v = a.out = 1 << 20
    a.q_stride[:] = a.out_stride[:] = a.k_stride[:] = a.v_stride[:] = (512, 512, 64)
    a.episodes, a.tokens, a.keys, a.heads, a.kv_heads, a.head_dim, a.scale = 1, 1, 64, 8, 1, 64, 0.1
    for name, value in kw.items():
        setattr(a, name, value)
    assert _lib.load().fvla_attention_run(ctypes.byref(a), None) == -1 and b"finite" in _lib.load().fvla_last_error()
