"""Masked attention and the 8-bit cache: tables, refusals and plans, without a GPU."""
from __future__ import annotations

import ctypes
from types import SimpleNamespace

import pytest
import torch

from flash_vla_b200 import op_table
from flash_vla_b200.hardware.nvidia.b200.pi0 import backends
from flash_vla_b200.hardware.nvidia.b200.pi0.backends.cuda import _lib
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
