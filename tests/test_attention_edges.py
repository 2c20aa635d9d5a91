"""Masked attention and the 8-bit cache: tables, refusals and plans, without a GPU."""
from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

from flash_vla_b200 import op_table
from flash_vla_b200.hardware.nvidia.b200.pi0 import backends
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
