"""Hand-written sm_100a CUDA backend for the Pi0 call sites.

Exposes the registry contract of the reference's backends
(`.../h100/pi0/backends/__init__.py:10-14`): `ALL_WRAPPERS` and `FUSED_WRAPPERS`; `STAGES` holds what this
backend offers as one call per pipeline stage, `OPERATORS` the attention with masks and the 8-bit cache, which the
reference's pipeline has no call site for.
"""
from __future__ import annotations

from . import attention_ops, fused_wrappers, stages, wrappers

ALL_WRAPPERS = dict(wrappers.ALL_WRAPPERS)
FUSED_WRAPPERS = dict(fused_wrappers.FUSED_WRAPPERS)
STAGES = dict(stages.STAGES)
OPERATORS = dict(attention_ops.OPERATORS)

__all__ = ["ALL_WRAPPERS", "FUSED_WRAPPERS", "STAGES", "OPERATORS", "attention_ops", "wrappers", "fused_wrappers"]
