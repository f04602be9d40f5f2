"""Calls on a plan: which error comes first."""
from __future__ import annotations

import numpy as np
import pytest

import satori_amd as S
from satori_amd.cache import CacheLayout, PagedCache
from test_gpu_cache import F32, device  # noqa: F401  (device: a fixture)

pytestmark = pytest.mark.gpu


def test_missing_inputs_are_named_before_a_wrong_rotation(context, device):
    cache = PagedCache(context, CacheLayout(1, 1, 32, 32, F32), 2)
    plan = cache.plan(1)
    x = device(np.zeros(256, np.float32))
    inputs = dict(q=x, q_bias=0, q_out=x + 256, k=x + 512, k_bias=0, v=x + 768, v_bias=0)
    for name in ("q", "q_out", "k", "v"):
        for base, rotary, positions in ((1e4, 7, 0), (-1.0, 32, 0), (1e4, 32, -1)):
            with pytest.raises(S.ArgumentNullException):
                plan.append(0, **{**inputs, name: 0}, base=base, rotary=rotary, rope_table=x, rope_positions=positions)
    with pytest.raises(S.ArgumentOutOfRangeException):
        plan.append(0, **inputs, base=1e4, rotary=7)
    plan.dispose()
    cache.dispose()
