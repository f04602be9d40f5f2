"""Calls on a plan: which error comes first, and batches without trees on a plan that has held one."""
from __future__ import annotations

import numpy as np
import pytest

import satori_amd as S
from helpers import rng
from satori_amd.cache import CacheLayout, PagedCache
from test_gpu_cache import F16, F32, Pool, device  # noqa: F401  (device: a fixture)
from test_gpu_trees import mixed

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


@pytest.mark.parametrize("type_,heads,kv_heads,head_dim", [(F16, 12, 2, 128), (F32, 5, 1, 48), (F16, 4, 2, 256)])
def test_batches_without_trees_on_a_plan_that_has_held_one(context, device, type_, heads, kv_heads, head_dim):
    # Eager launches look for a tree where the batch has one, captured ones where any had: the same bits as from a plan without, and
    # a tree behind them is found again.
    g = rng(head_dim)
    pool = Pool(context, device, CacheLayout(1, kv_heads, head_dim, 32, type_), 96)
    sequences = [pool.cache.open() for _ in range(3)]
    pool.cache.extend(sequences, [700, 90, 40])
    rows = 150
    q, k, v = (device(g.standard_normal((rows, n * head_dim)).astype(np.float32)) for n in (heads, kv_heads, kv_heads))
    turned, out = (device(np.zeros((rows, heads * head_dim), np.float32)) for _ in range(2))

    def run(plan):
        plan.append(0, q, 0, turned, k, 0, v, 0, 1e4, head_dim)
        plan.attention(0, turned, out)

    def results(go, n):
        pool.write(rng(1), sequences)
        for p in (turned, out):
            context.upload(p, np.full((rows, heads * head_dim), np.nan, np.float32))
        go()
        context.synchronize()
        got = [context.download(np.zeros((rows, heads * head_dim), np.float32), p)[:n] for p in (turned, out)]
        return got + [pool.download().host.copy()]

    trees = [mixed(60, 1), mixed(50, 2), mixed(40, 3)]
    plain, held = pool.cache.plan(heads), pool.cache.plan(heads)
    held.set_tree(sequences, trees)
    tree = results(lambda: run(held), 150)
    context.capture_begin()
    run(held)
    step = context.capture_end()
    for new in ([1, 1, 1], [60, 50, 40], [3, 0, 33], [1, 90, 0]):
        n = sum(new)
        plain.set(sequences, new)
        held.set(sequences, new)
        wanted = results(lambda: run(plain), n)
        for go in (lambda: run(held), step.execute):
            for a, b in zip(results(go, n), wanted):
                assert np.array_equal(a, b, equal_nan=True)
        held.set_tree(sequences, trees)
        for go in (step.execute, lambda: run(held)):
            for a, b in zip(results(go, 150), tree):
                assert np.array_equal(a, b, equal_nan=True)
    step.dispose()
    plain.dispose()
    held.dispose()
