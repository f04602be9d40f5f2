"""Plans of batches while captured steps read them, page moves on the plan's stream and what a call that fails leaves: the
paged cache's calls in orders and sizes beside those of test_gpu_cache.py, whose helpers and bounds serve here."""
from __future__ import annotations

import numpy as np
import pytest

import satori_amd as S
from helpers import rng
from satori_amd.cache import CacheLayout, ElementType
from test_gpu_cache import Pool, check_attention, device  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu

F32, F16 = ElementType.F32, ElementType.F16


def test_a_prompt_in_one_chunk_needs_no_partial_results(context, device):  # noqa: F811
    # 90 rows of 256 heads would take 12 MB of partial results, more than the plan has when the step is captured; each row is
    # one part, so nothing is joined and the batch is taken.
    g = rng(90)
    rows, heads, kv, D = 90, 256, 32, 128
    pool = Pool(context, device, CacheLayout(1, kv, D, 32, F16), 4)
    c = pool.cache
    s = c.open()
    c.extend([s], [1])
    q = g.standard_normal((rows, heads, D)).astype(np.float32)
    dq, out = device(q), device(np.zeros_like(q))
    plan = c.plan(heads)
    plan.set([s], [1])
    context.capture_begin()
    plan.attention(0, dq, out)
    step = context.capture_end()
    c.extend([s], [rows - 1])
    pool.write(g, [s])
    plan.set([s], [rows])
    step.execute()
    check_attention(pool, [s], [rows], heads, q, context.download(np.zeros_like(q), out))
    step.dispose()
    plan.dispose()
