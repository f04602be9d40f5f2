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


def test_a_captured_step_goes_from_long_sequences_to_short_ones(context, device):  # noqa: F811
    # 32 sequences over 2000 shared positions: with 10 positions of their own the usual division asks for more partial results
    # than with 390, and than the plan has; the batch is divided into fewer parts.
    g = rng(390)
    heads, kv, D, count = 32, 8, 256, 32
    pool = Pool(context, device, CacheLayout(1, kv, D, 32, F16), 63 + 32 * 14)
    c = pool.cache
    first = c.open()
    c.extend([first], [2000])
    sequences = [first] + c.fork(first, count - 1)
    c.extend(sequences, [390] * count)
    pool.write(g, sequences)
    q = g.standard_normal((count, heads, D)).astype(np.float32)
    dq, out = device(q), device(np.zeros_like(q))
    plan, ones = c.plan(heads), [1] * count
    plan.set(sequences, ones)
    context.capture_begin()
    plan.attention(0, dq, out)
    step = context.capture_end()
    some = [0, 1, 17, 31]
    for own in (390, 10, 200, 1):
        for s in sequences:
            c.truncate(s, 2000 + own) if c.tokens(s) > 2000 + own else c.extend([s], [2000 + own - c.tokens(s)])
        if own == 200:  # (positions that were given up hold whatever they held: written anew)
            pool.write(g, sequences)
        plan.set(sequences, ones)
        context.upload(out, np.full_like(q, np.nan))
        step.execute()
        got = context.download(np.zeros_like(q), out)
        check_attention(pool, [sequences[i] for i in some], [1] * 4, heads, q[some], got[some], label=str(own))
        assert np.isfinite(got).all()
    step.dispose()
    plan.dispose()


def test_a_plan_is_written_by_the_steps_that_append(context, device):  # noqa: F811
    # Two steps read a plan and the first of them writes its rows; once that one is gone, batches in shared pages are taken
    # again, whatever the other does. A plan whose only append was captured in a step that is gone is written by nothing.
    pool = Pool(context, device, CacheLayout(1, 1, 32, 32, F16), 8)
    c = pool.cache
    s = c.open()
    c.extend([s], [40])
    plan = c.plan(1)
    plan.set([s], [1])
    q, out = device(np.zeros((1, 32), np.float32)), device(np.zeros((1, 32), np.float32))

    def captured(*calls):
        context.capture_begin()
        for call in calls:
            call()
        return context.capture_end()

    append = lambda: plan.append(0, q, 0, out, q, 0, q, 0, 1e4, 32)  # noqa: E731
    attend = lambda: plan.attention(0, q, out)  # noqa: E731
    both, reads, again = captured(attend, append, attend, append), captured(attend), captured(append)
    other = c.fork(s)[0]
    for step in (both, again):
        with pytest.raises(S.InvalidOperationException):
            plan.set([s, other], [1, 0])
        step.dispose()
    plan.set([s, other], [1, 0])  # `reads` alone is left
    reads.execute()
    with pytest.raises(S.InvalidOperationException):
        append()
    context.synchronize()
    reads.dispose()
    plan.set([s, other], [1, 0])
    plan.dispose()


def test_page_moves_on_a_plans_stream(context, device):  # noqa: F811
    # A position is appended on another stream, behind page copies that keep it busy; a fork made after it on the same stream
    # holds the position in a page of its own.
    layout = CacheLayout(64, 2, 64, 32, F16)
    pool = Pool(context, device, layout, 400)
    c = pool.cache
    pool.host[...] = 0
    pool.upload()
    s = c.open()
    c.extend([s], [40])
    kv = rng(5).standard_normal((1, 2 * 64)).astype(np.float32)
    q, dkv, out = device(np.zeros((1, 2 * 64), np.float32)), device(kv), device(np.zeros((1, 2 * 64), np.float32))
    plan = c.plan(2)
    context.synchronize()
    with S.HipContext(0) as elsewhere:
        stream = elsewhere.stream
        plan.set([s], [1], stream)
        for _ in range(40):
            c.copy_pages(range(10, 200), range(200, 390), stream)
        plan.append(63, q, 0, out, dkv, 0, dkv, 0, 1e4, 2, stream=stream)
        fork = c.fork(s)[0]
        c.extend([fork], [1], stream)
        twin = c.copy(s, stream)
        c.free([s])
        c.compact(stream)
        elsewhere.synchronize()
    pool.download()
    assert len({c.pages(t)[1] for t in (fork, twin)}) == 2
    for t in (fork, twin):
        assert np.array_equal(pool.of(t, 63)[1][39], kv.reshape(2, 64).astype(np.float16).astype(np.float64)), t
    plan.dispose()
