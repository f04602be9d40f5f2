"""Drafts verified by steps that were captured once: append, attention and the rules of logits replayed over batches of other trees,
with everything that a replay is to write spoiled before it. The plain loop's tokens, and the bits of eager calls."""
from __future__ import annotations

import numpy as np
import pytest

from helpers import rng
from satori_amd.cache import CacheLayout
from satori_amd.logits import LOGIT_ROW, LogitBatch, LogitRules
from satori_amd.rotary import Rotation, RotaryLayout
from test_gpu_cache import F16, F32, Pool, device  # noqa: F401  (device: a fixture)
from test_gpu_draft_step import (BIASED, HEAD_DIM, HEADS, KV_HEADS, PENALTIES, ROWS, VOCABULARY, Model, allowed, drafts, plainly)
from test_gpu_trees import star

pytestmark = pytest.mark.gpu

LARGEST = ROWS // 3  # rows of a request's tree, at most


@pytest.mark.parametrize("type_", [F32, F16])
def test_steps_captured_once_follow_every_tree(context, device, type_):
    model, g = Model(), rng(23)
    half = (lambda x: x.astype(np.float16).astype(np.float64)) if type_ == F16 else (lambda x: x.astype(np.float32).astype(np.float64))
    prompts = [g.integers(0, VOCABULARY, n).tolist() for n in (45, 1, 70)]
    count = 40
    wanted = []
    for r, p in enumerate(prompts):
        tokens, least = plainly(model, r, p, count, half)
        assert least > 1e-4  # (no choice hangs on a rounding)
        wanted.append(tokens)

    pool = Pool(context, device, CacheLayout(1, KV_HEADS, HEAD_DIM, 32, type_), 40)
    cache = pool.cache
    plan = cache.plan(HEADS)
    rotation = Rotation(context, model.frequencies, model.magnitude, RotaryLayout.INTERLEAVED, 64)
    rules = LogitRules(context, VOCABULARY, 1, len(BIASED))
    rules.set_biases(0, list(BIASED), list(BIASED.values()))
    zeros = lambda *shape: device(np.zeros(shape, np.float32))  # noqa: E731
    q, turned, attended = (zeros(ROWS, HEADS * HEAD_DIM) for _ in range(3))
    k, v = zeros(ROWS, KV_HEADS * HEAD_DIM), zeros(ROWS, KV_HEADS * HEAD_DIM)
    logits, best = zeros(ROWS, VOCABULARY), device(np.zeros(ROWS, np.int32))
    stride, words = 200, -(-VOCABULARY // 32)
    history, lengths = device(np.zeros((3, stride), np.int32)), device(np.zeros(3, np.int32))
    masks, table = device(np.zeros((ROWS, words), np.uint32)), device(np.zeros(ROWS, LOGIT_ROW))
    batch = LogitBatch(rows=table, count=ROWS, logits=logits, logits_stride=VOCABULARY, output=logits, output_stride=VOCABULARY, best=best,
                       history=history, history_stride=stride, histories=3, lengths=lengths, masks=masks, mask_count=ROWS,
                       mask_stride=words)

    def attend():
        plan.append_rotated(0, q, 0, turned, k, 0, v, 0, rotation)
        plan.attention(0, turned, attended)

    def spoil(new):
        """Nothing that a step is to write holds a number: the rows' outputs, and the places of their keys and values."""
        for p in (turned, attended):
            context.upload(p, np.full((ROWS, HEADS * HEAD_DIM), np.nan, np.float32))
        pool.download()
        for s, n in zip(sequences, new):
            for at in range(cache.tokens(s) - n, cache.tokens(s)):
                page = cache.pages(s)[at // 32]
                pool.keys(0)[page, :, at % 32] = np.nan
                pool.values(0)[page, :, :, at % 32] = np.nan
        pool.upload()

    def results(n):
        context.synchronize()
        pool.download()
        return ([context.download(np.zeros((ROWS, HEADS * HEAD_DIM), np.float32), p)[:n] for p in (turned, attended)] +
                [np.concatenate([x.ravel() for s in sequences for x in pool.of(s, 0)])])

    # Before the captures a batch as large as any: the longest lists of pages, the largest trees.
    sequences = [cache.open() for _ in prompts]
    longest = [len(p) + count + 8 + LARGEST for p in prompts]
    cache.extend(sequences, longest)
    plan.set_tree(sequences, [star(LARGEST)] * 3)
    attend()
    context.synchronize()
    context.capture_begin()
    attend()
    step = context.capture_end()
    context.capture_begin()
    rules.apply(batch)
    choose = context.capture_end()
    for s in sequences:
        cache.truncate(s, 0)

    def upload(tokens):
        for p, x in zip((q, k, v), model.projections(tokens)):
            context.upload(p, x.astype(np.float32))

    answers = [list(p) for p in prompts]
    for i, p in enumerate(prompts):  # prompts by themselves, but for their last token, by the same step
        if len(p) > 1:
            for first in range(0, len(p) - 1, LARGEST):
                part = p[first:min(first + LARGEST, len(p) - 1)]
                cache.extend([sequences[i]], [len(part)])
                plan.set([sequences[i]], [len(part)])
                upload(part)
                step.execute()
                context.synchronize()
    taken = accepted = 0
    while any(len(a) < len(w) for a, w in zip(answers, wanted)):
        trees = []
        for a, w in zip(answers, wanted):
            tokens, parents = drafts(g, a[-1], w[len(a):])
            trees.append((tokens[:LARGEST], parents[:LARGEST]))
        tokens = [t for tree, _ in trees for t in tree]
        n, new = len(tokens), [len(t) for t, _ in trees]
        cache.extend(sequences, new)
        plan.set_tree(sequences, [p for _, p in trees])
        upload(tokens)
        rows, bits, first = [(1.0, 0.0, 0.0, -1, -1, -1, -1, -1)] * ROWS, np.zeros((ROWS, words * 32), np.uint32), 0
        for r, (tree, parents) in enumerate(trees):
            for j, (t, p) in enumerate(zip(tree, parents)):
                rows[first + j] = (*PENALTIES[r], r, first + p if p >= 0 else -1, t, 0 if r == 1 else -1, first + j)
                bits[first + j, :VOCABULARY] = allowed(r, t)
            first += len(tree)
        past = np.zeros((3, stride), np.int32)
        for r, a in enumerate(answers):
            past[r, :len(a) - 1] = a[:-1]
        context.upload(history, past)
        context.upload(lengths, np.array([len(a) - 1 for a in answers], np.int32))
        context.upload(table, np.array(rows, LOGIT_ROW))
        context.upload(masks, (bits.reshape(ROWS, words, 32) << np.arange(32, dtype=np.uint32)).sum(2, dtype=np.uint32))

        spoil(new)
        step.execute()
        replayed = results(n)
        assert all(np.all(np.isfinite(x)) for x in replayed)
        spoil(new)
        attend()
        for a, b in zip(results(n), replayed):
            assert np.array_equal(a, b)
        x = np.zeros((ROWS, VOCABULARY), np.float32)
        x[:n] = model.logits(tokens, replayed[1].astype(np.float64))
        choices = []
        for go in (choose.execute, lambda: rules.apply(batch)):
            context.upload(logits, x)
            context.upload(best, np.full(ROWS, -5, np.int32))
            go()
            choices.append((context.download(np.zeros(ROWS, np.int32), best), context.download(np.zeros_like(x), logits)))
        assert all(np.array_equal(a, b) for a, b in zip(*choices))
        choice = choices[0][0]
        kept, first = [], 0
        for r, (tree, parents) in enumerate(trees):
            way = [0]
            answers[r].append(int(choice[first]))
            while True:
                following = [j for j, p in enumerate(parents) if p == way[-1] and tree[j] == answers[r][-1]]
                if not following:
                    break
                way.append(following[0])
                answers[r].append(int(choice[first + following[0]]))
            kept.append(way)
            first += len(tree)
            accepted += len(way) - 1
        plan.keep(kept)
        for s, a in zip(sequences, answers):
            cache.truncate(s, len(a) - 1)
        taken += 1
        assert all(len(a) <= n - LARGEST for a, n in zip(answers, longest))
    for a, w in zip(answers, wanted):
        assert a[:len(w)] == w
    assert accepted > 30 and taken < 40
    context.synchronize()
    for s in (step, choose):
        s.dispose()
    plan.dispose()
    rotation.dispose()
    rules.dispose()
