"""The operators for drafted trees together, as a host that verifies drafts runs them: a prompt, then steps that write a tree's
positions (scaled, interleaved rotation), attend it, put penalties, a bias and a grammar to its logits, take the branch that
the best tokens agree with, keep its rows and cut the rest. Three requests must come to the tokens that a plain loop
in 64 bits comes to one at a time, whatever was drafted, eagerly and as a captured step."""
from __future__ import annotations

import numpy as np
import pytest

from helpers import rng
from satori_amd.cache import CacheLayout
from satori_amd.logits import LOGIT_ROW, LogitBatch, LogitRules
from satori_amd.rotary import Rotation, RotaryLayout, RotaryScaling, rotary_frequencies
from test_gpu_cache import F16, F32, Pool, device  # noqa: F401  (device: a fixture)
from test_gpu_trees import rotated

pytestmark = pytest.mark.gpu

VOCABULARY, HIDDEN, HEADS, KV_HEADS, HEAD_DIM, ROTARY = 517, 96, 6, 2, 48, 32
ROWS = 48  # of a step, at most
PENALTIES = [(1.2, 0.4, 0.1), (1.0, 0.0, 0.0), (1.3, 0.0, 0.3)]
BIASED = {7: 1.5, 400: 2.0}


class Model:
    """One attention layer between an embedding and an output projection, on the host in 64 bits."""

    def __init__(self):
        g = rng(7)
        self.embedding = g.standard_normal((VOCABULARY, HIDDEN))
        self.q, self.k, self.v = (g.standard_normal((HIDDEN, n * HEAD_DIM)) * HIDDEN ** -0.5 for n in (HEADS, KV_HEADS, KV_HEADS))
        self.out = g.standard_normal((HEADS * HEAD_DIM, HIDDEN)) * (HEADS * HEAD_DIM) ** -0.5
        self.head = g.standard_normal((HIDDEN, VOCABULARY)) * 0.4
        self.frequencies, self.magnitude = rotary_frequencies(ROTARY, 1e4, RotaryScaling.WAVELENGTH, 4.0, 64, 1.0, 4.0)

    def projections(self, tokens):
        x = self.embedding[tokens]
        return [(x @ w).reshape(len(tokens), -1, HEAD_DIM) for w in (self.q, self.k, self.v)]

    def logits(self, tokens, attended):
        return np.tanh(self.embedding[tokens] + 3 * attended.reshape(len(tokens), -1) @ self.out) @ self.head

    def turn(self, x, positions):
        return rotated(x, positions, self.frequencies, self.magnitude, True)


def allowed(request, token):
    """A grammar: which tokens may follow one."""
    mask = np.ones(VOCABULARY, bool)
    if request == 2:
        mask[:] = np.arange(VOCABULARY) % 5 == (token + 1) % 5
    return mask


def chosen(request, logits, had):
    repetition, presence, frequency = PENALTIES[request]
    count = np.bincount(had, minlength=VOCABULARY)
    x = np.where(logits > 0, logits / repetition, logits * repetition) - (presence + frequency * count)
    x = np.where(count > 0, x, logits)
    if request == 1:
        for t, b in BIASED.items():
            x[t] += b
    x[~allowed(request, had[-1])] = -np.inf
    best = int(x.argmax())
    return best, x[best] - np.delete(x, best).max()


def plainly(model, request, prompt, count, exactly):
    """`count` tokens after a prompt, one at a time; keys and values kept as the cache keeps them."""
    tokens, keys, values, least = list(prompt), [], [], np.inf
    for _ in range(count):
        for position in range(len(keys), len(tokens)):
            _, k, v = model.projections([tokens[position]])
            keys.append(exactly(model.turn(k.astype(np.float32), [position])[0]))
            values.append(exactly(v[0].astype(np.float32)))
        q = model.turn(model.projections([tokens[-1]])[0].astype(np.float32), [len(tokens) - 1])[0]
        k, v = np.array(keys), np.array(values)
        attended = np.zeros((HEADS, HEAD_DIM))
        for h in range(HEADS):
            s = k[:, h * KV_HEADS // HEADS] @ q[h] / np.sqrt(HEAD_DIM)
            p = np.exp(s - s.max())
            attended[h] = p @ v[:, h * KV_HEADS // HEADS] / p.sum()
        best, gap = chosen(request, model.logits(tokens[-1:], attended[None])[0], np.array(tokens))
        least = min(least, gap)
        tokens.append(best)
    return tokens, least


def drafts(g, last, true):
    """A tree behind a request's last token: right and wrong continuations in several branches."""
    tokens, parents = [last], [-1]
    depth, at = int(g.integers(0, 6)), 0
    for i in range(depth):
        for _ in range(int(g.integers(0, 3))):
            tokens.append(int(g.integers(0, VOCABULARY)))
            parents.append(int(g.integers(0, len(parents))))
        if i < len(true):
            tokens.append(int(true[i]))
            parents.append(at)
            at = len(tokens) - 1
    return tokens, parents


@pytest.mark.parametrize("type_", [F32, F16])
@pytest.mark.parametrize("captured", [False, True])
def test_verified_drafts_come_to_the_plain_loops_tokens(context, device, type_, captured):
    model, g = Model(), rng(11)
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

    def attend():
        plan.append_rotated(0, q, 0, turned, k, 0, v, 0, rotation)
        plan.attention(0, turned, attended)

    def batch(rows):
        return LogitBatch(rows=table, count=rows, logits=logits, logits_stride=VOCABULARY, output=logits, output_stride=VOCABULARY,
                          best=best, history=history, history_stride=stride, histories=3, lengths=lengths, masks=masks,
                          mask_count=ROWS, mask_stride=words)

    def upload(tokens):
        for p, x in zip((q, k, v), model.projections(tokens)):
            context.upload(p, x.astype(np.float32))

    sequences = [cache.open() for _ in prompts]
    answers = [list(p) for p in prompts]
    for s, p in zip(sequences, prompts):  # prompts in chunks, but for their last token
        for first in range(0, len(p) - 1, ROWS):
            part = p[first:min(first + ROWS, len(p) - 1)]
            cache.extend([s], [len(part)])
            plan.set([s], [len(part)])
            upload(part)
            attend()
            context.synchronize()
    steps = {}
    taken = accepted = 0
    while any(len(a) < len(w) for a, w in zip(answers, wanted)):
        trees = [drafts(g, a[-1], w[len(a):]) for a, w in zip(answers, wanted)]
        tokens = [t for tree, _ in trees for t in tree]
        n = len(tokens)
        cache.extend(sequences, [len(t) for t, _ in trees])
        plan.set_tree(sequences, [p for _, p in trees])
        upload(tokens)
        rows, bits, first = [], np.zeros((n, words * 32), np.uint32), 0
        for r, (tree, parents) in enumerate(trees):
            for j, (t, p) in enumerate(zip(tree, parents)):
                rows.append((*PENALTIES[r], r, first + p if p >= 0 else -1, t, 0 if r == 1 else -1, len(rows)))
                bits[len(rows) - 1, :VOCABULARY] = allowed(r, t)
            first += len(tree)
        past = np.zeros((3, stride), np.int32)
        for r, a in enumerate(answers):
            past[r, :len(a) - 1] = a[:-1]
        context.upload(history, past)
        context.upload(lengths, np.array([len(a) - 1 for a in answers], np.int32))
        context.upload(table, np.array(rows, LOGIT_ROW))
        context.upload(masks, (bits.reshape(n, words, 32) << np.arange(32, dtype=np.uint32)).sum(2, dtype=np.uint32))
        if captured:
            if n not in steps:  # (a step for each number of rows)
                attend()  # (a plan that has held a tree before its first capture)
                context.synchronize()
                context.capture_begin()
                attend()
                one = context.capture_end()
                context.capture_begin()
                rules.apply(batch(n))
                steps[n] = one, context.capture_end()
            steps[n][0].execute()
        else:
            attend()
        got = context.download(np.zeros((n, HEADS * HEAD_DIM), np.float32), attended)
        context.upload(logits, model.logits(tokens, got.astype(np.float64)).astype(np.float32))
        steps[n][1].execute() if captured else rules.apply(batch(n))
        choice = context.download(np.zeros(n, np.int32), best)
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
        if captured:  # (the plan is read by steps: they go before a batch that would not fit)
            for pair in steps.values():
                for step in pair:
                    step.dispose()
            steps.clear()
        taken += 1
    for a, w in zip(answers, wanted):
        assert a[:len(w)] == w
    assert accepted > 30 and taken < 40
    context.synchronize()
    plan.dispose()
    rotation.dispose()
    rules.dispose()
