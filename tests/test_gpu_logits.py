"""Penalties, biases, grammar masks and best tokens against the definition in FP32, operation for operation: the same bits."""
from __future__ import annotations

import numpy as np
import pytest

import satori_amd as S
from helpers import rng
from satori_amd.logits import LOGIT_ROW, LogitBatch, LogitRules
from test_gpu_cache import device  # noqa: F401  (a fixture)

pytestmark = pytest.mark.gpu


def row(repetition=1.0, presence=0.0, frequency=0.0, history=-1, parent=-1, token=-1, biases=-1, mask=-1):
    return (repetition, presence, frequency, history, parent, token, biases, mask)


def expected(logits, rows, histories, sets, masks):
    """Rows as `row` gives them, histories as token lists, sets as dicts, masks as boolean arrays."""
    out, best = logits.copy(), []
    v = logits.shape[1]
    f = np.float32
    for i, (rep, presence, frequency, history, parent, token, biases, mask) in enumerate(rows):
        had = list(histories[history]) if 0 <= history < len(histories) else []
        at = i
        while True:
            had.append(rows[at][5])
            if not 0 <= rows[at][4] < at:
                break
            at = rows[at][4]
        had = np.array([t for t in had if 0 <= t < v], np.int64)
        count = np.bincount(had, minlength=v)
        x, n = out[i], count > 0
        with np.errstate(all="ignore"):
            l = np.where(x > 0, x / f(rep), x * f(rep)).astype(f)
            l = l - (f(presence) + f(frequency) * count.astype(f))
        x[n] = l[n]
        if 0 <= biases < len(sets):
            for t, b in sets[biases].items():
                if b != 0:
                    with np.errstate(all="ignore"):
                        x[t] = x[t] + f(b)
        if 0 <= mask < len(masks):
            x[~masks[mask]] = -np.inf
        top = np.nanmax(np.append(x, f(-np.inf)))
        best.append(int(np.flatnonzero(x == top)[0]) if top > -np.inf else -1)
    return out, np.array(best, np.int32)


class Batch:
    """A call's arrays on the device."""

    def __init__(self, context, device, logits, rows, histories=(), masks=(), stride=0, output="apart", best=True, history_stride=0,
                 mask_stride=0, place=0):
        self.context, self.logits = context, logits
        n, v = logits.shape
        self.stride = stride or v
        whole = np.full(place + n * self.stride + 8, 3, np.float32)
        for i in range(n):
            whole[place + i * self.stride:][:v] = logits[i]
        self.whole, self.place = whole, place
        self.source = device(whole)
        self.output = {"apart": device(np.full_like(whole, 9)) if output == "apart" else 0, "in place": self.source, "none": 0}[output]
        self.kind = output
        self.best = device(np.full(n, -5, np.int32)) if best else 0
        longest = max([history_stride] + [len(h) for h in histories])
        table = np.full((max(len(histories), 1), max(longest, 1)), 0, np.int32)
        for i, h in enumerate(histories):
            table[i, :len(h)] = h
        words = max(mask_stride, -(-v // 32))
        bits = np.full((max(len(masks), 1), words), 0xffffffff, np.uint32)
        for i, m in enumerate(masks):
            padded = np.zeros(words * 32, np.uint32)
            padded[:v] = m
            bits[i] = (padded.reshape(-1, 32) << np.arange(32, dtype=np.uint32)).sum(1, dtype=np.uint32)
        self.rows = device(np.array(rows, LOGIT_ROW))
        self.lengths = device(np.array([len(h) for h in histories] or [0], np.int32))
        self.arguments = dict(
            rows=self.rows, count=n, logits=self.source + 4 * place, logits_stride=self.stride,
            output=self.output + 4 * place if self.output else 0, output_stride=self.stride, best=self.best, history=device(table),
            history_stride=table.shape[1], histories=len(histories), lengths=self.lengths, masks=device(bits), mask_count=len(masks),
            mask_stride=words)
        self.call = LogitBatch(**self.arguments)

    def result(self):
        n, v = self.logits.shape
        got = None
        if self.output:
            whole = self.context.download(np.zeros_like(self.whole), self.output)
            got = np.stack([whole[self.place + i * self.stride:][:v] for i in range(n)])
            outside = np.ones(whole.size, bool)
            for i in range(n):
                outside[self.place + i * self.stride:][:v] = False
            assert np.all(whole[outside] == (9 if self.kind == "apart" else 3))
        best = self.context.download(np.zeros(n, np.int32), self.best) if self.best else None
        return got, best


def same(a, b):
    return np.array_equal(a, b, equal_nan=True)


def make_rules(context, vocabulary, sets):
    rules = LogitRules(context, vocabulary, len(sets), max([len(s) for s in sets] + [0]))
    for i, s in enumerate(sets):
        rules.set_biases(i, list(s), list(s.values()))
    return rules


def case(g, v, n, lists=3, longest=500, coarse=False):
    logits = (g.standard_normal((n, v)) * 3).astype(np.float32)
    if coarse:
        logits = np.round(logits * 4) / 4
    histories = [g.integers(0, v, g.integers(0, longest)).tolist() + g.integers(0, max(1, v // 50), 60).tolist() for _ in range(lists)]
    sets = [{int(t): float(np.float32(b)) for t, b in zip(g.permutation(v)[:min(v, 40)], g.standard_normal(40) * 5)} for _ in range(2)] + [{}]
    masks = [g.random(v) < 0.5, g.random(v) < 0.01, np.zeros(v, bool), np.ones(v, bool)]
    rows = []
    for i in range(n):
        rows.append(row(*[(1.0, 0.0, 0.0), (1.3, 0.5, 0.25), (0.7, -0.5, 0.1), (1.0, 1.5, 0.0)][i % 4], history=int(g.integers(-1, lists + 1)),
                        parent=int(g.integers(-1, i)) if i and i % 3 else -1, token=int(g.integers(-1, v)),
                        biases=int(g.integers(-1, 4)), mask=int(g.integers(-1, 5))))
    return logits, rows, histories, sets, masks


@pytest.mark.parametrize("v", [1, 2, 31, 32, 33, 1001, 4095, 4096, 4097, 8193, 32003])
@pytest.mark.parametrize("output", ["apart", "in place", "none"])
def test_rows_of_all_kinds(context, device, v, output):
    g = rng(v)
    logits, rows, histories, sets, masks = case(g, v, 23, coarse=v % 2 == 0)
    rules = make_rules(context, v, sets)
    want, best = expected(logits, rows, histories, sets, masks)
    for stride, place in ((0, 0), (v + 5, 3)):
        b = Batch(context, device, logits, rows, histories, masks, stride, output, place=place, history_stride=700, mask_stride=v // 32 + 3)
        rules.apply(b.call)
        got, chosen = b.result()
        assert got is None or same(got, want)
        assert np.array_equal(chosen, best)
    b = Batch(context, device, logits, rows, histories, masks, best=False)
    rules.apply(b.call)
    assert same(b.result()[0], want)
    rules.dispose()


def test_a_large_vocabulary_and_long_histories(context, device):
    g = rng(2)
    logits, rows, histories, sets, masks = case(g, 151936, 40, longest=20000)
    rules = make_rules(context, 151936, sets)
    want, best = expected(logits, rows, histories, sets, masks)
    b = Batch(context, device, logits, rows, histories, masks)
    rules.apply(b.call)
    got, chosen = b.result()
    assert same(got, want) and np.array_equal(chosen, best)
    rules.dispose()


@pytest.mark.parametrize("n", [70, 1024, 1025, 2500])
def test_branches_and_many_rows(context, device, n):
    # Chains longer than any window, trees, and parents that are none.
    g = rng(n)
    v = 300
    logits = (g.standard_normal((n, v)) * 3).astype(np.float32)
    rows = []
    for i in range(n):
        parent = [i - 1, int(g.integers(-1, i)) if i else -1, max(-1, i - 70), i - 1, i][int(g.integers(0, 5))] if i % 50 else -1
        rows.append(row(1.1, 0.5, 0.25, parent=[parent, i - 1][n == 70], token=int(g.integers(0, v))))
    rows[n // 2] = row(1.1, 0.5, 0.25, parent=n + 5, token=7)
    rows[n // 3] = row(1.1, 0.5, 0.25, parent=-7, token=7)
    rules = make_rules(context, v, [])
    want, best = expected(logits, rows, [], [], [])
    b = Batch(context, device, logits, rows)
    for _ in range(2):
        rules.apply(b.call)
        got, chosen = b.result()
        assert same(got, want) and np.array_equal(chosen, best)
    rules.dispose()


def test_rows_of_a_tree_share_a_history(context, device):
    # Several rows with one history, in runs of every length, among rows with others and with none.
    g = rng(77)
    v, n = 5000, 90
    logits = (g.standard_normal((n, v)) * 3).astype(np.float32)
    histories = [g.integers(0, v, k).tolist() for k in (0, 1, 37, 900, 4100)]
    rows, owner = [], 0
    for i in range(n):
        owner = int(g.integers(-1, 6)) if g.random() < 0.25 else owner
        rows.append(row(*[(1.2, 0.1, 0.3), (1.0, 0.0, 0.0)][i % 7 == 3], history=owner, parent=i - 1 if i % 4 else -1,
                        token=int(g.integers(0, v))))
    rules = make_rules(context, v, [])
    want, best = expected(logits, rows, histories, [], [])
    b = Batch(context, device, logits, rows, histories)
    rules.apply(b.call)
    got, chosen = b.result()
    assert same(got, want) and np.array_equal(chosen, best)
    rules.dispose()


def test_values_at_the_edges(context, device):
    v = 4200
    f = np.float32
    logits = np.zeros((9, v), f)
    logits[0] = -np.inf                       # nothing to choose
    logits[1] = -np.inf
    logits[1, 4199] = np.finfo(f).min         # the only one
    logits[2] = np.nan
    logits[2, 70] = -5                        # the only number
    logits[3] = np.nan                        # none
    logits[4, :] = -0.0
    logits[4, 9] = 0.0                        # zeros are equal: the lowest
    logits[5, 4100] = np.inf
    logits[5, 4150] = np.inf
    logits[6] = np.finfo(f).smallest_subnormal
    logits[6, 33] = 3 * np.finfo(f).smallest_subnormal
    logits[7, ::3] = [np.nan, np.inf, -np.inf, 1.0] * 350
    logits[8, 1] = np.finfo(f).max
    masks = [np.arange(v) % 3 != 0]
    sets = [{5: np.inf, 6: -np.inf, 7: 0.0, 8: float(np.finfo(f).max), 4199: 2.0, 1: float(np.finfo(f).max)}]
    histories = [list(range(0, v, 2)) * 3]
    for rows in ([row()] * 9, [row(2.0, 0.0, 0.0, 0)] * 9, [row(2.0, 1.0, 0.5, 0, biases=0, mask=0)] * 9, [row(biases=0)] * 9,
                 [row(mask=0)] * 9):
        rules = make_rules(context, v, sets)
        want, best = expected(logits, rows, histories, sets, masks)
        b = Batch(context, device, logits, rows, histories, masks)
        rules.apply(b.call)
        got, chosen = b.result()
        assert same(got, want) and np.array_equal(chosen, best)
        # A logit that nothing concerns keeps its bits.
        if rows[0] == row():
            assert np.array_equal(got.view(np.uint32), logits.view(np.uint32))
        rules.dispose()


def test_biases_that_change(context, device):
    g = rng(13)
    v = 9000
    logits = g.standard_normal((2, v)).astype(np.float32)
    rules = LogitRules(context, v, 2, v)
    b = Batch(context, device, logits, [row(biases=0), row(biases=1)])
    for s in ({}, {int(t): 3.5 for t in g.permutation(v)}, {v - 1: 100.0}, {0: 50.0, 4096: -1.0, 4095: 9.0}, {}):
        rules.set_biases(1, list(s), list(s.values()))
        rules.apply(b.call)
        want, best = expected(logits, [row(biases=0), row(biases=1)], [], [{}, s], [])
        got, chosen = b.result()
        assert same(got, want) and np.array_equal(chosen, best)
    rules.dispose()


def test_captured_calls_read_what_the_arrays_hold(context, device):
    g = rng(21)
    v, n = 12345, 12
    logits, rows, histories, sets, masks = case(g, v, n)
    rules = make_rules(context, v, sets)
    b = Batch(context, device, logits, rows, histories, masks)
    context.capture_begin()
    rules.apply(b.call)
    with pytest.raises(S.InvalidOperationException):
        rules.set_biases(0, [1], [1.0])
    step = context.capture_end()
    with pytest.raises(S.ArgumentException):
        rules.dispose()
    for i in range(4):
        rows = [rows[(i + j) % n][:3] + rows[j][3:] for j in range(n)]
        histories = [h[:len(h) // (i + 1)] for h in histories]
        sets[0] = {i: 30.0 * i}
        rules.set_biases(0, list(sets[0]), list(sets[0].values()))
        context.upload(b.rows, np.array(rows, LOGIT_ROW))
        context.upload(b.lengths, np.array([len(h) for h in histories], np.int32))
        step.execute()
        got, chosen = b.result()
        want, best = expected(logits, rows, histories, sets, masks)
        assert same(got, want) and np.array_equal(chosen, best)
        rules.apply(b.call)
        assert same(b.result()[0], got) and np.array_equal(b.result()[1], chosen)
    step.dispose()
    rules.dispose()


def test_lengths_that_say_too_much(context, device):
    # A history's length is at most its stride, and at least nothing.
    v = 50
    logits = np.ones((2, v), np.float32)
    rows = [row(1.0, 1.0, 0.0, 0), row(1.0, 1.0, 0.0, 1)]
    b = Batch(context, device, logits, rows, [[1, 2, 3], [4, 5, 6]])
    rules = make_rules(context, v, [])
    context.upload(b.lengths, np.array([2 ** 31 - 1, -3], np.int32))
    rules.apply(b.call)
    want, best = expected(logits, rows, [[1, 2, 3], []], [], [])
    got, chosen = b.result()
    assert same(got, want) and np.array_equal(chosen, best)
    rules.dispose()


def test_rows_behind_the_fourth_gibibyte(context, device):
    v, n, stride = 500, 3, 1_600_000_001
    g = rng(14)
    logits = g.standard_normal((n, v)).astype(np.float32)
    p, best = context.alloc(((n - 1) * stride + v) * 4), device(np.zeros(n, np.int32))
    for i in range(n):
        context.upload(p + i * stride * 4, logits[i])
    history = [[1, 1, 2, 499]]
    rows = [row(1.5, 0.25, 0.5, 0), row(), row(1.0, 1.0, 0.0, 0, parent=1, token=7)]
    rules = make_rules(context, v, [])
    rules.apply(LogitBatch(rows=device(np.array(rows, LOGIT_ROW)), count=n, logits=p, logits_stride=stride, output=p, output_stride=stride,
                           best=best, history=device(np.array(history, np.int32)), history_stride=4, histories=1,
                           lengths=device(np.array([4], np.int32))))
    got = np.stack([context.download(np.zeros(v, np.float32), p + i * stride * 4) for i in range(n)])
    chosen = context.download(np.zeros(n, np.int32), best)
    context.free(p)
    want, expected_best = expected(logits, rows, history, [], [])
    assert same(got, want) and np.array_equal(chosen, expected_best)
    rules.dispose()


def test_refused_calls(context, device):
    for bad in ((0, 0, 0), (-1, 0, 0), (10, -1, 0), (10, 1, -1), (10, 1, 11), (2 ** 28 + 1, 0, 0)):
        with pytest.raises(S.ArgumentOutOfRangeException):
            LogitRules(context, *bad)
    rules = LogitRules(context, 100, 2, 5)
    for index, tokens, values in ((2, [1], [1.0]), (-1, [1], [1.0]), (0, [100], [1.0]), (0, [-1], [1.0]), (0, [1], [np.nan]),
                                  (0, [1, 2, 3, 4, 5, 6], [1.0] * 6)):
        with pytest.raises(S.ArgumentOutOfRangeException):
            rules.set_biases(index, tokens, values)
    for tokens, values in (([1, 1], [1.0, 2.0]), ([1], [1.0, 2.0])):
        with pytest.raises(S.ArgumentException):
            rules.set_biases(0, tokens, values)
    b = Batch(context, device, np.zeros((3, 100), np.float32), [row()] * 3, [[1]], [np.ones(100, bool)])
    apply = lambda **k: rules.apply(LogitBatch(**{**b.arguments, **k}))  # noqa: E731
    apply(count=0)
    apply(histories=0, history=0, lengths=0, mask_count=0, masks=0)
    for bad in (dict(count=-1), dict(histories=-1), dict(mask_count=-1), dict(logits_stride=99), dict(output_stride=99),
                dict(mask_stride=3), dict(history_stride=-1), dict(logits_stride=2 ** 62)):
        with pytest.raises(S.ArgumentOutOfRangeException):
            apply(**bad)
    for bad in (dict(rows=0), dict(logits=0), dict(history=0), dict(lengths=0), dict(masks=0)):
        with pytest.raises(S.ArgumentNullException):
            apply(**bad)
    for bad in (dict(output=0, best=0), dict(output=b.source + 4), dict(output=b.source, output_stride=101), dict(best=b.source + 8),
                dict(best=b.output), dict(logits=b.source + 2), dict(best=b.rows), dict(output=b.arguments["masks"], count=1),
                dict(best=b.lengths, count=1)):
        with pytest.raises(S.ArgumentException):
            apply(**bad)
    apply()
    got, chosen = b.result()
    assert not got.any() and not chosen.any()
    rules.dispose()
    rules.dispose()
    with pytest.raises(S.ObjectDisposedException):
        apply()
    with pytest.raises(S.ObjectDisposedException):
        rules.set_biases(0, [1], [1.0])


def test_strides_of_what_is_not_there_are_not_looked_at(context, device):
    rules = LogitRules(context, 100)
    b = Batch(context, device, np.arange(300, dtype=np.float32).reshape(3, 100), [row()] * 3, [[1]], [np.ones(100, bool)])
    for stride in (2 ** 63 - 1, -2 ** 63):
        rules.apply(LogitBatch(**{**b.arguments, "output": 0, "output_stride": stride, "histories": 0, "history_stride": stride,
                                  "mask_count": 0, "mask_stride": stride}))
        assert context.download(np.zeros(3, np.int32), b.arguments["best"]).tolist() == [99] * 3
    rules.dispose()


def test_rules_keep_their_context(device):
    other = S.HipContext(0)
    rules = LogitRules(other, 10)
    with pytest.raises(S.ArgumentException):
        other.dispose()
    rules.dispose()
    other.dispose()
