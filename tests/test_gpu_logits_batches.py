"""Rules of logits at sizes that change how a launch works: histories of nearly 2^31 tokens, and workgroups of several rows. The
definition in FP32, the same bits."""
from __future__ import annotations

import numpy as np
import pytest

from helpers import rng
from satori_amd.logits import LOGIT_ROW, LogitBatch
from test_gpu_cache import device  # noqa: F401  (a fixture)
from test_gpu_logits import Batch, expected, make_rules, row, same

pytestmark = pytest.mark.gpu


def test_the_longest_history(context, device):
    # 2^31 - 1 tokens, the most that a length can say: those that are none (-1) but for the first and the last few.
    v, length = 64, 2 ** 31 - 1
    logits = rng(5).standard_normal((2, v)).astype(np.float32)
    some = np.full(1 << 26, -1, np.int32)
    history = context.alloc(length * 4)
    try:
        for first in range(0, length, some.size):
            context.upload(history + 4 * first, some[:min(some.size, length - first)])
        context.upload(history, np.array([9], np.int32))
        context.upload(history + 4 * (length - 5), np.array([5, 7, 5, 5, 63], np.int32))
        rows = [row(1.0, 1.0, 0.5, 0), row(1.5, 0.0, 0.25, 0, token=7)]
        rules = make_rules(context, v, [])
        out, best = device(np.zeros_like(logits)), device(np.zeros(2, np.int32))
        rules.apply(LogitBatch(rows=device(np.array(rows, LOGIT_ROW)), count=2, logits=device(logits), logits_stride=v, output=out,
                               output_stride=v, best=best, history=history, history_stride=length, histories=1,
                               lengths=device(np.array([length], np.int32))))
        want, chosen = expected(logits, rows, [[9, 5, 7, 5, 5, 63]], [], [])
        assert same(context.download(np.zeros_like(logits), out), want)
        assert np.array_equal(context.download(np.zeros(2, np.int32), best), chosen)
        rules.dispose()
    finally:
        context.free(history)


# A workgroup takes slices * rows / 4096 rows, 1 to 16 (slices of 4096 tokens, at most 1024 rows a launch), one after another: what one
# row leaves in its counts, its lists, its biases and its branch is undone or kept for the next. Below two, three and sixteen of them,
# with rows left over for the last one.

def several(g, v, n):
    """Rows in runs that share a history, among them ones without penalties; every kind of parent, bias set and mask."""
    dense = g.permutation(4096)[:3000].tolist()  # (more of a slice's tokens than the list of them holds)
    histories = [[], g.integers(0, v, 900).tolist(), dense + g.integers(0, v, 50).tolist(), g.integers(0, 64, 400).tolist(),
                 [v - 1, 0, v, -1, v - 1]]
    # More than 256 entries in one slice, few, and none.
    sets = [{int(t): float(np.float32(b)) for t, b in zip(g.permutation(min(v, 4096))[:700], g.standard_normal(700) * 5)},
            {int(t): float(np.float32(b)) for t, b in zip(g.integers(0, v, 5), g.standard_normal(5) * 5)}, {}]
    masks = [g.random(v) < 0.5, g.random(v) < 0.001, np.zeros(v, bool)]
    penalties = [(1.3, 0.5, 0.25), (0.7, -0.5, 0.1), (1.0, 1.5, 0.0), (1.0, 0.0, 0.0)]
    rows, history, biases = [], -1, -1
    for i in range(n):
        if g.random() < 0.3:
            history = int(g.integers(-1, len(histories) + 1))
        if g.random() < 0.4:
            biases = int(g.integers(-1, len(sets) + 1))
        parent = [i - 1, int(g.integers(-1, i)) if i else -1, i - 70, -1, i + 1][int(g.choice(5, p=[0.55, 0.2, 0.1, 0.1, 0.05]))]
        token = int(g.integers(0, v)) if g.random() < 0.5 else int(g.integers(-1, 64))
        rows.append(row(*penalties[int(g.choice(4, p=[0.4, 0.2, 0.15, 0.25]))], history=history, parent=max(parent, -1) if i % 40 else -1,
                        token=token, biases=biases, mask=int(g.integers(-1, 8))))
    return rows, histories, sets, masks


@pytest.mark.parametrize("v,n,outputs", [
    (8 * 4096 - 5, 1024, ("apart", "in place", "none")),     # two
    (8 * 4096 - 5, 1025 + 1023, ("apart",)),                 # two of each of two launches
    (19 * 4096 + 1, 700, ("apart", "in place")),             # three, and one row over
    (64 * 4096, 1024, ("in place",)),                        # sixteen
])
def test_several_rows_of_a_workgroup(context, device, v, n, outputs):
    g = rng(v + n)
    logits = g.standard_normal((n, v), np.float32) * 3
    rows, histories, sets, masks = several(g, v, n)
    rules = make_rules(context, v, sets)
    want, best = expected(logits, rows, histories, sets, masks)
    for output in outputs:
        b = Batch(context, device, logits, rows, histories, masks, output=output)
        rules.apply(b.call)
        got, chosen = b.result()
        assert got is None or same(got, want)
        assert np.array_equal(chosen, best)
    rules.dispose()
