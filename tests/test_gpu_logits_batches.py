"""Rules of logits at sizes that change how a launch works: histories of nearly 2^31 tokens. The definition in FP32, the same
bits."""
from __future__ import annotations

import numpy as np
import pytest

from helpers import rng
from satori_amd.logits import LOGIT_ROW, LogitBatch
from test_gpu_cache import device  # noqa: F401  (a fixture)
from test_gpu_logits import expected, make_rules, row, same

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
