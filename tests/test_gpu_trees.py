"""Drafted trees over the paged cache: their attention, the write of their positions and the rows that a sequence keeps,
against the definition in 64 bits over the pool's own bytes. Whatever no row may see is NaN. The bound of the attention is
that of test_gpu_cache.py, over the positions that a row sees (in as many tiles as the sequence has)."""
from __future__ import annotations

import numpy as np
import pytest

import satori_amd as S
from helpers import rng
from satori_amd.cache import CacheLayout
from satori_amd.rotary import Rotation, RotaryLayout, RotaryScaling, rotary_frequencies
from test_gpu_cache import E, F16, F32, SHAPES, Pool, device, forked  # noqa: F401  (device: a fixture)

pytestmark = pytest.mark.gpu


def chain(n):
    return list(range(-1, n - 1))


def star(n):
    return [-1] + [0] * (n - 1)


def roots(n):
    return [-1] * n


def binary(n):
    return [(j - 1) // 2 if j else -1 for j in range(n)]


def mixed(n, seed):
    g = rng(seed)
    return [int(g.integers(-1, j)) for j in range(n)]


def branch(parents, row):
    found = [row]
    while parents[found[-1]] >= 0:
        found.append(parents[found[-1]])
    return found[::-1]


def depths(parents):
    return [len(branch(parents, j)) - 1 for j in range(len(parents))]


def check_tree(pool, sequences, trees, heads, q, got, layer=0, label="", without=None):
    """`without`: rows that see this one are not looked at."""
    row = 0
    for s, parents in zip(sequences, trees):
        k, v = pool.of(s, layer)
        context, D = len(k) - len(parents), k.shape[2]
        for j in range(len(parents)):
            if without in branch(parents, j):
                row += 1
                continue
            seen = list(range(context)) + [context + a for a in branch(parents, j)]
            ks, vs, group = k[seen], v[seen], heads // k.shape[1]
            for h in range(heads):
                kh, vh, x = ks[:, h // group], vs[:, h // group], q[row, h].astype(np.float64)
                scores = kh @ x / np.sqrt(D)
                p = np.exp(scores - scores.max())
                p /= p.sum()
                a = (np.abs(kh) @ np.abs(x) / np.sqrt(D)).max()
                bound = 1.01 * (2 * (D + 8) * E * a + 2 * (len(k) / 32 + 80) * E) * (p @ np.abs(vh))
                err = np.abs(got[row, h].astype(np.float64) - p @ vh)
                assert np.all(err <= bound), (f"{label} sequence {s} row {j} head {h}: {err.max()} over "
                                              f"{bound[err.argmax()]}")
            row += 1


def attend_tree(context, device, pool, sequences, trees, heads, g, layer=0, scale=1.0, plan=None, stream=0):
    rows = sum(map(len, trees))
    q = (g.standard_normal((rows, heads, pool.layout.head_dim)) * scale).astype(np.float32)
    made = plan or pool.cache.plan(heads)
    try:
        made.set_tree(sequences, trees)
        out = device(np.full(q.shape, 7, np.float32))
        made.attention(layer, device(q), out)
        return q, context.download(np.zeros(q.shape, np.float32), out)
    finally:
        context.synchronize()
        if not plan:
            made.dispose()


# ---- attention ----

@pytest.mark.parametrize("type_,heads,kv_heads,head_dim,page_tokens", SHAPES)
def test_trees_of_all_kinds(context, device, type_, heads, kv_heads, head_dim, page_tokens):
    g = rng(31 * head_dim + heads)
    pool = Pool(context, device, CacheLayout(2, kv_heads, head_dim, page_tokens, type_), 128)
    trees = [star(2), binary(7), roots(3), chain(5), mixed(33, 1), star(40), binary(1), mixed(64, 2), roots(1) + [-1, 0, 1, 1, 2]]
    contexts = [0, 1, 31, 32, 33, 100, 63, 300, 257]
    sequences = [pool.cache.open() for _ in trees]
    pool.cache.extend(sequences, [c + len(t) for c, t in zip(contexts, trees)])
    pool.write(g, sequences)
    q, got = attend_tree(context, device, pool, sequences, trees, heads, g, layer=1)
    check_tree(pool, sequences, trees, heads, q, got, layer=1)


@pytest.mark.parametrize("type_,heads,kv_heads,head_dim,page_tokens", SHAPES[:10])
def test_trees_behind_a_common_prefix_beside_prompts(context, device, type_, heads, kv_heads, head_dim, page_tokens):
    g = rng(17 * head_dim)
    pool = Pool(context, device, CacheLayout(1, kv_heads, head_dim, page_tokens, type_), 160)
    trees = [binary(15), chain(40), mixed(61, 3), chain(1), star(9), [], roots(5)]
    own = [t + 3 * i for i, t in enumerate(map(len, trees))]
    sequences = forked(pool, 333, own)
    pool.write(g, sequences)
    q, got = attend_tree(context, device, pool, sequences, trees, heads, g)
    check_tree(pool, sequences, trees, heads, q, got)


@pytest.mark.parametrize("type_", [F16, F32])
@pytest.mark.parametrize("rows,heads,kv_heads", [(1024, 2, 1), (300, 8, 8), (128, 14, 2)])
def test_large_trees(context, device, type_, rows, heads, kv_heads):
    g = rng(rows)
    pool = Pool(context, device, CacheLayout(1, kv_heads, 64, 32, type_), 160)
    trees = [mixed(rows, rows)]
    sequences = [pool.cache.open()]
    pool.cache.extend(sequences, [rows + 77])
    pool.write(g, sequences)
    q, got = attend_tree(context, device, pool, sequences, trees, heads, g)
    # (a quarter of the rows: the check in 64 bits is slow)
    keep = np.arange(0, rows, 4)
    k, v = pool.of(sequences[0], 0)
    for j in keep:
        seen = list(range(77)) + [77 + a for a in branch(trees[0], j)]
        for h in range(heads):
            kh, vh, x = k[seen, h * kv_heads // heads], v[seen, h * kv_heads // heads], q[j, h].astype(np.float64)
            scores = kh @ x / 8
            p = np.exp(scores - scores.max())
            p /= p.sum()
            a = (np.abs(kh) @ np.abs(x) / 8).max()
            bound = 1.01 * (2 * (64 + 8) * E * a + 2 * (len(k) / 32 + 80) * E) * (p @ np.abs(vh))
            assert np.all(np.abs(got[j, h] - p @ vh) <= bound)


@pytest.mark.parametrize("type_,heads,kv_heads,head_dim,page_tokens", SHAPES[:8])
def test_what_a_row_does_not_see_never_reaches_it(context, device, type_, heads, kv_heads, head_dim, page_tokens):
    # One draft's key and value are infinite and NaN: the rows behind it show it, the others do not.
    g = rng(head_dim)
    for fill in (np.nan, np.inf):
        pool = Pool(context, device, CacheLayout(1, kv_heads, head_dim, page_tokens, type_), 64)
        trees = [star(30), binary(63), mixed(20, 4)]
        contexts = [35, 100, 0]
        sequences = [pool.cache.open() for _ in trees]
        pool.cache.extend(sequences, [c + len(t) for c, t in zip(contexts, trees)])
        pool.write(g, sequences)
        bad = 2
        for s, c in zip(sequences, contexts):
            page, at = pool.cache.pages(s)[(c + bad) // page_tokens], (c + bad) % page_tokens
            pool.values(0)[page, :, :head_dim, at] = fill
            if fill != fill:
                pool.keys(0)[page, :, at, :head_dim] = fill
        pool.upload()
        q, got = attend_tree(context, device, pool, sequences, trees, heads, g)
        row = 0
        for i, parents in enumerate(trees):
            for j in range(len(parents)):
                if bad in branch(parents, j):
                    assert not np.isfinite(got[row]).any()
                else:
                    assert np.isfinite(got[row]).all(), (i, j)
                row += 1
        check_tree(pool, sequences, trees, heads, q, got, without=bad)


def test_rows_that_follow_one_another_are_no_tree(context, device):
    # The same bits as without parents, also from a plan that has held trees.
    g = rng(5)
    pool = Pool(context, device, CacheLayout(1, 2, 128, 32, F16), 64)
    sequences = [pool.cache.open() for _ in range(3)]
    pool.cache.extend(sequences, [700, 40, 5])
    pool.write(g, sequences)
    new = [20, 40, 1]
    q = g.standard_normal((sum(new), 12, 128)).astype(np.float32)
    dq, out = device(q), device(np.zeros_like(q))
    results = []
    for trees in (False, True, True):
        plan = pool.cache.plan(12)
        if trees and len(results) == 2:
            plan.set_tree(sequences, [star(n) for n in new])
            plan.attention(0, dq, out)
        plan.set_tree(sequences, [chain(n) for n in new]) if trees else plan.set(sequences, new)
        plan.attention(0, dq, out)
        results.append(context.download(np.zeros_like(q), out))
        plan.dispose()
    assert np.array_equal(results[0], results[1]) and np.array_equal(results[0], results[2])


def test_a_long_context(context, device):
    g = rng(12)
    pool = Pool(context, device, CacheLayout(1, 2, 64, 256, F16), 140)
    trees = [mixed(48, 9), binary(31)]
    sequences = [pool.cache.open() for _ in trees]
    pool.cache.extend(sequences, [30000, 4000])
    pool.write(g, sequences)
    q, got = attend_tree(context, device, pool, sequences, trees, 8, g)
    check_tree(pool, sequences, trees, 8, q, got)


# ---- the write of new positions ----

def rotated(x, positions, frequencies, magnitude, interleaved):
    """[rows][heads][head_dim] in 64 bits."""
    r = 2 * len(frequencies)
    out = x.astype(np.float64)
    angle = np.asarray(positions, np.float64)[:, None, None] * frequencies
    sn, cs = np.sin(angle) * magnitude, np.cos(angle) * magnitude
    a, b = (out[..., 0:r:2].copy(), out[..., 1:r:2].copy()) if interleaved else (out[..., :r // 2].copy(), out[..., r // 2:r].copy())
    first, second = a * cs - b * sn, a * sn + b * cs
    if interleaved:
        out[..., 0:r:2], out[..., 1:r:2] = first, second
    else:
        out[..., :r // 2], out[..., r // 2:r] = first, second
    return out


def near(got, want, type_=F32):
    # One rounding to FP32 (half a step, 2^-24) and, of F16, one more (2^-11, or half the smallest step, 2^-25); what 64 bits
    # leave open of the angles below 10^6 and of the sums is under 2^-31 of the largest lanes (here under 16).
    rel = 2.0 ** -24 + (2.0 ** -11 if type_ == F16 else 0)
    return np.abs(got.astype(np.float64) - want) <= 1.001 * rel * np.abs(want) + 2.0 ** -27 + (2.0 ** -25 if type_ == F16 else 0)


@pytest.mark.parametrize("layout", list(RotaryLayout))
@pytest.mark.parametrize("type_,heads,kv_heads,head_dim,rotary,page_tokens", [
    (F32, 12, 2, 128, 128, 32), (F16, 12, 2, 128, 64, 64), (F16, 7, 1, 80, 80, 32), (F32, 3, 3, 33, 2, 32), (F32, 2, 1, 256, 250, 128),
    (F16, 4, 2, 48, 42, 256)])
@pytest.mark.parametrize("table", [0, 90])
def test_the_write_of_a_tree(context, device, layout, type_, heads, kv_heads, head_dim, rotary, page_tokens, table):
    g = rng(head_dim + rotary)
    pool = Pool(context, device, CacheLayout(2, kv_heads, head_dim, page_tokens, type_), 64)
    trees = [binary(15), chain(40), mixed(61, 3), [], roots(5), star(1)]
    own = [len(t) + 5 for t in trees]
    sequences = forked(pool, 77, own)
    rows = sum(map(len, trees))
    q = g.standard_normal((rows, heads, head_dim)).astype(np.float32)
    k, v = (g.standard_normal((rows, kv_heads, head_dim)).astype(np.float32) for _ in range(2))
    bq, bk, bv = (g.standard_normal((n, head_dim)).astype(np.float32) for n in (heads, kv_heads, kv_heads))
    frequencies, magnitude = (rotary_frequencies(rotary, 10000.0, RotaryScaling.YARN, 4.0, 4096) if rotary > 2 else
                              (np.array([0.37]), 1.5))
    rotation = Rotation(context, frequencies, magnitude, layout, table)
    plan = pool.cache.plan(heads)
    plan.set_tree(sequences, trees)
    dq = device(q)
    plan.append_rotated(1, dq, device(bq), dq, device(k), 0, device(v), device(bv), rotation)
    out = context.download(np.zeros_like(q), dq)
    before = pool.host.copy()
    pool.download()
    positions, places = [], []
    for s, t in zip(sequences, trees):
        c = pool.cache.tokens(s) - len(t)
        positions += [c + d for d in depths(t)]
        places += [(pool.cache.pages(s)[(c + j) // page_tokens], (c + j) % page_tokens) for j in range(len(t))]
    interleaved = layout == RotaryLayout.INTERLEAVED
    assert np.all(near(out, rotated(q + bq, positions, frequencies, magnitude, interleaved)))
    want_k, want_v = rotated(k, positions, frequencies, magnitude, interleaved), (v + bv).astype(np.float64)
    for row, (page, at) in enumerate(places):
        got = pool.keys(1)[page, :, at]
        assert np.all(near(got[:, :head_dim], want_k[row], type_)) and not got[:, head_dim:].any()
        assert np.all(near(pool.values(1)[page, :, :head_dim, at], want_v[row], type_))
        # What was written is put back: nothing else has changed.
        pool.keys(1)[page, :, at] = before[page, 1, 0].reshape(kv_heads, page_tokens, -1)[:, at]
        pool.values(1)[page, :, :head_dim, at] = before[page, 1, 1].reshape(kv_heads, -1, page_tokens)[:, :head_dim, at]
    assert np.array_equal(pool.host.view(np.uint8), before.view(np.uint8))
    context.synchronize()
    plan.dispose()
    rotation.dispose()


@pytest.mark.parametrize("table", [False, True])
def test_a_trees_rows_turn_as_rows_at_their_positions(context, device, table):
    # append with plain frequencies, of a tree and of rows one after another that stand for the same positions: the same bits.
    g = rng(3)
    heads, kv, D = 6, 2, 64
    pool = Pool(context, device, CacheLayout(1, kv, D, 32, F32), 64)
    first, second = pool.cache.open(), pool.cache.open()
    tree = binary(15)
    pool.cache.extend([first, second], [50 + 15, 50 + 4])
    q = g.standard_normal((15, heads * D)).astype(np.float32)
    k = g.standard_normal((15, kv * D)).astype(np.float32)
    angles = 0
    if table:
        angles = device(np.zeros(52 * D))
        S.DeviceOps(context).rope_table(52, D, 1e4, angles)
    plan = pool.cache.plan(heads)
    plan.set_tree([first], [tree])
    out = device(np.zeros_like(q))
    plan.append(0, device(q), 0, out, device(k), 0, device(k), 0, 1e4, D, angles, 52 if table else 0)
    got = context.download(np.zeros_like(q), out)
    way = [0, 2, 6, 14]
    plan.set([second], [4])
    plan.append(0, device(q[way]), 0, out, device(k[way]), 0, device(k[way]), 0, 1e4, D, angles, 52 if table else 0)
    want = context.download(np.zeros((4, heads * D), np.float32), out)
    assert np.array_equal(got[way], want)
    pool.download()
    a, b = pool.cache.pages(first), pool.cache.pages(second)
    for i, j in enumerate(way):
        x, y = 50 + j, 50 + i
        assert np.array_equal(pool.keys(0)[a[x // 32], :, x % 32], pool.keys(0)[b[y // 32], :, y % 32])
    plan.dispose()


# ---- rows that a sequence keeps ----

@pytest.mark.parametrize("type_,kv_heads,head_dim,page_tokens,layers", [
    (F16, 2, 128, 32, 3), (F32, 2, 128, 32, 1), (F16, 1, 80, 64, 2), (F32, 3, 33, 256, 2), (F16, 5, 1, 32, 4), (F32, 1, 256, 128, 1)])
@pytest.mark.parametrize("count", [1, 7, 300])
def test_kept_rows(context, device, type_, kv_heads, head_dim, page_tokens, layers, count):
    g = rng(head_dim + count)
    most = 90 if count < 100 else 3
    new = [int(g.integers(1, most + 1)) for _ in range(count)]
    contexts = [int(g.integers(0, 2 * page_tokens)) if count < 100 else 1 for _ in range(count)]
    pages = sum(-(-(c + n) // page_tokens) for c, n in zip(contexts, new)) + 1
    pool = Pool(context, device, CacheLayout(layers, kv_heads, head_dim, page_tokens, type_), pages)
    pool.host[:] = g.standard_normal(pool.host.shape).astype(pool.host.dtype)
    pool.host[:, :, 1, 0, 3] = np.nan
    pool.upload()
    sequences = [pool.cache.open() for _ in new]
    pool.cache.extend(sequences, [c + n for c, n in zip(contexts, new)])
    plan = pool.cache.plan(kv_heads)
    plan.set_tree(sequences, [mixed(n, n) for n in new])
    kept = []
    for i, n in enumerate(new):
        rows = np.sort(g.permutation(n)[:g.integers(0, n + 1)]).tolist()
        kept.append([list(range(n)), rows, [n - 1], [], rows[::-1][::-1]][i % 5])
    plan.keep(kept)
    for s, c, rows in zip(sequences, contexts, kept):
        table = pool.cache.pages(s)
        for i, j in enumerate(rows):
            (a, x), (b, y) = divmod(c + j, page_tokens), divmod(c + i, page_tokens)
            for layer in range(layers):
                pool.keys(layer)[table[b], :, y] = pool.keys(layer)[table[a], :, x]
                pool.values(layer)[table[b], :, :head_dim, y] = pool.values(layer)[table[a], :, :head_dim, x]
    want = pool.host.copy()
    got = pool.download().host
    assert np.array_equal(got.view(np.uint8), want.view(np.uint8))
    plan.dispose()


def test_kept_rows_that_chain_over_one_another(context, device):
    # Each destination is the source before the last: more moves than one launch takes, in their order.
    g = rng(8)
    n = 700
    pool = Pool(context, device, CacheLayout(1, 1, 32, 32, F32), 30)
    pool.host[:] = g.standard_normal(pool.host.shape).astype(np.float32)
    pool.upload()
    s = pool.cache.open()
    pool.cache.extend([s], [n + 3])
    plan = pool.cache.plan(1)
    plan.set([s], [n])
    kept = list(range(2, n))
    keys, values = pool.of(s, 0)
    plan.keep([kept])
    pool.download()
    pool.cache.truncate(s, 3 + len(kept))
    got_k, got_v = pool.of(s, 0)
    order = [0, 1, 2] + [3 + j for j in kept]
    assert np.array_equal(got_k, keys[order]) and np.array_equal(got_v, values[order])
    plan.dispose()


def test_refused_rows(context, device):
    pool = Pool(context, device, CacheLayout(1, 1, 32, 32, F16), 20)
    a, b = pool.cache.open(), pool.cache.open()
    pool.cache.extend([a, b], [10, 5])
    plan = pool.cache.plan(2)
    with pytest.raises(S.InvalidOperationException):
        plan.keep([[0]])
    plan.set_tree([a, b], [star(4), chain(2)])
    for bad in ([[0]], [[0], [0], [0]]):
        with pytest.raises(S.ArgumentException):
            plan.keep(bad)
    for bad in ([[4], []], [[-1], []], [[1, 1], []], [[2, 1], []], [[], [2]], [[0, 1, 2, 3, 3], []], [[0], [0, 1, 2]]):
        with pytest.raises(S.ArgumentOutOfRangeException):
            plan.keep(bad)
    for bad in ([[0], [-1]], [[-2], [-1]], [[-1, 1], [-1]], [[-1, 5], [-1]]):
        with pytest.raises(S.ArgumentOutOfRangeException):
            plan.set_tree([a, b], bad)
    with pytest.raises(S.ArgumentException):
        plan.set_tree([a], [star(4), chain(2)])
    with pytest.raises(S.ArgumentException):
        plan.set_tree([a, a], [star(4), star(4)])
    with pytest.raises(S.ArgumentOutOfRangeException):
        plan.set_tree([b], [star(6)])
    plan.keep([[0, 2], []])  # the batch that was set is still there
    rotation = Rotation(context, [1.0] * 17)
    x = device(np.zeros((6, 2, 32), np.float32))
    with pytest.raises(S.ArgumentOutOfRangeException):
        plan.append_rotated(0, x, 0, x, device(np.zeros((6, 32))), 0, device(np.zeros((6, 32))), 0, rotation)
    rotation.dispose()
    with pytest.raises(S.ObjectDisposedException):
        plan.append_rotated(0, x, 0, x, device(np.zeros((6, 32))), 0, device(np.zeros((6, 32))), 0, rotation)
    other = S.HipContext(0)
    rotation = Rotation(other, [1.0])
    with pytest.raises(S.ArgumentException):
        plan.append_rotated(0, x, 0, x, device(np.zeros((6, 32))), 0, device(np.zeros((6, 32))), 0, rotation)
    with pytest.raises(S.ArgumentException):
        other.dispose()
    rotation.dispose()
    other.dispose()
    c = pool.cache.fork(a)[0]
    plan.set_tree([a], [star(4)])  # in a page that another sequence holds
    with pytest.raises(S.InvalidOperationException):
        plan.keep([[0, 2]])
    pool.cache.free([c])
    plan.set_tree([a], [star(4)])
    context.capture_begin()
    with pytest.raises(S.InvalidOperationException):
        plan.keep([[0, 2]])
    context.capture_end().dispose()
    plan.keep([[0, 2]])
    plan.set_tree([], [])
    plan.keep([])
    context.synchronize()
    plan.dispose()


# ---- captured steps ----

@pytest.mark.parametrize("type_,heads,kv_heads,head_dim", [(F16, 12, 2, 128), (F32, 4, 4, 48), (F16, 8, 1, 256)])
def test_a_captured_step_follows_trees(context, device, type_, heads, kv_heads, head_dim):
    g = rng(99)
    pool = Pool(context, device, CacheLayout(1, kv_heads, head_dim, 32, type_), 200)
    lengths = [500, 70, 333, 31]
    sequences = forked(pool, 256, lengths)
    pool.write(g, sequences)
    rows = 80
    q = g.standard_normal((rows, heads, head_dim)).astype(np.float32)
    k, v = (g.standard_normal((rows, kv_heads, head_dim)).astype(np.float32) for _ in range(2))
    dq, dk, dv, turned, out = device(q), device(k), device(v), device(np.zeros_like(q)), device(np.zeros_like(q))
    rotation = Rotation(context, *rotary_frequencies(head_dim, 1e4), RotaryLayout.INTERLEAVED, 100)
    plan, eager = pool.cache.plan(heads), pool.cache.plan(heads)

    def step(p):
        p.append_rotated(0, dq, 0, turned, dk, 0, dv, 0, rotation)
        p.attention(0, turned, out)

    plan.set_tree(sequences, [mixed(31, 1), binary(15), star(20), roots(14)])
    context.capture_begin()
    step(plan)
    captured = context.capture_end()
    with pytest.raises(S.ArgumentException):
        rotation.dispose()
    batches = [[mixed(31, 1), binary(15), star(20), roots(14)], [star(5), chain(30), chain(1), star(31)],
               [chain(1), chain(1), chain(1), chain(1)], [binary(31), [], roots(2), star(3)], [chain(31), chain(2), [], []]]
    for trees in batches + batches[:1]:
        results = []
        for p, run in ((plan, captured.execute), (eager, lambda: step(eager))):
            p.set_tree(sequences, trees)
            context.upload(out, np.full(q.shape, 7, np.float32))
            context.upload(turned, np.full(q.shape, 5, np.float32))
            run()
            results.append([context.download(np.zeros_like(q), x) for x in (turned, out)] + [pool.download().host.copy()])
        n = sum(map(len, trees))
        for x, y in zip(results[0], results[1]):
            assert np.array_equal(x.view(np.uint8), y.view(np.uint8))
        assert np.all(results[0][1][n:] == 7) and np.all(results[0][0][n:] == 5)
        check_tree(pool, sequences, trees, heads, results[0][0], results[0][1])
    with pytest.raises(S.InvalidOperationException):
        plan.set_tree(sequences, [mixed(31, 1), binary(15), star(64), roots(14)])
    captured.dispose()
    rotation.dispose()
    plan.dispose()
    eager.dispose()


def test_a_captured_step_takes_a_tree_behind_any_context(context, device):
    # Where a tree's context ends within 32 positions changes what the plan keeps for it.
    g = rng(15)
    pool = Pool(context, device, CacheLayout(1, 1, 32, 32, F32), 30)
    s, other = pool.cache.open(), pool.cache.open()
    pool.cache.extend([s, other], [320 + 61, 40])
    pool.write(g, [s, other])
    q = g.standard_normal((65, 2, 32)).astype(np.float32)
    dq, out = device(q), device(np.zeros_like(q))
    plan = pool.cache.plan(2)
    plan.set_tree([s], [mixed(40, 1)])  # (leaves some room, not enough)
    plan.set_tree([s, other], [mixed(61, 1), star(4)])
    context.capture_begin()
    plan.attention(0, dq, out)
    step = context.capture_end()
    for more in (0, 1, 3, 26, 1, 1, 17):
        pool.cache.extend([s], [more])
        pool.write(g, [s, other])
        trees = [mixed(61, more), star(4)]
        plan.set_tree([s, other], trees)
        step.execute()
        check_tree(pool, [s, other], trees, 2, q, context.download(np.zeros_like(q), out))
    step.dispose()
    plan.dispose()


def test_a_step_captured_without_trees_takes_none(context, device):
    g = rng(4)
    pool = Pool(context, device, CacheLayout(1, 2, 64, 32, F16), 40)
    s = pool.cache.open()
    pool.cache.extend([s], [90])
    pool.write(g, [s])
    q = g.standard_normal((9, 4, 64)).astype(np.float32)
    dq, out = device(q), device(np.zeros_like(q))
    plan = pool.cache.plan(4)
    plan.set([s], [9])
    context.capture_begin()
    plan.attention(0, dq, out)
    captured = context.capture_end()
    with pytest.raises(S.InvalidOperationException):
        plan.set_tree([s], [star(9)])
    plan.set_tree([s], [chain(9)])  # no tree
    captured.execute()
    got = context.download(np.zeros_like(q), out)
    check_tree(pool, [s], [chain(9)], 4, q, got)
    captured.dispose()
    plan.set_tree([s], [star(9)])
    plan.attention(0, dq, out)
    check_tree(pool, [s], [star(9)], 4, q, context.download(np.zeros_like(q), out))
    plan.dispose()
