"""The paged key/value cache on the device: page copies, the batched cache write and the attention of a batch whose sequences
share pages, against the definition in 64 bits over the pool's own bytes. Whatever no row may see is NaN in every pool.

Attention's bound. A score is a sum of D products in FP32 (any order) times a factor: with e = 2^-24 it is off by at most
(D + 8) e A, A = sum |q k| / sqrt(D) (8: the factor's and the subtraction's roundings, the 2^-22 of a query kept in two
halves, exp2's argument). A relative error x of exp enters the weights and their sum once each. The sums over tokens run over
tiles of 32 (at most T / 32 tiles and the joining of four waves and of the parts) with up to 32 products a tile in one
instruction: (T / 32 + 64) e, and 16 e for probabilities in two halves, exp2 and the division (of F16 pages a probability is off
by up to 2^-36 of its row's largest where that is more: over T random values less than the 80 e below while T < 2^16). So
|o - exact| <= (2 (D + 8) e max A + 2 (T / 32 + 80) e) * sum p |v|, which the tests take times 1.01 (second order)."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

import satori_amd as S
from helpers import rng
from satori_amd.cache import CacheLayout, ElementType, PagedCache

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
NUMPY = {ElementType.F32: np.float32, ElementType.F16: np.float16}
F32, F16 = ElementType.F32, ElementType.F16


class Device:
    """Device copies of host arrays, freed at the end of a test."""

    def __init__(self, context):
        self.context, self.held = context, []

    def __call__(self, array):
        array = np.ascontiguousarray(array)
        p = self.context.alloc(max(array.nbytes, 16))
        self.held.append(p)
        if array.nbytes:
            self.context.upload(p, array)
        return p

    def close(self):
        self.context.synchronize()
        for p in self.held:
            self.context.free(p)


@pytest.fixture
def device(context):
    d = Device(context)
    yield d
    d.close()


class Pool:
    """A cache with a host copy of its pool; `written` positions hold numbers, everything else NaN."""

    def __init__(self, context, device, layout, pages):
        self.layout, self.context = layout, context
        self.width = next(w for w in (32, 64, 96, 128, 192, 256) if w >= layout.head_dim)
        self.host = np.full((pages, layout.layers, 2, layout.kv_heads, layout.page_tokens * self.width), np.nan,
                            NUMPY[layout.type])
        self.at = device(self.host)
        self.cache = PagedCache(context, layout, pages, self.at)

    def keys(self, layer):
        shape = (self.host.shape[0], self.layout.kv_heads, self.layout.page_tokens, self.width)
        return self.host[:, layer, 0].reshape(shape)

    def values(self, layer):
        shape = (self.host.shape[0], self.layout.kv_heads, self.width, self.layout.page_tokens)
        return self.host[:, layer, 1].reshape(shape)

    def write(self, g, sequences):
        """Random keys and values for every position of the sequences (shared ones the same)."""
        L, P, D = self.layout, self.layout.page_tokens, self.layout.head_dim
        places = {(page, p) for s in sequences for i, page in enumerate(self.cache.pages(s))
                  for p in range(min(P, self.cache.tokens(s) - i * P))}
        for layer in range(L.layers):
            for page, p in sorted(places):
                k = self.host[page, layer, 0].reshape(L.kv_heads, P, self.width)
                k[:, p] = 0
                k[:, p, :D] = g.standard_normal((L.kv_heads, D))
                self.host[page, layer, 1].reshape(L.kv_heads, self.width, P)[:, :D, p] = \
                    g.standard_normal((L.kv_heads, D))
        self.upload()

    def upload(self):
        self.context.upload(self.at, self.host)

    def download(self):
        self.context.download(self.host, self.at)
        return self

    def of(self, sequence, layer):
        """Keys and values [tokens][kv_heads][head_dim] of a sequence, in 64 bits."""
        table, n, D = self.cache.pages(sequence), self.cache.tokens(sequence), self.layout.head_dim
        k = self.keys(layer)[table][..., :D].transpose(0, 2, 1, 3).reshape(-1, self.layout.kv_heads, D)
        v = self.values(layer)[table][:, :, :D].transpose(0, 3, 1, 2).reshape(-1, self.layout.kv_heads, D)
        return k[:n].astype(np.float64), v[:n].astype(np.float64)


def exact_attention(q, k, v, position):
    """One row [heads][head_dim] over positions 0 .. position, and the bound of the module's docstring."""
    heads, D = q.shape
    group = heads // k.shape[1]
    k, v, q = k[:position + 1], v[:position + 1], q.astype(np.float64)
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    for h in range(heads):
        kh, vh = k[:, h // group], v[:, h // group]
        s = kh @ q[h] / np.sqrt(D)
        a = (np.abs(kh) @ np.abs(q[h]) / np.sqrt(D)).max()
        p = np.exp(s - s.max())
        p /= p.sum()
        out[h] = p @ vh
        bound[h] = 1.01 * (2 * (D + 8) * E * a + 2 * ((position + 1) / 32 + 80) * E) * (p @ np.abs(vh))
    return out, bound


def check_attention(pool, sequences, new, heads, q, got, layer=0, label=""):
    row = 0
    for s, n in zip(sequences, new):
        k, v = pool.of(s, layer)
        for position in range(len(k) - n, len(k)):
            expected, bound = exact_attention(q[row], k, v, position)
            err = np.abs(got[row].astype(np.float64) - expected)
            assert np.all(err <= bound), (f"{label} sequence {s} position {position}: {err.max()} over "
                                          f"{bound.flat[err.argmax()]}")
            row += 1


def attend(context, device, pool, sequences, new, heads, g, layer=0, scale=1.0, stream=0):
    rows = int(sum(new))
    q = (g.standard_normal((rows, heads, pool.layout.head_dim)) * scale).astype(np.float32)
    plan = pool.cache.plan(heads)
    try:
        plan.set(sequences, new)
        out = device(np.full(q.shape, 7, np.float32))
        plan.attention(layer, device(q), out)
        return q, context.download(np.zeros(q.shape, np.float32), out)
    finally:
        context.synchronize()
        plan.dispose()


def forked(pool, prefix, own):
    """Sequences forked from one of `prefix` tokens, own[i] tokens longer."""
    first = pool.cache.open()
    pool.cache.extend([first], [prefix])
    sequences = [first] + pool.cache.fork(first, len(own) - 1)
    pool.cache.extend(sequences, own)
    return sequences


SHAPES = [  # type, heads, kv_heads, head_dim, page_tokens
    (F16, 12, 2, 128, 32), (F32, 12, 2, 128, 32), (F16, 7, 1, 80, 64), (F32, 7, 1, 80, 64), (F16, 4, 4, 64, 32),
    (F32, 4, 4, 48, 128), (F16, 2, 2, 32, 256), (F32, 6, 3, 32, 32), (F16, 6, 2, 96, 32), (F32, 6, 2, 96, 64),
    (F16, 8, 2, 192, 32), (F32, 8, 2, 192, 32), (F16, 8, 1, 256, 32), (F32, 20, 1, 256, 64), (F16, 34, 1, 129, 32),
    (F16, 3, 3, 1, 32), (F32, 3, 1, 2, 32),
]


@pytest.mark.parametrize("type_,heads,kv_heads,head_dim,page_tokens", SHAPES)
def test_lengths_without_anything_in_common(context, device, type_, heads, kv_heads, head_dim, page_tokens):
    g = rng(head_dim * heads)
    pool = Pool(context, device, CacheLayout(2, kv_heads, head_dim, page_tokens, type_), 100)
    own = [1, 2, 31, 32, 33, 63, 127, 128, 129, 300]
    sequences = [pool.cache.open() for _ in own]
    pool.cache.extend(sequences, own)
    pool.write(g, sequences)
    q, got = attend(context, device, pool, sequences, [1] * len(own), heads, g, layer=1)
    check_attention(pool, sequences, [1] * len(own), heads, q, got, layer=1)


@pytest.mark.parametrize("type_,heads,kv_heads,head_dim,page_tokens", SHAPES)
@pytest.mark.parametrize("prefix", [200, 777])
def test_a_common_prefix(context, device, type_, heads, kv_heads, head_dim, page_tokens, prefix):
    g = rng(prefix + head_dim)
    pool = Pool(context, device, CacheLayout(1, kv_heads, head_dim, page_tokens, type_), 128)
    own = [1, 5, 40, 64, 1, 130, 2, 33, 9]
    sequences = forked(pool, prefix, own)
    pool.write(g, sequences)
    q, got = attend(context, device, pool, sequences, [1] * len(own), heads, g)
    check_attention(pool, sequences, [1] * len(own), heads, q, got)


@pytest.mark.parametrize("type_,heads,kv_heads,head_dim,page_tokens", SHAPES)
def test_several_new_positions_see_only_their_past(context, device, type_, heads, kv_heads, head_dim, page_tokens):
    # Chunks of a prompt and drafts: causal tiles, rows that end inside a tile, a whole sequence that is new.
    g = rng(7 * head_dim)
    pool = Pool(context, device, CacheLayout(1, kv_heads, head_dim, page_tokens, type_), 128)
    own, new = [70, 3, 40, 1, 150], [70, 3, 17, 1, 33]
    sequences = forked(pool, 161, own)
    whole = pool.cache.open()
    pool.cache.extend([whole], [45])
    sequences, new = sequences + [whole], new + [45]
    pool.write(g, sequences)
    q, got = attend(context, device, pool, sequences, new, heads, g)
    check_attention(pool, sequences, new, heads, q, got)


@pytest.mark.parametrize("type_", [F16, F32])
def test_a_tree_of_prefixes(context, device, type_):
    # Forks of forks: three prefixes of different depth, a short one that is not worth sharing, rows of none.
    g = rng(99)
    pool = Pool(context, device, CacheLayout(1, 2, 64, 32, type_), 200)
    c = pool.cache
    root = c.open()
    c.extend([root], [333])
    left, right = c.fork(root, 2)
    c.extend([left, right], [200, 40])
    leaves = [root] + [left] + c.fork(left, 3) + [right] + c.fork(right, 2)
    deeper = c.fork(leaves[2], 2)
    c.extend(leaves[2:3] + deeper, [150, 1, 500])
    everyone = leaves + deeper
    c.extend(everyone, [1 + i % 4 for i in range(len(everyone))])
    alone = c.open()
    c.extend([alone], [10])
    batch = [deeper[1], root, alone] + leaves[1:] + [deeper[0]]
    new = [1, 0, 3] + [1] * (len(batch) - 3)
    pool.write(g, batch)
    q, got = attend(context, device, pool, batch, new, 6, g)
    check_attention(pool, batch, new, 6, q, got)


@pytest.mark.parametrize("type_,sequences,heads,kv_heads,head_dim,prefix", [
    (F16, 64, 16, 4, 128, 5000), (F32, 33, 12, 2, 128, 3000), (F16, 1, 8, 1, 64, 20011), (F32, 1, 4, 4, 64, 9001),
    (F16, 130, 1, 1, 32, 1000)])
def test_long_prefixes_and_large_batches(context, device, type_, sequences, heads, kv_heads, head_dim, prefix):
    g = rng(prefix)
    pool = Pool(context, device, CacheLayout(1, kv_heads, head_dim, 32, type_), prefix // 32 + 8 * sequences)
    own = [1 + int(n) for n in g.integers(0, 150, sequences)]
    batch = forked(pool, prefix, own)
    L = pool.layout  # everything written, then what is behind the sequences' ends spoiled
    pool.host[...] = g.standard_normal(pool.host.shape, np.float32).astype(pool.host.dtype)
    for s in batch:
        last, n = pool.cache.pages(s)[-1], pool.cache.tokens(s) % 32
        if n:
            pool.keys(0)[last, :, n:] = np.nan
            pool.host[last, 0, 1].reshape(L.kv_heads, pool.width, 32)[..., n:] = np.inf
    pool.upload()
    q, got = attend(context, device, pool, batch, [1] * sequences, heads, g)
    some = sorted({0, sequences // 2, sequences - 1})
    check_attention(pool, [batch[i] for i in some], [1] * len(some), heads, q[some], got[some])
    for i in range(sequences):  # and every row, by a common bound on the whole
        k, v = pool.of(batch[i], 0)
        s = np.einsum("thd,hgd->hgt", k, q[i].reshape(kv_heads, -1, head_dim).astype(np.float64)) / np.sqrt(head_dim)
        p = np.exp(s - s.max(-1, keepdims=True))
        expected = np.einsum("hgt,thd->hgd", p / p.sum(-1, keepdims=True), v).reshape(heads, head_dim)
        assert np.abs(got[i] - expected).max() <= 2e-5, f"row {i}"


@pytest.mark.parametrize("type_", [F16, F32])
def test_large_and_tiny_queries_and_scores(context, device, type_):
    # Scores of hundreds (one token takes all), of nothing (all alike), and queries far outside a half's range.
    g = rng(5)
    pool = Pool(context, device, CacheLayout(1, 1, 64, 32, type_), 40)
    own = [1, 33, 64, 95, 128, 200]
    sequences = forked(pool, 130, own)
    pool.write(g, sequences)
    for scale in (30.0, 1e-6, 1e-30, 0.0):
        q, got = attend(context, device, pool, sequences, [1] * len(own), 4, g, scale=scale)
        check_attention(pool, sequences, [1] * len(own), 4, q, got, label=str(scale))
    pool.host[...] = pool.host * NUMPY[type_](2.0 ** -14)
    pool.upload()
    q, got = attend(context, device, pool, sequences, [1] * len(own), 4, g, scale=2.0 ** 18)
    check_attention(pool, sequences, [1] * len(own), 4, q, got, label="small keys")


@pytest.mark.parametrize("type_", [F16, F32])
@pytest.mark.parametrize("new", [2, 40])
def test_a_value_that_is_not_finite_reaches_only_rows_that_see_it(context, device, type_, new):
    g = rng(new)
    pool = Pool(context, device, CacheLayout(1, 2, 64, 32, type_), 20)
    s = pool.cache.open()
    pool.cache.extend([s], [100])
    pool.write(g, [s])
    spoiled = 100 - new // 2
    page, at = pool.cache.pages(s)[spoiled // 32], spoiled % 32
    for what in ("value", "key"):
        kept = pool.host.copy()
        if what == "value":
            pool.host[page, 0, 1].reshape(2, 64, 32)[0, 5, at] = np.inf
            pool.host[page, 0, 1].reshape(2, 64, 32)[1, 9, at] = np.nan
        else:
            pool.host[page, 0, 0].reshape(2, 32, 64)[:, at, 3] = np.nan
        pool.upload()
        q, got = attend(context, device, pool, [s], [new], 4, g)
        for row, position in enumerate(range(100 - new, 100)):
            finite = np.isfinite(got[row])
            if position < spoiled:
                k, v = pool.of(s, 0)
                expected, bound = exact_attention(q[row], k, v, position)
                assert finite.all() and np.all(np.abs(got[row] - expected) <= bound), f"{what} row {row}"
            elif what == "value":
                assert not finite[:2, 5].any() and not finite[2:, 9].any(), f"row {row} sees it"
                assert finite.sum() == finite.size - 4, "other lanes do not"
            else:
                assert not finite.any()
        pool.host[...] = kept


def test_a_row_whose_query_is_not_finite_spoils_no_other(context, device):
    g = rng(3)
    pool = Pool(context, device, CacheLayout(1, 1, 128, 32, F16), 40)
    sequences = forked(pool, 160, [1, 40, 70])
    pool.write(g, sequences)
    q = g.standard_normal((3, 3, 128)).astype(np.float32)
    q[1, 2, 7], q[0, 0, 0] = np.nan, np.inf
    plan = pool.cache.plan(3)
    plan.set(sequences, [1, 1, 1])
    out = device(np.zeros_like(q))
    plan.attention(0, device(q), out)
    got = context.download(np.zeros_like(q), out)
    plan.dispose()
    for row, s in enumerate(sequences):
        k, v = pool.of(s, 0)
        expected, bound = exact_attention(np.where(np.isfinite(q[row]), q[row], 0), k, v, len(k) - 1)
        for h in range(3):
            if np.isfinite(q[row, h]).all():
                assert np.all(np.abs(got[row, h] - expected[h]) <= bound[h])
            else:
                assert not np.isfinite(got[row, h]).any()


# ---- the cache write ----

@pytest.mark.parametrize("type_,heads,kv_heads,head_dim,rotary,page_tokens", [
    (F32, 12, 2, 128, 128, 32), (F16, 12, 2, 128, 128, 32), (F16, 7, 1, 80, 64, 64), (F32, 4, 4, 48, 48, 32),
    (F16, 3, 3, 33, 2, 32), (F32, 2, 1, 256, 200, 128)])
@pytest.mark.parametrize("table", [False, True])
def test_append_equals_the_single_sequence_operator(context, device, type_, heads, kv_heads, head_dim, rotary, page_tokens,
                                                    table):
    g = rng(head_dim + rotary)
    pool = Pool(context, device, CacheLayout(2, kv_heads, head_dim, page_tokens, type_), 60)
    own, new = [1, 70, 33, 5], [1, 70, 2, 0]
    sequences = forked(pool, 301, own)
    rows, base = sum(new), 1e6
    q = g.standard_normal((rows, heads * head_dim)).astype(np.float32)
    k, v = (g.standard_normal((rows, kv_heads * head_dim)).astype(np.float32) for _ in range(2))
    bq, bk, bv = (g.standard_normal(n * head_dim).astype(np.float32) for n in (heads, kv_heads, kv_heads))
    dq, dk, dv, dbq, dbk = device(q), device(k), device(v), device(bq), device(bk)
    out = device(np.zeros_like(q))
    angles, positions = 0, 320  # fewer than the longest sequence has
    ops = S.DeviceOps(context)
    if table:
        angles = device(np.zeros(positions * rotary))
        ops.rope_table(positions, rotary, base, angles)
    plan = pool.cache.plan(heads)
    plan.set(sequences, new)
    plan.append(1, dq, dbq, out, dk, dbk, dv, 0, base, rotary, angles, positions if table else 0)
    got_q = context.download(np.zeros_like(q), out)
    before = pool.host.copy()
    pool.download()
    after, row, kw = before.copy(), 0, kv_heads * head_dim
    ek, ev = device(np.zeros(kw, np.float32)), device(np.zeros(kw, np.float32))
    for s, n in zip(sequences, new):
        tokens, pages = pool.cache.tokens(s), pool.cache.pages(s)
        for p in range(tokens - n, tokens):
            one = device(q[row])
            ops.attention_inputs(one, dbq, dk + 4 * row * kw, dbk, ek, dv + 4 * row * kw, 0, ev, heads, kv_heads,
                                 head_dim, p, base, rotary)
            assert np.array_equal(context.download(np.zeros_like(q[row]), one), got_q[row]), f"query of row {row}"
            key = context.download(np.zeros(kw, np.float32), ek).reshape(kv_heads, head_dim)
            value = context.download(np.zeros(kw, np.float32), ev).reshape(kv_heads, head_dim)
            page, at = pages[p // page_tokens], p % page_tokens
            after[page, 1, 0].reshape(kv_heads, page_tokens, pool.width)[:, at] = 0
            after[page, 1, 0].reshape(kv_heads, page_tokens, pool.width)[:, at, :head_dim] = key.astype(NUMPY[type_])
            after[page, 1, 1].reshape(kv_heads, pool.width, page_tokens)[:, :head_dim, at] = value.astype(NUMPY[type_])
            row += 1
    assert np.array_equal(pool.host, after, equal_nan=True), "the rows' places, and nothing else"
    assert np.array_equal(context.download(np.zeros_like(q), dq), q), "the query is left as it was"
    plan.append(1, dq, dbq, dq, dk, dbk, dv, 0, base, rotary, angles, positions if table else 0)
    assert np.array_equal(context.download(np.zeros_like(q), dq), got_q), "in place"
    plan.dispose()


# ---- page copies ----

def copy_pages(cache, sources, destinations):
    cache.copy_pages(sources, destinations)


@pytest.mark.parametrize("layers,pages", [(1, 3), (5, 700)])
def test_page_copies(context, device, layers, pages):
    layout = CacheLayout(layers, 1, 32, 32, F16)
    pool = Pool(context, device, layout, pages)
    pool.host.view(np.uint16)[...] = rng(pages).integers(0, 2 ** 16, pool.host.shape)
    pool.upload()
    g = rng(1)
    order = g.permutation(pages)
    destinations = order[:pages // 2]
    sources = g.choice(order[pages // 2:], destinations.size)  # one page can go to several places
    copy_pages(pool.cache, sources, destinations)
    expected = pool.host.view(np.uint16).copy()
    expected[destinations] = expected[sources]
    assert np.array_equal(pool.download().host.view(np.uint16), expected)


def test_forks_copies_and_compaction_keep_what_sequences_hold(context, device):
    g = rng(11)
    pool = Pool(context, device, CacheLayout(3, 2, 64, 32, F32), 64)
    c = pool.cache
    a, b = c.open(), c.open()
    c.extend([a, b], [75, 200])
    pool.write(g, [a, b])
    kept = {s: [np.stack(pool.of(s, layer)) for layer in range(3)] for s in (a, b)}
    forks = c.fork(a, 4)
    c.extend(forks + [a], [1, 0, 3, 40, 2])
    twin = c.copy(b)
    c.free([b, forks[1]])
    c.compact()
    pool.download()
    assert c.free_pages == 64 - len({p for s in (a, twin, *forks[:1], *forks[2:]) for p in c.pages(s)})
    for s, of in [(a, a), (forks[0], a), (forks[2], a), (forks[3], a), (twin, b)]:
        for layer in range(3):
            n = len(kept[of][layer][0])
            assert np.array_equal(np.stack(pool.of(s, layer))[:, :n], kept[of][layer]), f"sequence {s} layer {layer}"


# ---- plans in use ----

def test_a_captured_step_follows_its_plan(context, device):
    # Captured once, replayed per token with the plan set to the sequences as they have grown (more pages, more chunks,
    # another division of the batch), each replay against an eager call on a plan of its own, with eager work between.
    g = rng(21)
    heads, kv, D = 6, 2, 64
    pool = Pool(context, device, CacheLayout(1, kv, D, 32, F16), 400)
    c = pool.cache
    sequences = forked(pool, 150, [1, 20, 31, 1])
    pool.write(g, sequences)
    rows = len(sequences)
    q = device(np.zeros((rows, heads * D), np.float32))
    k, v = (device(np.zeros((rows, kv * D), np.float32)) for _ in range(2))
    turned, out, eager_out = (device(np.zeros((rows, heads * D), np.float32)) for _ in range(3))
    largest = c.plan(heads)
    plan, other = c.plan(heads), c.plan(heads)
    ones = [1] * rows
    plan.set(sequences, ones)
    context.capture_begin()
    plan.append(0, q, 0, turned, k, 0, v, 0, 1e4, D)
    plan.attention(0, turned, out)
    step = context.capture_end()
    with pytest.raises(S.ArgumentException):
        plan.dispose()
    for growth in (1, 1, 17, 200, 1, 900, 1):
        # Everything up to the new position is written by eager appends, the new one by the replay.
        for s in sequences:
            if growth > 1:
                c.extend([s], [growth - 1])
                many = growth - 1
                other.set([s], [many])
                other.append(0, device(g.standard_normal((many, heads * D)).astype(np.float32)), 0,
                             device(np.zeros((many, heads * D), np.float32)),
                             device(g.standard_normal((many, kv * D)).astype(np.float32)), 0,
                             device(g.standard_normal((many, kv * D)).astype(np.float32)), 0, 1e4, D)
        c.extend(sequences, ones)
        plan.set(sequences, ones)
        for p, width in ((q, heads), (k, kv), (v, kv)):
            context.upload(p, g.standard_normal((rows, width * D)).astype(np.float32))
        step.execute()
        got = context.download(np.zeros((rows, heads, D), np.float32), out)
        other.set(sequences, ones)
        other.attention(0, turned, eager_out)
        eager = context.download(np.zeros((rows, heads, D), np.float32), eager_out)
        assert np.array_equal(got, eager), f"after {growth}"
        pool.download()
        check_attention(pool, sequences, ones, heads, context.download(np.zeros((rows, heads, D), np.float32), turned),
                        got, label=f"after {growth}")
    step.dispose()
    for p in (plan, other, largest):
        p.dispose()


def test_two_plans_on_two_streams(context, device):
    g = rng(31)
    pool = Pool(context, device, CacheLayout(1, 2, 128, 32, F16), 300)
    first, second = forked(pool, 900, [1, 30, 9]), forked(pool, 2000, [5, 1])
    pool.write(g, first + second)
    with S.HipContext(0) as elsewhere:
        plans, results = [], []
        for batch, stream in ((first, 0), (second, elsewhere.stream)):
            q = g.standard_normal((len(batch), 8, 128)).astype(np.float32)
            plan, dq, out = pool.cache.plan(8), device(q), device(np.zeros_like(q))
            plan.set(batch, [1] * len(batch), stream)
            plans.append(plan)
            results.append((batch, q, dq, out, stream))
        for _ in range(20):
            for plan, (_, _, dq, out, stream) in zip(plans, results):
                plan.attention(0, dq, out, stream)
        elsewhere.synchronize()
        context.synchronize()
        for plan, (batch, q, _, out, _) in zip(plans, results):
            check_attention(pool, batch, [1] * len(batch), 8, q, context.download(np.zeros_like(q), out))
            plan.dispose()


def test_the_same_call_twice_gives_the_same_bits(context, device):
    g = rng(41)
    pool = Pool(context, device, CacheLayout(1, 2, 128, 32, F16), 200)
    batch = forked(pool, 1500, [1, 30, 9, 200])
    pool.write(g, batch)
    q = device(g.standard_normal((4, 12, 128)).astype(np.float32))
    plan, outs = pool.cache.plan(12), []
    plan.set(batch, [1] * 4)
    for _ in range(5):
        out = device(np.zeros((4, 12, 128), np.float32))
        plan.attention(0, q, out)
        outs.append(context.download(np.zeros((4, 12, 128), np.float32), out))
    assert all(np.array_equal(o, outs[0]) for o in outs)
    plan.dispose()


def test_refusals(context, device):
    layout = CacheLayout(2, 2, 64, 32, F16)
    pool = Pool(context, device, layout, 8)
    c = pool.cache
    s = c.open()
    c.extend([s], [40])
    q, kv = device(np.zeros((1, 4 * 64), np.float32)), device(np.zeros((1, 2 * 64), np.float32))
    out = device(np.zeros((1, 4 * 64), np.float32))
    plan = c.plan(4)
    with pytest.raises(S.InvalidOperationException):
        plan.attention(0, q, out)
    with pytest.raises(S.InvalidOperationException):
        plan.append(0, q, 0, out, kv, 0, kv, 0, 1e4, 64)
    for arguments in (([s, s], [1, 1]), ([5], [1]), ([-1], [1]), ([s], [1, 2])):
        with pytest.raises(S.ArgumentException):
            plan.set(*arguments)
    for fresh in (41, -1):
        with pytest.raises(S.ArgumentOutOfRangeException):
            plan.set([s], [fresh])
    plan.set([], [])
    plan.attention(0, q, out)
    plan.append(0, q, 0, out, kv, 0, kv, 0, 1e4, 64)
    plan.set([s], [0])
    plan.attention(0, q, out)
    plan.set([s], [1])
    for layer in (-1, 2):
        with pytest.raises(S.ArgumentOutOfRangeException):
            plan.attention(layer, q, out)
    for arguments in ((0, out), (q, 0)):
        with pytest.raises(S.ArgumentNullException):
            plan.attention(0, *arguments)
    for a, b in ((q, q), (q, pool.at), (q, q + 64)):
        with pytest.raises(S.ArgumentException):
            plan.attention(0, a, b)
    for rotary, base in ((0, 1e4), (65, 1e4), (66, 1e4), (3, 1e4), (64, 0.0), (64, float("nan"))):
        with pytest.raises(S.ArgumentOutOfRangeException):
            plan.append(0, q, 0, out, kv, 0, kv, 0, base, rotary)
    with pytest.raises(S.ArgumentException):
        plan.append(0, q, 0, q + 16, kv, 0, kv, 0, 1e4, 64)
    with pytest.raises(S.ArgumentException):
        plan.append(0, q, 0, out, pool.at + 64, 0, kv, 0, 1e4, 64)
    other = c.fork(s)[0]
    plan.set([s, other], [1, 0])
    with pytest.raises(S.InvalidOperationException):  # the page is another sequence's too
        plan.append(0, q, 0, out, kv, 0, kv, 0, 1e4, 64)
    stranger = PagedCache(context, layout, 9, pool.at)
    lent = c.plan(4)
    lent.cache = stranger
    with pytest.raises(S.ArgumentException):
        lent.set([], [])
    lent.dispose()
    context.capture_begin()
    with pytest.raises(S.InvalidOperationException):
        plan.set([s], [1])
    with pytest.raises(S.InvalidOperationException):
        c.plan(4)
    context.capture_end().dispose()
    for moves in (([0], [0]), ([0, 1], [2, 2]), ([0, 1], [1, 2])):
        with pytest.raises(S.ArgumentException):
            copy_pages(c, *moves)
    for moves in (([8], [0]), ([0], [8]), ([-1], [0])):
        with pytest.raises(S.ArgumentOutOfRangeException):
            copy_pages(c, *moves)
    with pytest.raises(S.ArgumentException):
        PagedCache(context, layout, 8, pool.at + 4).plan(4)
    for heads in (3, 0, -2):
        with pytest.raises(S.ArgumentException):
            c.plan(heads)
    plan.dispose()
    plan.dispose()
    with pytest.raises(S.ObjectDisposedException):
        plan.set([s], [1])
    own = S.HipContext(0)
    cache = PagedCache(own, layout, 4)
    held = cache.plan(4)
    with pytest.raises(S.ArgumentException):
        own.dispose()
    held.dispose()
    cache.dispose()
    own.dispose()


def test_a_step_keeps_its_plans_memory(context, device):
    pool = Pool(context, device, CacheLayout(1, 1, 32, 32, F16), 4000)
    c = pool.cache
    s = c.open()
    c.extend([s], [32])
    plan = c.plan(1)
    plan.set([s], [1])
    q, out = device(np.zeros((1, 32), np.float32)), device(np.zeros((1, 32), np.float32))
    context.capture_begin()
    plan.attention(0, q, out)
    step = context.capture_end()
    others = [c.open() for _ in range(3000)]
    c.extend(others, [1] * 3000)
    with pytest.raises(S.InvalidOperationException):
        plan.set(others, [1] * 3000)
    step.dispose()
    plan.set(others, [1] * 3000)
    plan.dispose()


def test_a_batch_whose_memory_cannot_be_had_leaves_no_plan(context, device):
    # The partial results of 500,000 rows of 512 heads take 264 GB and half as much again; only page 0 is behind the pool, and
    # nothing is launched on others.
    layout = CacheLayout(1, 512, 256, 256, F16)
    first = PagedCache(context, layout, 1)
    cache = PagedCache(context, layout, 2100, first.pool)
    small, large = cache.open(), cache.open()
    cache.extend([small], [1])
    cache.extend([large], [500000])
    plan = cache.plan(512)
    q, out = device(np.ones((1, 512 * 256), np.float32)), device(np.zeros((1, 512 * 256), np.float32))
    plan.set([small], [1])
    with pytest.raises(S.OutOfMemoryException):
        plan.set([large], [500000])
    for call in (lambda: plan.attention(0, q, out), lambda: plan.append(0, q, 0, out, q, 0, q, 0, 1e4, 256)):
        with pytest.raises(S.InvalidOperationException):
            call()
    plan.set([small], [1])  # the plan can be set again
    plan.dispose()
    cache.dispose()
    first.dispose()


@pytest.mark.parametrize("type_,heads,kv,D", [(F32, 16, 1, 128), (F16, 12, 2, 192), (F32, 3, 1, 200)])
def test_the_largest_tiles_captured_first(type_, heads, kv, D):
    # Kernels that take more than 64 KB of LDS, launched by a capture before any eager call of theirs (a context of its own;
    # the process may have run them before), then replayed as the sequences grow, against eager calls on another plan.
    g = rng(77)
    context = S.HipContext(0)
    device = Device(context)
    pool = Pool(context, device, CacheLayout(1, kv, D, 64, type_), 40)
    c = pool.cache
    first = c.open()
    c.extend([first], [300])
    sequences = [first] + c.fork(first, 2)
    c.extend(sequences, [9, 1, 3])
    pool.write(g, sequences)
    new = [9, 1, 3]
    q, out, eager_out = (device(g.standard_normal((13, heads, D)).astype(np.float32)) for _ in range(3))
    plan, other = c.plan(heads), c.plan(heads)
    plan.set(sequences, new)
    context.capture_begin()
    plan.attention(0, q, out)
    step = context.capture_end()
    for turn in range(3):
        step.execute()
        got = context.download(np.zeros((13, heads, D), np.float32), out)
        other.set(sequences, new)
        other.attention(0, q, eager_out)
        assert np.array_equal(got, context.download(np.zeros((13, heads, D), np.float32), eager_out)), turn
        check_attention(pool, sequences, new, heads, context.download(np.zeros((13, heads, D), np.float32), q), got)
        c.extend(sequences, [40, 70, 5])
        pool.download().write(g, sequences)
        plan.set(sequences, new)
    step.dispose()
    plan.dispose()
    other.dispose()
    device.close()
    context.dispose()


def test_another_librarys_capture(context, device):
    # The plan cannot know when such a graph ends: its memory stays where it is from then on. While the capture lasts (in the
    # global mode, which forbids allocations), another plan grows and runs on the context stream.
    hip = ctypes.CDLL("libamdhip64.so")
    P = ctypes.c_void_p
    hip.hipStreamCreateWithFlags.argtypes = [ctypes.POINTER(P), ctypes.c_uint]
    hip.hipStreamBeginCapture.argtypes = [P, ctypes.c_int]
    hip.hipStreamEndCapture.argtypes = [P, ctypes.POINTER(P)]
    hip.hipGraphInstantiate.argtypes = [ctypes.POINTER(P), P, P, P, ctypes.c_size_t]
    hip.hipGraphLaunch.argtypes = [P, P]
    hip.hipStreamSynchronize.argtypes = hip.hipStreamDestroy.argtypes = [P]
    hip.hipGraphExecDestroy.argtypes = hip.hipGraphDestroy.argtypes = [P]
    g = rng(78)
    pool = Pool(context, device, CacheLayout(1, 1, 32, 32, F16), 4000)
    c = pool.cache
    s = c.open()
    c.extend([s], [50])
    others = [c.open() for _ in range(3000)]
    c.extend(others, [1] * 3000)
    pool.write(g, [s] + others)
    plan, other = c.plan(4), c.plan(4)
    plan.set([s], [1])
    q, out = device(g.standard_normal((1, 4, 32)).astype(np.float32)), device(np.zeros((1, 4, 32), np.float32))
    many = g.standard_normal((3000, 4, 32)).astype(np.float32)
    q_many, out_many = device(many), device(np.zeros_like(many))
    foreign, graph, exe = P(), P(), P()
    context.synchronize()
    assert hip.hipStreamCreateWithFlags(ctypes.byref(foreign), 1) == 0
    try:
        assert hip.hipStreamBeginCapture(foreign, 0) == 0  # global
        try:
            plan.attention(0, q, out, foreign.value)
            other.set(others, [1] * 3000)
            other.attention(0, q_many, out_many)
        finally:
            ended = hip.hipStreamEndCapture(foreign, ctypes.byref(graph))
        assert ended == 0
        check_attention(pool, others, [1] * 3000, 4, many, context.download(np.zeros_like(many), out_many))
        assert hip.hipGraphInstantiate(ctypes.byref(exe), graph, None, None, 0) == 0
        with pytest.raises(S.InvalidOperationException):
            plan.set(others, [1] * 3000)
        for replay in range(3):
            context.upload(out, np.zeros((1, 4, 32), np.float32))
            context.synchronize()
            assert hip.hipGraphLaunch(exe, foreign) == 0
            assert hip.hipStreamSynchronize(foreign) == 0
            got = context.download(np.zeros((1, 4, 32), np.float32), out)
            check_attention(pool, [s], [1], 4, context.download(np.zeros((1, 4, 32), np.float32), q), got, label=f"{replay}")
            c.extend([s], [60])
            pool.write(g, [s])
            plan.set([s], [1])
        hip.hipGraphExecDestroy(exe)
        hip.hipGraphDestroy(graph)
    finally:
        hip.hipStreamDestroy(foreign)
    plan.dispose()
    other.dispose()


def test_a_captured_write_keeps_to_pages_of_its_own(context, device):
    pool = Pool(context, device, CacheLayout(1, 1, 32, 32, F16), 8)
    c = pool.cache
    s = c.open()
    c.extend([s], [40])
    plan = c.plan(1)
    plan.set([s], [1])
    q, out = device(np.zeros((1, 32), np.float32)), device(np.zeros((1, 32), np.float32))
    context.capture_begin()
    plan.append(0, q, 0, out, q, 0, q, 0, 1e4, 32)
    step = context.capture_end()
    other = c.fork(s)[0]
    with pytest.raises(S.InvalidOperationException):  # the replay would write the page that both hold
        plan.set([s, other], [1, 0])
    c.extend([s], [1])
    plan.set([s, other], [1, 0])
    step.dispose()
    context.capture_begin()
    plan.attention(0, q, out)
    step = context.capture_end()
    plan.set([other], [1])
    c.free([s])
    s = c.fork(other)[0]
    plan.set([s], [1])  # nothing is written
    step.dispose()
    plan.dispose()


def test_sizes_that_overflow(context, device):
    for heads, kv, D in ((1 << 20, 1, 8), (1 << 20, 1 << 20, 8)):
        with pytest.raises(S.OverflowException):
            PagedCache(context, CacheLayout(1, 1, D, 32, F16), 4, 16).plan(heads) if kv == 1 else \
                CacheLayout(1, kv, D, 32, F16).page_bytes
    lib = S._ffi.lib()
    a = np.zeros(1, np.int32)
    from satori_amd import _check
    for page_bytes, pages in ((1 << 37, 1), (1 << 36, 1 << 30), (24, 4), (0, 4)):
        with pytest.raises((S.OverflowException, S.ArgumentOutOfRangeException)):
            _check(lib.satori_hip_cache_copy_pages(context.handle, 16, page_bytes, pages, a.ctypes.data, a.ctypes.data, 1, None))


@pytest.mark.parametrize("type_", [F16, F32])
@pytest.mark.parametrize("new", [1, 40])
def test_small_weights_beside_one_that_takes_all(context, device, type_, new):
    # One key has all the weight and a value of zero; the others' weights are 2^-22 of its, and make the output. Its score is
    # one product of 1 and 122 (exact) over 8, off by less than 8 e 15.25 of the factor's and the subtraction's roundings; the
    # others' as in the module's bound. Of F16 pages a weight in two halves is off by half a step of the smallest half, 2^-25,
    # where the largest is at least 2^11: 2^-36 of it.
    g = rng(41)
    heads, D, tokens = 4, 64, 80
    pool = Pool(context, device, CacheLayout(1, 1, D, 32, type_), 4)
    s = pool.cache.open()
    pool.cache.extend([s], [tokens])
    pool.write(g, [s])
    first = pool.cache.pages(s)[0]
    pool.keys(0)[..., 0] = 0
    pool.keys(0)[first, 0, 0] = 0
    pool.keys(0)[first, 0, 0, 0] = 122
    pool.values(0)[first, 0, :, 0] = 0
    pool.upload()
    q = (g.standard_normal((new, heads, D)) / 4).astype(np.float32)
    q[..., 0] = 1
    plan = pool.cache.plan(heads)
    plan.set([s], [new])
    out = device(np.zeros_like(q))
    plan.attention(0, device(q), out)
    got = context.download(np.zeros_like(q), out)
    k, v = pool.of(s, 0)
    for row in range(new):
        n = tokens - new + row + 1
        for h in range(heads):
            scores = k[:n, 0] @ q[row, h].astype(np.float64) / 8
            p = np.exp(scores - scores.max())
            p /= p.sum()
            a = (np.abs(k[1:n, 0]) @ np.abs(q[row, h].astype(np.float64))).max() / 8
            bound = 1.01 * E * (2 * (8 * 15.25 + (D + 8) * a) + 2 * (n / 32 + 80)) * (p @ np.abs(v[:n, 0]))
            if type_ == F16:
                bound = bound + 1.01 * 2.0 ** -36 * np.abs(v[:n, 0]).sum(0)
            err = np.abs(got[row, h] - p @ v[:n, 0])
            assert np.all(err <= bound), (row, h, (err / bound).max())
    plan.dispose()


@pytest.mark.parametrize("type_,heads,kv_heads,head_dim,page_tokens", SHAPES)
def test_many_rows_over_many_positions(context, device, type_, heads, kv_heads, head_dim, page_tokens):
    # Enough positions that blocks of 16 (row, head) pairs would read 128 MiB and more: tiles then pass through LDS. Some rows
    # against the definition; then a value that is infinite and a key that is NaN, each inside a tile that some rows see and
    # some do not, change what sees them and no bit of anything else.
    g = rng(heads + head_dim)
    own = [300, 20, 61]
    pool = Pool(context, device, CacheLayout(1, kv_heads, head_dim, page_tokens, type_), 1)
    blocks = (sum(own) * (heads // kv_heads) + 15) // 16
    prefix = (128 << 20) // (blocks * kv_heads * 2 * pool.width * (2 if type_ == F16 else 4)) + 200
    pool.cache.dispose()
    pool = Pool(context, device, pool.layout, prefix // page_tokens + 2 * 300 // page_tokens + 8)
    batch = forked(pool, prefix, own)
    pool.host[...] = g.standard_normal(pool.host.shape, np.float32).astype(pool.host.dtype)
    for s in batch:
        last, n = pool.cache.pages(s)[-1], pool.cache.tokens(s) % page_tokens
        if n:
            pool.keys(0)[last, :, n:] = np.nan
            pool.values(0)[last, ..., n:] = np.inf
    pool.upload()
    q, got = attend(context, device, pool, batch, own, heads, g)
    row = 0
    for s, n in zip(batch, own):
        k, v = pool.of(s, 0)
        for r in sorted({0, 1, n // 2, n - 2, n - 1} | {int(i) for i in g.integers(0, n, 4)}):
            expected, bound = exact_attention(q[row + r], k, v, len(k) - n + r)
            err = np.abs(got[row + r].astype(np.float64) - expected)
            assert np.all(err <= bound), f"row {r} of {n}: {(err / bound).max()}"
        row += n
    group, table = heads // kv_heads, pool.cache.pages(batch[0])
    place = lambda i: (table[(prefix + i) // page_tokens], (prefix + i) % page_tokens)  # noqa: E731
    page, at = place(100)
    pool.values(0)[page, 0, 0, at] = np.inf
    page, at = place(155)
    pool.keys(0)[page, 0, at, 0] = np.nan
    pool.upload()
    plan, out = pool.cache.plan(heads), device(np.zeros_like(q))
    plan.set(batch, own)
    plan.attention(0, device(q), out)
    spoiled = context.download(np.zeros_like(q), out)
    plan.dispose()
    want = got.copy()
    want[100:300, :group, 0] = np.nan
    want[155:300, :group] = np.nan
    hit = np.isnan(want)
    assert not np.isfinite(spoiled[hit]).any()
    assert np.array_equal(spoiled[~hit], want[~hit])


@pytest.mark.parametrize("type_,heads,kv_heads,head_dim", [(F16, 16, 2, 128), (F32, 12, 1, 128), (F16, 8, 1, 256)])
def test_a_captured_step_follows_batches_of_other_kinds(context, device, type_, heads, kv_heads, head_dim):
    # The same 200 rows as one prompt without a past, as ten forks of a short prefix and as a chunk behind a long one (whose
    # tiles pass through LDS), each replay against an eager call on another plan.
    g = rng(head_dim + heads)
    rows, group = 200, heads // kv_heads
    width, size = head_dim, 2 if type_ == F16 else 4
    past = (128 << 20) // ((rows * group + 15) // 16 * kv_heads * 2 * width * size) + 100
    pool = Pool(context, device, CacheLayout(1, kv_heads, head_dim, 32, type_), past // 32 + 60)
    c = pool.cache
    prompt, behind, short = c.open(), c.open(), c.open()
    c.extend([prompt, behind, short], [rows, past + rows, 70])
    forks = [short] + c.fork(short, 9)
    c.extend(forks, [20] * 10)
    pool.write(g, [prompt, behind] + forks)
    batches = [([behind], [rows]), ([prompt], [rows]), (forks, [20] * 10)]
    q = g.standard_normal((rows, heads, head_dim)).astype(np.float32)
    dq, out, eager_out = device(q), device(np.zeros_like(q)), device(np.zeros_like(q))
    plan, other = c.plan(heads), c.plan(heads)
    plan.set(*batches[0])  # the largest, before the capture
    plan.set(*batches[1])
    context.capture_begin()
    plan.attention(0, dq, out)
    step = context.capture_end()
    for turn, i in enumerate((1, 0, 2, 0, 1)):
        context.upload(out, np.full_like(q, np.nan))
        plan.set(*batches[i])
        step.execute()
        got = context.download(np.zeros_like(q), out)
        other.set(*batches[i])
        other.attention(0, dq, eager_out)
        assert np.array_equal(got, context.download(np.zeros_like(q), eager_out)), (turn, i)
        if turn < 3:
            sequences, new = batches[i]
            some = rng(turn).integers(0, rows, 6)
            starts = np.cumsum([0] + new)
            for r in some:
                s = int(np.searchsorted(starts, r, side="right") - 1)
                k, v = pool.of(sequences[s], 0)
                expected, bound = exact_attention(q[r], k, v, len(k) - new[s] + int(r) - starts[s])
                assert np.all(np.abs(got[r] - expected) <= bound), (turn, int(r))
    step.dispose()
    plan.dispose()
    other.dispose()


def test_numbers_that_are_no_32_bit_integers(context, device):
    pool = Pool(context, device, CacheLayout(1, 1, 32, 32, F16), 8)
    c = pool.cache
    s = c.open()
    c.extend([s], [5])
    plan = c.plan(1)
    for bad in ([1 << 32], [1.5], np.array([1 << 32]), np.array([1.0])):
        with pytest.raises((OverflowError, TypeError)):
            plan.set([s], bad)
        with pytest.raises((OverflowError, TypeError)):
            c.extend([s], bad)
        with pytest.raises((OverflowError, TypeError)):
            c.copy_pages(bad, [2])
    with pytest.raises(S.ArgumentException):
        c.copy_pages([0, 1], [2])
    plan.set(np.array([s]), np.array([1]))  # 64-bit numpy integers that fit
    plan.dispose()
