"""The operators that serve several sequences at once, as programs that use this package run them: pages of a key/value
cache that sequences share, the batched cache write, the attention of a batch over such pages and low-rank adapters of
many requests beside one projection.

A case is a dict of plain values. `listed()` gives the fixed ones, `draw(rng)` another of the same ranges,
`prepare(case, seed)` what a program holds before the call, `run(state)` one pass: where `own` is false in plain torch,
where it is true through the package's entry points. `exact(case, seed)` gives the outputs from the definition in 64
bits, `work(case)` the bytes and operations nobody can do without.

Kinds:
  pages      forking a sequence, or copying one and closing the gap that freeing it leaves (whole cache pages move)
  append     bias, rotation and cache write of new positions of several sequences
  attention  new positions of several sequences over their pages, a common prefix in pages that all of them hold
  adapters   y = base + scale * up (down x), each row with the adapter of its request

A cache pool is [pages][layers][keys, values], a layer's keys [kv_heads][page_tokens][width] and its values
[kv_heads][width][page_tokens]; `width` is the head dimension rounded up to 32, 64, 96, 128, 192 or 256.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

PAGE = 32  # tokens of a page
TYPES = {"f32": torch.float32, "f16": torch.float16}
WIDTHS = (32, 64, 96, 128, 192, 256)
ROPE_BASE = 1e6

# The most a drawn case may do, which is what the largest listed ones do.
MOST_SCORES = 64 * 32 * 17000 * 128
MOST_POOL = 1536 * 28 * 2 * 2 * PAGE * 128 * 2
MOST_ADAPTED = 256 * 64 * (4096 + 11008)


def listed() -> list[dict]:
    return [
        # Three answers sampled from one prompt of a small model: the smallest fork.
        {"name": "fork_3", "kind": "pages", "mode": "fork", "type": "f16", "layers": 4, "kv_heads": 2, "head_dim": 64,
         "tokens": 75, "forks": 3, "pages": 64},
        # A beam of 48 over a 28-layer model: 48 last pages copied at once.
        {"name": "fork_48", "kind": "pages", "mode": "fork", "type": "f16", "layers": 28, "kv_heads": 2,
         "head_dim": 128, "tokens": 1000, "forks": 48, "pages": 256},
        # A long conversation copied and the gap that its original leaves closed: every page moves twice.
        {"name": "compact_16384", "kind": "pages", "mode": "compact", "type": "f16", "layers": 28, "kv_heads": 2,
         "head_dim": 128, "tokens": 16384, "behind": 9000, "pages": 1536},
        # One decode position of 16 sequences.
        {"name": "append_16", "kind": "append", "type": "f32", "heads": 12, "kv_heads": 2, "head_dim": 128,
         "sequences": 16, "new": 1, "longest": 2000},
        # Prompt chunks of 8 sequences, none on a page's border.
        {"name": "append_8x61", "kind": "append", "type": "f16", "heads": 32, "kv_heads": 8, "head_dim": 128,
         "sequences": 8, "new": 61, "longest": 3000},
        # Four short chats without anything in common: the smallest attention.
        {"name": "attention_4", "kind": "attention", "type": "f32", "heads": 12, "kv_heads": 2, "head_dim": 128,
         "sequences": 4, "new": 1, "prefix": 0, "shortest": 20, "longest": 120},
        # 24 requests of one application: a system prompt in common, ragged conversations of their own.
        {"name": "attention_24_f32", "kind": "attention", "type": "f32", "heads": 12, "kv_heads": 2, "head_dim": 128,
         "sequences": 24, "new": 1, "prefix": 4000, "shortest": 1, "longest": 700},
        # Drafts to verify: five positions of each of nine sequences, an odd head size.
        {"name": "attention_9x5", "kind": "attention", "type": "f16", "heads": 14, "kv_heads": 2, "head_dim": 80,
         "sequences": 9, "new": 5, "prefix": 1500, "shortest": 5, "longest": 400},
        # 64 questions about one long document.
        {"name": "attention_64_f16", "kind": "attention", "type": "f16", "heads": 32, "kv_heads": 8, "head_dim": 128,
         "sequences": 64, "new": 1, "prefix": 16384, "shortest": 64, "longest": 600},
        # One decode position of 32 requests, each with its own adapter of a 1.5B model's q projection.
        {"name": "adapters_32", "kind": "adapters", "type": "f16", "rows": 1536, "columns": 1536, "rank": 16,
         "adapters": 32, "positions": 32},
        # Seven rows, odd sizes, FP32 adapters of different ranks.
        {"name": "adapters_7_f32", "kind": "adapters", "type": "f32", "rows": 1001, "columns": 1477, "rank": 11,
         "adapters": 3, "positions": 7},
        # A prompt chunk of two requests with large adapters on a wide projection.
        {"name": "adapters_256", "kind": "adapters", "type": "f16", "rows": 11008, "columns": 4096, "rank": 64,
         "adapters": 2, "positions": 256},
    ]


def _log(rng, low: int, high: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng) -> dict:
    kind = rng.choice(["pages", "append", "attention", "attention", "adapters", "adapters"])
    type_ = rng.choice(["f32", "f16"])
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 4, 6, 7])
    head_dim = rng.choice([48, 64, 80, 96, 128, 128, 192, 256])
    if kind == "pages":
        layers = _log(rng, 2, 32)
        most = MOST_POOL // _page_bytes(type_, layers, kv_heads, head_dim)
        if rng.random() < 0.5:
            tokens, forks = _log(rng, 33, 4000) | 1, _log(rng, 2, 64)
            if tokens // PAGE + forks + 2 <= most:
                return {"kind": kind, "mode": "fork", "type": type_, "layers": layers, "kv_heads": kv_heads,
                        "head_dim": head_dim, "tokens": tokens, "forks": forks, "pages": tokens // PAGE + forks + 2}
        used = max(2, most // 3)
        tokens = min(_log(rng, 40, 16384), used * PAGE)
        behind = min(_log(rng, 40, 9000), used * PAGE)
        return {"kind": kind, "mode": "compact", "type": type_, "layers": layers, "kv_heads": kv_heads,
                "head_dim": head_dim, "tokens": tokens, "behind": behind,
                "pages": 2 * _pages(tokens) + _pages(behind) + rng.randint(0, 9)}
    if kind == "append":
        sequences = _log(rng, 1, 64)
        return {"kind": kind, "type": type_, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
                "sequences": sequences, "new": rng.choice([1, _log(rng, 1, max(1, 512 // sequences))]),
                "longest": _log(rng, 600, 9000)}
    if kind == "attention":
        while True:
            sequences = _log(rng, 1, 64)
            new = rng.choice([1, 1, _log(rng, 2, 96)])
            prefix, longest = rng.choice([0, _log(rng, 32, 16384)]), _log(rng, max(new, 16), 4000)
            if sequences * new <= 512 and sequences * new * heads * (prefix + longest) * head_dim <= MOST_SCORES:
                return {"kind": kind, "type": type_, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
                        "sequences": sequences, "new": new, "prefix": prefix,
                        "shortest": rng.randint(new, longest), "longest": longest}
    while True:
        rows, columns, rank = _log(rng, 200, 14336), _log(rng, 200, 14336), _log(rng, 1, 128)
        positions = rng.choice([1, _log(rng, 2, 256), _log(rng, 2, 256)])
        if positions * rank * (rows + columns) <= MOST_ADAPTED:
            return {"kind": kind, "type": type_, "rows": rows, "columns": columns, "rank": rank,
                    "adapters": _log(rng, 1, min(64, positions)), "positions": positions}


# ---- sizes ----

def _pages(tokens: int) -> int:
    return -(-tokens // PAGE)


def _width(head_dim: int) -> int:
    return next(w for w in WIDTHS if w >= head_dim)


def _page_bytes(type_: str, layers: int, kv_heads: int, head_dim: int) -> int:
    return layers * 2 * kv_heads * PAGE * _width(head_dim) * TYPES[type_].itemsize


def _spread(low: int, high: int, count: int) -> list[int]:
    """`count` lengths from low to high, unevenly spaced and out of order."""
    if count == 1:
        return [high]
    steps = [low + round((high - low) * (i / (count - 1)) ** 2) for i in range(count)]
    return steps[::2] + steps[1::2][::-1]


def _lengths(case: dict) -> list[int]:
    """Tokens of each sequence of an attention or append case, its new ones among them."""
    if case["kind"] == "append":
        return [n + case["new"] for n in _spread(case["longest"] // 8, case["longest"], case["sequences"])]
    return [case["prefix"] + n for n in _spread(case["shortest"], case["longest"], case["sequences"])]


def _shared_pages(case: dict) -> int:
    """Pages that all sequences of an attention case hold: the prefix's whole pages (its last tokens, in a page that is
    not full, are each sequence's own copy)."""
    return case["prefix"] // PAGE if case["sequences"] > 1 else 0


def work(case: dict) -> dict:
    kind = case["kind"]
    if kind == "pages":
        moves = case["forks"] if case["mode"] == "fork" else 2 * _pages(case["tokens"])
        return {"bytes": 2 * moves * _page_bytes(case["type"], case["layers"], case["kv_heads"], case["head_dim"]),
                "flops": 0}
    size = TYPES[case["type"]].itemsize
    if kind == "append":
        h, kv, d, n = case["heads"], case["kv_heads"], case["head_dim"], case["sequences"] * case["new"]
        return {"bytes": n * (8 * h * d + kv * d * (8 + 2 * size) + 8 * d) + 4 * d * (h + 2 * kv),
                "flops": 7 * n * d * (h + kv)}
    if kind == "attention":
        h, kv, d, new = case["heads"], case["kv_heads"], case["head_dim"], case["new"]
        lengths, shared = _lengths(case), _shared_pages(case) * PAGE
        tokens = shared + sum(n - shared for n in lengths)
        pairs = sum(new * n - new * (new - 1) // 2 for n in lengths)
        return {"bytes": 2 * size * kv * d * tokens + 8 * len(lengths) * new * h * d, "flops": 4 * h * d * pairs}
    ranks, wide = _ranks(case), case["rows"] + case["columns"]
    return {"bytes": sum(ranks) * wide * size + 4 * case["positions"] * (case["columns"] + 2 * case["rows"]),
            "flops": sum(2 * ranks[a] * wide for a in _selection(case) if a >= 0)}


# ---- inputs, from the seed alone ----

def _generator(seed: int) -> torch.Generator:
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, *shape, scale: float = 1.0, type_: str = "f32") -> torch.Tensor:
    return torch.empty(*shape, device="cuda", dtype=TYPES[type_]).normal_(0, scale, generator=g)


def _pool(g, case: dict, pages: int, layers: int) -> torch.Tensor:
    return _normal(g, pages, layers, 2, case["kv_heads"] * PAGE * _width(case["head_dim"]), type_=case["type"])


def _keys(pool: torch.Tensor, case: dict, layer: int) -> torch.Tensor:
    """[pages][kv_heads][tokens][head_dim]"""
    return pool[:, layer, 0].view(pool.shape[0], case["kv_heads"], PAGE, -1)[..., :case["head_dim"]]


def _values(pool: torch.Tensor, case: dict, layer: int) -> torch.Tensor:
    """[pages][kv_heads][head_dim][tokens]"""
    return pool[:, layer, 1].view(pool.shape[0], case["kv_heads"], -1, PAGE)[:, :, :case["head_dim"]]


def _tables(case: dict) -> list[list[int]]:
    """The pages of each sequence: the common prefix first, then every sequence's own in turn."""
    shared = _shared_pages(case) if case["kind"] == "attention" else 0
    tables, following = [], shared
    for n in _lengths(case):
        mine = _pages(n) - shared
        tables.append(list(range(shared)) + list(range(following, following + mine)))
        following += mine
    return tables


def _positions(case: dict) -> list[int]:
    return [p for n in _lengths(case) for p in range(n - case["new"], n)]


def _rope_table(positions: int, rotary: int) -> torch.Tensor:
    """Sines, then cosines, of every position's angles, in 64 bits."""
    k = torch.arange(rotary // 2, device="cuda", dtype=torch.float64)
    angle = torch.arange(positions, device="cuda", dtype=torch.float64)[:, None] / ROPE_BASE ** (2 * k / rotary)
    return torch.cat([torch.sin(angle), torch.cos(angle)], dim=1)


def _append_inputs(case: dict, seed: int):
    g = _generator(seed)
    n, h, kv, d = case["sequences"] * case["new"], case["heads"], case["kv_heads"], case["head_dim"]
    q, k, v = _normal(g, n, h, d), _normal(g, n, kv, d), _normal(g, n, kv, d)
    biases = _normal(g, h, d, scale=0.1), _normal(g, kv, d, scale=0.1), _normal(g, kv, d, scale=0.1)
    pool = _pool(g, case, sum(map(len, _tables(case))), 1)
    if _width(d) > d:  # the padding of what is written is zero
        pool.view(-1, 2, case["kv_heads"], PAGE * _width(d)).zero_()
    return q, k, v, biases, pool


def _attention_inputs(case: dict, seed: int):
    g = _generator(seed)
    pool = _pool(g, case, max(max(t) for t in _tables(case)) + 1, 1)
    if _width(case["head_dim"]) > case["head_dim"]:
        pool[:, 0, 0].view(pool.shape[0], case["kv_heads"], PAGE, -1)[..., case["head_dim"]:] = 0
    return _normal(g, case["sequences"] * case["new"], case["heads"], case["head_dim"]), pool


def _ranks(case: dict) -> list[int]:
    return [max(1, case["rank"] - (i % 4) * (case["rank"] // 8)) for i in range(case["adapters"])]


def _selection(case: dict) -> list[int]:
    """The adapter of each row: consecutive rows are a request's; with more than two rows one of them has none."""
    n = case["positions"]
    selection = [i * case["adapters"] // n for i in range(n)]
    if n > 2:
        selection[n // 2] = -1
    return selection


def _adapter_inputs(case: dict, seed: int):
    g = _generator(seed)
    count, n, ranks = case["adapters"], case["positions"], _ranks(case)
    down = [_normal(g, r, case["columns"], scale=case["columns"] ** -0.5, type_=case["type"]) for r in ranks]
    up = [_normal(g, case["rows"], r, scale=r ** -0.5, type_=case["type"]) for r in ranks]
    scales = [2.0 / (1 + i % 3) for i in range(count)]
    return down, up, scales, _selection(case), _normal(g, n, case["columns"]), _normal(g, n, case["rows"])


# ---- what a program keeps ----

class _State:
    """Tensors and, for the package's own calls, handles, which are released from the last to the first."""

    def __init__(self, case: dict):
        self.case, self.owned = case, []

    def hold(self, thing):
        self.owned.append(thing)
        return thing

    def __del__(self):
        while self.owned:
            self.owned.pop().dispose()


def _cache(state, pool: torch.Tensor, layers: int):
    import satori_amd as S
    from satori_amd.cache import CacheLayout, ElementType, PagedCache

    case = state.case
    layout = CacheLayout(layers=layers, kv_heads=case["kv_heads"], head_dim=case["head_dim"], page_tokens=PAGE,
                         type=ElementType[case["type"].upper()])
    torch.cuda.synchronize()  # the pool is filled on another stream than the cache's
    return state.hold(PagedCache(S.default_context(), layout, pool.shape[0], pool.data_ptr()))


def _open(cache, case: dict) -> list[int]:
    """Sequences that hold the pages of _tables(case): the prefix once, the others forked from it."""
    lengths, shared = _lengths(case), _shared_pages(case) * PAGE if case["kind"] == "attention" else 0
    first = cache.open()
    cache.extend([first], [shared])
    sequences = [first] + cache.fork(first, len(lengths) - 1)
    for s, n in zip(sequences, lengths):
        cache.extend([s], [n - shared])
    return sequences


def prepare(case: dict, seed: int):
    state = _State(case)
    kind = case["kind"]
    if kind == "pages":
        state.pool = _pool(_generator(seed), case, case["pages"], case["layers"])
        if own:
            state.cache = _cache(state, state.pool, case["layers"])
            state.first = state.cache.open()
            state.cache.extend([state.first], [case["tokens"]])
            if case["mode"] == "compact":
                state.behind = state.cache.open()
                state.cache.extend([state.behind], [case["behind"]])
        else:
            state.first = list(range(_pages(case["tokens"])))
            if case["mode"] == "compact":
                state.behind = list(range(len(state.first), len(state.first) + _pages(case["behind"])))
    elif kind == "adapters":
        state.down, state.up, state.scales, state.selection, state.x, state.base = _adapter_inputs(case, seed)
        state.y = torch.zeros_like(state.base)
        if own:
            import satori_amd as S
            from satori_amd.adapters import LowRankAdapters
            from satori_amd.cache import ElementType

            torch.cuda.synchronize()
            weights = [(a.data_ptr(), b.data_ptr(), a.shape[0], s)
                       for a, b, s in zip(state.down, state.up, state.scales)]
            state.adapters = state.hold(LowRankAdapters(S.default_context(), case["rows"], case["columns"], weights,
                                                        ElementType[case["type"].upper()]))
            state.arguments = (np.array(state.selection, np.int32), state.x.data_ptr(), state.base.data_ptr(),
                               state.y.data_ptr())
        else:
            ranks = torch.tensor(_ranks(case), device="cuda")
            state.owner = torch.arange(case["adapters"], device="cuda").repeat_interleave(ranks)
            state.factor = torch.tensor(state.scales, device="cuda").repeat_interleave(ranks)
            state.chosen = torch.tensor(state.selection, device="cuda")
    else:
        if kind == "append":
            state.q, state.k, state.v, state.biases, state.pool = _append_inputs(case, seed)
            state.rope = _rope_table(max(_lengths(case)), case["head_dim"])
        else:
            state.q, state.pool = _attention_inputs(case, seed)
        state.out = torch.zeros_like(state.q)
        if own:
            cache = _cache(state, state.pool, 1)
            state.sequences = _open(cache, case)
            state.plan = state.hold(cache.plan(case["heads"]))
            state.plan.set(state.sequences, [case["new"]] * case["sequences"])
        else:
            tables = _tables(case)
            most = max(map(len, tables))
            state.table = torch.tensor([t + [0] * (most - len(t)) for t in tables], device="cuda")
            state.row_sequence = torch.arange(case["sequences"], device="cuda").repeat_interleave(case["new"])
            state.positions = torch.tensor(_positions(case), device="cuda")
    return state


# ---- one pass ----

def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(state):
    case = state.case
    if case["kind"] == "pages":
        cache = state.cache
        if case["mode"] == "fork":
            forks = cache.fork(state.first, case["forks"])
            cache.extend(forks, [1] * len(forks))
            tables = [cache.pages(f) for f in forks]
            cache.free(forks)
            return {"pool": state.pool, "tables": torch.tensor(tables)}
        copied = cache.copy(state.first)
        cache.free([state.first])
        state.first = copied
        cache.compact()
        return {"pool": state.pool, "tables": torch.tensor(cache.pages(state.first) + cache.pages(state.behind))}
    if case["kind"] == "append":
        d = case["head_dim"]
        state.plan.append(0, state.q.data_ptr(), state.biases[0].data_ptr(), state.out.data_ptr(), state.k.data_ptr(),
                          state.biases[1].data_ptr(), state.v.data_ptr(), state.biases[2].data_ptr(), ROPE_BASE, d,
                          state.rope.data_ptr(), state.rope.shape[0])
        return {"q": state.out, "pool": state.pool}
    if case["kind"] == "attention":
        state.plan.attention(0, state.q.data_ptr(), state.out.data_ptr())
        return state.out
    state.adapters.apply(*state.arguments)
    return state.y


def _move(pool: torch.Tensor, sources: list[int], destinations: list[int]) -> None:
    pool[torch.tensor(destinations, device=pool.device)] = pool[torch.tensor(sources, device=pool.device)]


def _run_plain(state):
    case = state.case
    if case["kind"] == "pages":
        count = len(state.first)
        if case["mode"] == "fork":
            new = list(range(count, count + case["forks"]))  # the lowest free pages
            _move(state.pool, [state.first[-1]] * len(new), new)
            return {"pool": state.pool, "tables": torch.tensor([state.first[:-1] + [p] for p in new])}
        new = list(range(count + len(state.behind), 2 * count + len(state.behind)))
        _move(state.pool, state.first, new)  # the copy; its original is freed,
        _move(state.pool, new[-count:], state.first)  # and the pages behind move into the gap
        return {"pool": state.pool, "tables": torch.tensor(state.first + state.behind)}
    if case["kind"] == "append":
        return _append_plain(state)
    if case["kind"] == "attention":
        return _attention_plain(state)
    # Every row times every adapter in two products, the others' parts of a row set to zero between them.
    down, up = torch.cat(state.down).float(), torch.cat(state.up, dim=1).float()
    mine = state.owner == state.chosen[:, None]
    state.y.copy_(state.base + torch.where(mine, state.x @ down.T * state.factor, 0) @ up.T)
    return state.y


def _rotate(x: torch.Tensor, sn: torch.Tensor, cs: torch.Tensor) -> torch.Tensor:
    """[rows][heads][head_dim] by each row's angles, the first half of a head with the second, rounded to FP32."""
    a, b = x.double().chunk(2, dim=-1)
    return torch.cat([a * cs[:, None] - b * sn[:, None], a * sn[:, None] + b * cs[:, None]], dim=-1).float()


def _append_plain(state):
    case = state.case
    sn, cs = state.rope[state.positions].chunk(2, dim=1)
    state.out.copy_(_rotate(state.q + state.biases[0], sn, cs))
    pages = state.table[state.row_sequence, state.positions // PAGE]
    offsets = state.positions % PAGE
    _keys(state.pool, case, 0)[pages, :, offsets] = _rotate(state.k + state.biases[1], sn, cs).to(state.pool.dtype)
    _values(state.pool, case, 0)[pages, :, :, offsets] = (state.v + state.biases[2]).to(state.pool.dtype)
    return {"q": state.out, "pool": state.pool}


def _attention_plain(state):
    case = state.case
    b, new, kv, d = case["sequences"], case["new"], case["kv_heads"], case["head_dim"]
    group = case["heads"] // kv
    tokens = state.table.shape[1] * PAGE
    k = _keys(state.pool, case, 0)[state.table].permute(0, 2, 1, 3, 4).reshape(b * kv, tokens, d).float()
    v = _values(state.pool, case, 0)[state.table].permute(0, 2, 1, 4, 3).reshape(b * kv, tokens, d).float()
    q = state.q.view(b, new, kv, group, d).permute(0, 2, 1, 3, 4).reshape(b * kv, new * group, d)
    scores = (torch.bmm(q, k.transpose(1, 2).contiguous()) / math.sqrt(d)).view(b, kv, new, group, tokens)
    hidden = torch.arange(tokens, device=q.device) > state.positions.view(b, 1, new, 1, 1)
    scores = scores.masked_fill(hidden, -math.inf)
    p = (scores - scores.amax(-1, keepdim=True)).exp()
    p = (p / p.sum(-1, keepdim=True)).view(b * kv, new * group, tokens)
    out = torch.bmm(p, v).view(b, kv, new, group, d)
    state.out.copy_(out.permute(0, 2, 1, 3, 4).reshape(state.out.shape))
    return state.out


# ---- the outputs in 64 bits ----

def exact(case: dict, seed: int):
    kind = case["kind"]
    if kind == "pages":
        pool = _pool(_generator(seed), case, case["pages"], case["layers"])
        first = _pages(case["tokens"])
        if case["mode"] == "fork":
            pool[first:first + case["forks"]] = pool[first - 1].clone()
            return {"pool": pool, "tables": None}
        start = first + _pages(case["behind"])
        pool[start:start + first] = pool[:first].clone()
        return {"pool": pool, "tables": None}
    if kind == "append":
        q, k, v, (bq, bk, bv), pool = _append_inputs(case, seed)
        pool64 = pool.double()
        out = torch.zeros(q.shape, device="cuda", dtype=torch.float64)
        half = case["head_dim"] // 2
        frequency = ROPE_BASE ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
        tables, row = _tables(case), 0
        for s, n in enumerate(_lengths(case)):
            for position in range(n - case["new"], n):
                turn = torch.polar(torch.ones_like(frequency), position * frequency)

                def rotated(x):
                    z = torch.view_as_real(torch.complex(x[:, :half].contiguous(), x[:, half:].contiguous()) * turn)
                    return torch.cat([z[..., 0], z[..., 1]], dim=-1)

                page, offset = tables[s][position // PAGE], position % PAGE
                out[row] = rotated(q[row].double() + bq.double())
                _keys(pool64, case, 0)[page, :, offset] = rotated(k[row].double() + bk.double())
                _values(pool64, case, 0)[page, :, :, offset] = v[row].double() + bv.double()
                row += 1
        return {"q": out, "pool": pool64}
    if kind == "attention":
        q, pool = _attention_inputs(case, seed)
        q, new = q.double(), case["new"]
        kv, d = case["kv_heads"], case["head_dim"]
        out = torch.zeros_like(q)
        keys, values = _keys(pool, case, 0), _values(pool, case, 0)
        for s, (n, table) in enumerate(zip(_lengths(case), _tables(case))):
            at = torch.tensor(table, device="cuda")
            seen = torch.arange(n, device="cuda")[None] <= torch.arange(n - new, n, device="cuda")[:, None]
            for h in range(kv):
                k = keys[at, h].reshape(-1, d)[:n].double()
                v = values[at, h].transpose(1, 2).reshape(-1, d)[:n].double()
                for head in range(h * (case["heads"] // kv), (h + 1) * (case["heads"] // kv)):
                    scores = torch.where(seen, q[s * new:(s + 1) * new, head] @ k.T * d ** -0.5, -math.inf)
                    out[s * new:(s + 1) * new, head] = torch.softmax(scores, dim=-1) @ v
        return out
    down, up, scales, selection, x, base = _adapter_inputs(case, seed)
    out = base.double()
    for r, a in enumerate(selection):
        if a >= 0:
            out[r] += scales[a] * (up[a].double() @ (down[a].double() @ x[r].double()))
    return out
