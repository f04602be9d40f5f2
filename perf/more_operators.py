"""The operators that serve drafted trees of tokens, as programs that use this package run them: rotary positions of rows
(both layouts, part of a head, scaled for long contexts), alone and on the way into cache pages, the attention of a tree of
drafts over a cache, the copy that keeps an accepted branch, and the logits' penalties, biases and grammar masks.

A case is a dict of plain values. `listed()` gives the fixed ones, `draw(rng)` another of the same ranges,
`prepare(case, seed)` what a program holds before the call, `run(state)` one pass: where `own` is false in plain torch,
where it is true through the package's entry points. `exact(case, seed)` gives the outputs from the definition in 64
bits, `work(case)` the bytes and operations nobody can do without.

Kinds:
  rotate     every head of every row turned by its row's position
  append     bias, rotation at the tree's positions and cache write of drafted rows
  attention  drafted rows over their sequence's context and their own branch of the tree
  keep       the keys and values of accepted drafts moved to follow their contexts, in all layers
  logits     penalties for repeated tokens, biases and grammar masks, and the best token of each row

A tree: row j of a sequence follows row parent(j) < j of the same sequence, or its context (-1); row j lies at the cache
position behind the context that its number says, and stands for the position that its depth says.

A cache pool is [pages][layers][keys, values], a layer's keys [kv_heads][page_tokens][width] and its values
[kv_heads][width][page_tokens]; `width` is the head dimension rounded up to 32, 64, 96, 128, 192 or 256.
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

PAGE = 32  # tokens of a page
TYPES = {"f32": torch.float32, "f16": torch.float16}
WIDTHS = (32, 64, 96, 128, 192, 256)
TURNS = (1.0, 32.0)  # of a scaled rotation over its original positions: fewer are scaled in full, more not at all

# The most a drawn case may do, which is what the largest listed ones do.
MOST_ROTATED = 4096 * 32 * 128
MOST_SCORES = 8 * 64 * 32 * 17000 * 128
MOST_KEPT = 64 * 7 * 28 * 2 * 128
MOST_LOGITS = 512 * 151936
MOST_CACHE = 8 * 12000 * 2 * 8 * 128 * 2   # bytes of an attention's pool
MOST_POOL = 64 * 14 * 28 * 2 * 2 * PAGE * 128 * 2  # and of the pool that branches are kept in


def listed() -> list[dict]:
    return [
        # The queries of one decode position of eight requests, a context stretched four times.
        {"name": "rotate_8", "kind": "rotate", "type": "f32", "layout": "half", "rows": 8, "heads": 12, "head_dim": 128,
         "rotary": 128, "gap": 0, "base": 1e6, "scaling": "yarn", "factor": 4.0, "original": 32768, "longest": 100000},
        # A long prompt's queries inside a fused projection's rows, neighbouring lanes in pairs.
        {"name": "rotate_4096_f16", "kind": "rotate", "type": "f16", "layout": "interleaved", "rows": 4096, "heads": 32,
         "head_dim": 128, "rotary": 128, "gap": 2048, "base": 10000.0, "scaling": "linear", "factor": 2.0,
         "original": 4096, "longest": 8192},
        # Seven drafts of each of four chats, pairs half a head apart.
        {"name": "append_4x7", "kind": "append", "type": "f32", "layout": "half", "heads": 12, "kv_heads": 2,
         "head_dim": 128, "rotary": 128, "base": 1e6, "scaling": "yarn", "factor": 4.0, "original": 32768,
         "sequences": 4, "new": 7, "tree": 1, "shortest": 300, "longest": 40000},
        # Trees of 61 drafts of sixteen requests, part of each head rotated, in neighbouring lanes.
        {"name": "append_16x61_f16", "kind": "append", "type": "f16", "layout": "interleaved", "heads": 32,
         "kv_heads": 8, "head_dim": 128, "rotary": 64, "base": 10000.0, "scaling": "wavelength", "factor": 8.0,
         "original": 8192, "sequences": 16, "new": 61, "tree": 2, "shortest": 100, "longest": 3000},
        # One chat's small tree: the smallest attention.
        {"name": "attention_1x8", "kind": "attention", "type": "f32", "heads": 12, "kv_heads": 2, "head_dim": 128,
         "sequences": 1, "new": 8, "tree": 3, "prefix": 0, "shortest": 300, "longest": 300},
        # Nine requests of one application with a prompt in common, an odd head size.
        {"name": "attention_9x13_f16", "kind": "attention", "type": "f16", "heads": 14, "kv_heads": 2, "head_dim": 80,
         "sequences": 9, "new": 13, "tree": 4, "prefix": 1500, "shortest": 1, "longest": 700},
        # Large trees over long contexts.
        {"name": "attention_8x64_f16", "kind": "attention", "type": "f16", "heads": 32, "kv_heads": 8, "head_dim": 128,
         "sequences": 8, "new": 64, "tree": 5, "prefix": 0, "shortest": 4000, "longest": 16384},
        # One accepted branch of a small model.
        {"name": "keep_1", "kind": "keep", "type": "f16", "layers": 4, "kv_heads": 2, "head_dim": 64, "sequences": 1,
         "new": 8, "kept": 3, "shortest": 300, "longest": 300},
        # A whole batch's accepted branches over a 28-layer model.
        {"name": "keep_64", "kind": "keep", "type": "f16", "layers": 28, "kv_heads": 2, "head_dim": 128,
         "sequences": 64, "new": 61, "kept": 7, "shortest": 20, "longest": 900},
        # One request's next token: penalties over its conversation, a grammar.
        {"name": "logits_1", "kind": "logits", "vocabulary": 151936, "sequences": 1, "new": 1, "tree": 0,
         "shortest": 2000, "longest": 2000, "biases": 0, "masks": 1, "coarse": False, "written": True},
        # The best tokens of 24 requests, nothing else wanted, an odd vocabulary.
        {"name": "logits_24_best", "kind": "logits", "vocabulary": 32003, "sequences": 24, "new": 1, "tree": 0,
         "shortest": 0, "longest": 4000, "biases": 40, "masks": 5, "coarse": True, "written": False},
        # Every draft of eight large trees, its branch counted with its conversation, grammars of their own.
        {"name": "logits_8x64", "kind": "logits", "vocabulary": 151936, "sequences": 8, "new": 64, "tree": 6,
         "shortest": 100, "longest": 16384, "biases": 300, "masks": 64, "coarse": False, "written": True},
    ]


def _log(rng, low: int, high: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _draw_rotation(rng, head_dim: int) -> dict:
    return {"layout": rng.choice(["half", "interleaved"]), "rotary": rng.choice([head_dim, head_dim, 2 * rng.randint(2, head_dim // 2)]),
            "base": rng.choice([10000.0, 500000.0, 1e6]), "scaling": rng.choice(["none", "linear", "ntk", "yarn", "wavelength"]),
            "factor": rng.choice([2.0, 4.0, 8.0, rng.uniform(1.1, 20.0)]), "original": rng.choice([2048, 4096, 8192, 32768])}


def draw(rng) -> dict:
    kind = rng.choice(["rotate", "append", "attention", "attention", "keep", "logits", "logits"])
    type_ = rng.choice(["f32", "f16"])
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 4, 6, 7])
    head_dim = rng.choice([48, 64, 80, 96, 128, 128, 192, 256])
    tree = rng.randint(1, 10 ** 6)
    while kind == "rotate":
        rows, heads = _log(rng, 1, 8192), _log(rng, 1, 64)
        if rows * heads * head_dim <= MOST_ROTATED:
            return {"kind": kind, "type": type_, "rows": rows, "heads": heads, "head_dim": head_dim,
                    "gap": rng.choice([0, 0, rng.randint(1, 2000)]), "longest": _log(rng, 100, 131072),
                    **_draw_rotation(rng, head_dim)}
    if kind == "append":
        sequences = _log(rng, 1, 64)
        longest = _log(rng, 100, 9000)
        return {"kind": kind, "type": type_, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
                "sequences": sequences, "new": _log(rng, 1, max(1, 1000 // sequences)), "tree": tree,
                "shortest": rng.randint(0, longest), "longest": longest, **_draw_rotation(rng, head_dim)}
    while kind == "attention":
        sequences, new = _log(rng, 1, 64), _log(rng, 2, 256)
        prefix, longest = rng.choice([0, _log(rng, 32, 8192)]), _log(rng, 16, 16384)
        total = (prefix + longest + new) * sequences * new
        cache = (prefix + sequences * (longest + new)) * 2 * kv_heads * _width(head_dim) * TYPES[type_].itemsize
        if sequences * new <= 1024 and total * heads * head_dim <= MOST_SCORES and cache <= MOST_CACHE:
            return {"kind": kind, "type": type_, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
                    "sequences": sequences, "new": new, "tree": tree, "prefix": prefix,
                    "shortest": rng.randint(0, longest), "longest": longest}
    while kind == "keep":
        sequences, layers, new = _log(rng, 1, 64), _log(rng, 2, 32), _log(rng, 4, 128)
        kept, longest = rng.randint(2, max(2, min(9, new // 2))), _log(rng, 16, 1200)
        pool = sequences * (_pages(longest + new) + 1) * layers * 2 * kv_heads * PAGE * _width(head_dim) * TYPES[type_].itemsize
        if sequences * kept * layers * kv_heads * head_dim <= MOST_KEPT and pool <= MOST_POOL:
            return {"kind": kind, "type": type_, "layers": layers, "kv_heads": kv_heads, "head_dim": head_dim,
                    "sequences": sequences, "new": new, "kept": kept, "shortest": rng.randint(0, longest),
                    "longest": longest}
    while True:
        sequences, new, vocabulary = _log(rng, 1, 64), rng.choice([1, _log(rng, 2, 64)]), _log(rng, 200, 200000)
        if sequences * new * vocabulary <= MOST_LOGITS:
            longest = _log(rng, 10, 16384)
            return {"kind": "logits", "vocabulary": vocabulary, "sequences": sequences, "new": new,
                    "tree": tree if new > 1 else 0, "shortest": rng.randint(0, longest), "longest": longest,
                    "biases": rng.choice([0, _log(rng, 1, min(1000, vocabulary // 2))]),
                    "masks": rng.choice([0, 1, _log(rng, 2, 64)]), "coarse": rng.random() < 0.5,
                    "written": rng.random() < 0.7}


# ---- sizes ----

def _pages(tokens: int) -> int:
    return -(-tokens // PAGE)


def _width(head_dim: int) -> int:
    return next(w for w in WIDTHS if w >= head_dim)


def _spread(low: int, high: int, count: int) -> list[int]:
    """`count` lengths from low to high, unevenly spaced and out of order."""
    if count == 1:
        return [high]
    steps = [low + round((high - low) * (i / (count - 1)) ** 2) for i in range(count)]
    return steps[::2] + steps[1::2][::-1]


def _contexts(case: dict) -> list[int]:
    """Tokens of each sequence before its drafted rows."""
    return [case.get("prefix", 0) + n for n in _spread(case["shortest"], case["longest"], case["sequences"])]


def _parents(case: dict, sequence: int) -> list[int]:
    """The row that each row of a sequence follows: the first one the context, later ones an earlier one, near ones first."""
    r = random.Random(case["tree"] * 1000 + sequence)
    branch = r.choice([1, 2, 3, 4, 8])
    return [-1] + [r.randrange(j) if r.random() < 0.2 else (j - 1) // branch for j in range(1, case["new"])]


def _depths(parents: list[int]) -> list[int]:
    depths = []
    for p in parents:
        depths.append(0 if p < 0 else depths[p] + 1)
    return depths


def _branch(parents: list[int], row: int) -> list[int]:
    """A row and those it follows."""
    found = [row]
    while parents[found[-1]] >= 0:
        found.append(parents[found[-1]])
    return found


def _kept(case: dict, sequence: int) -> list[int]:
    """The rows that a keep case keeps: the first one and later ones, none of them at a place that the kept ones move to."""
    r = random.Random(sequence * 7919 + case["new"])
    count = r.randint(2, case["kept"])
    return [0] + sorted(r.sample(range(count, case["new"]), count - 1))


def _shared_pages(case: dict) -> int:
    """Pages that all sequences of an attention case hold: the prefix's whole pages."""
    return case["prefix"] // PAGE if case["kind"] == "attention" and case["sequences"] > 1 else 0


def _history(case: dict) -> list[int]:
    return _spread(case["shortest"], case["longest"], case["sequences"])


def work(case: dict) -> dict:
    kind = case["kind"]
    if kind == "logits":
        rows, v = case["sequences"] * case["new"], case["vocabulary"]
        masks = min(case["masks"], rows)
        sets = min(4, case["sequences"]) if case["biases"] else 0
        return {"bytes": 4 * rows * v * (2 if case["written"] else 1) + 4 * -(-v // 32) * masks + 4 * rows +
                4 * sum(_history(case)) + 8 * sets * case["biases"], "flops": rows * v}
    size, d = TYPES[case["type"]].itemsize, case["head_dim"]
    if kind == "rotate":
        n = case["rows"] * case["heads"]
        return {"bytes": 2 * n * d * size + 4 * case["rows"], "flops": 3 * n * case["rotary"]}
    kv, n = case["kv_heads"], case["sequences"] * case["new"]
    if kind == "keep":
        moved = sum(len(_kept(case, s)) - 1 for s in range(case["sequences"]))
        return {"bytes": 2 * moved * case["layers"] * 2 * kv * _width(d) * size, "flops": 0}
    h = case["heads"]
    if kind == "append":
        return {"bytes": n * (8 * h * d + kv * d * (8 + 2 * size)) + 4 * d * (h + 2 * kv),
                "flops": n * (h + kv) * (3 * case["rotary"] + d)}
    contexts, shared = _contexts(case), _shared_pages(case) * PAGE
    tokens = shared + sum(c + case["new"] - shared for c in contexts)
    seen = sum(case["new"] * c + sum(x + 1 for x in _depths(_parents(case, s))) for s, c in enumerate(contexts))
    return {"bytes": 2 * size * kv * d * tokens + 8 * n * h * d, "flops": 4 * h * d * seen}


# ---- inputs, from the seed alone ----

def _generator(seed: int) -> torch.Generator:
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, *shape, scale: float = 1.0, type_: str = "f32") -> torch.Tensor:
    return torch.empty(*shape, device="cuda", dtype=TYPES[type_]).normal_(0, scale, generator=g)


def _integers(g, low: int, high: int, *shape) -> torch.Tensor:
    return torch.randint(low, high, shape, device="cuda", generator=g, dtype=torch.int32)


def _pool(g, case: dict, pages: int, layers: int) -> torch.Tensor:
    """Pages whose keys' padding is zero."""
    pool = _normal(g, pages, layers, 2, case["kv_heads"] * PAGE * _width(case["head_dim"]), type_=case["type"])
    if _width(case["head_dim"]) > case["head_dim"]:
        pool[:, :, 0].unflatten(-1, (case["kv_heads"], PAGE, -1))[..., case["head_dim"]:] = 0
    return pool


def _keys(pool: torch.Tensor, case: dict) -> torch.Tensor:
    """[pages][layers][kv_heads][tokens][head_dim]"""
    return pool[:, :, 0].unflatten(-1, (case["kv_heads"], PAGE, -1))[..., :case["head_dim"]]


def _values(pool: torch.Tensor, case: dict) -> torch.Tensor:
    """[pages][layers][kv_heads][head_dim][tokens]"""
    return pool[:, :, 1].unflatten(-1, (case["kv_heads"], -1, PAGE))[:, :, :, :case["head_dim"]]


def _tables(case: dict) -> list[list[int]]:
    """The pages of each sequence: the common prefix first, then every sequence's own in turn."""
    shared = _shared_pages(case)
    tables, following = [], shared
    for c in _contexts(case):
        mine = _pages(c + case["new"]) - shared
        tables.append(list(range(shared)) + list(range(following, following + mine)))
        following += mine
    return tables


def _frequencies(case: dict) -> tuple[list[float], float]:
    """Angle per position of each pair, and the factor of the rotated lanes."""
    r, b, s, original = case["rotary"], case["base"], case["factor"], case["original"]
    scaling, (slow, fast) = case["scaling"], TURNS if case["scaling"] == "yarn" else (1.0, 4.0)
    if scaling == "ntk":
        b *= s ** (r / (r - 2))
    plain = [b ** (-2 * k / r) for k in range(r // 2)]
    if scaling == "linear":
        return [f / s for f in plain], 1.0
    if scaling == "yarn":
        pair = lambda turns: r * math.log(original / (2 * math.pi * turns)) / (2 * math.log(b))  # noqa: E731
        low, high = max(0, math.floor(pair(fast))), min(r - 1, math.ceil(pair(slow)))
        parts = [min(1.0, max(0.0, (k - low) / max(0.001, high - low))) for k in range(r // 2)]
        return [f * (1 - p) + f / s * p for f, p in zip(plain, parts)], 0.1 * math.log(s) + 1
    if scaling == "wavelength":
        turns = [original * f / (2 * math.pi) for f in plain]
        parts = [min(1.0, max(0.0, (t - slow) / (fast - slow))) for t in turns]
        return [f * p + f / s * (1 - p) for f, p in zip(plain, parts)], 1.0
    return plain, 1.0


def _rotate_inputs(case: dict, seed: int):
    g = _generator(seed)
    whole = _normal(g, case["rows"], case["heads"] * case["head_dim"] + case["gap"], type_=case["type"])
    return whole, _integers(g, 0, case["longest"], case["rows"])


def _append_inputs(case: dict, seed: int):
    g = _generator(seed)
    n, h, kv, d = case["sequences"] * case["new"], case["heads"], case["kv_heads"], case["head_dim"]
    q, k, v = _normal(g, n, h, d), _normal(g, n, kv, d), _normal(g, n, kv, d)
    biases = _normal(g, h, d, scale=0.1), _normal(g, kv, d, scale=0.1), _normal(g, kv, d, scale=0.1)
    return q, k, v, biases, _pool(g, case, sum(map(len, _tables(case))), 1)


def _attention_inputs(case: dict, seed: int):
    g = _generator(seed)
    pool = _pool(g, case, max(max(t) for t in _tables(case)) + 1, 1)
    return _normal(g, case["sequences"] * case["new"], case["heads"], case["head_dim"]), pool


def _logit_inputs(case: dict, seed: int) -> dict:
    g = _generator(seed)
    rows, v, s = case["sequences"] * case["new"], case["vocabulary"], case["sequences"]
    logits = _normal(g, rows, v, scale=3.0)
    if case["coarse"]:  # ties
        logits = (logits * 16).round() / 16
    # Conversations repeat themselves: half of a history comes from a few tokens.
    longest = max(1, case["longest"])
    history = torch.where(_integers(g, 0, 2, s, longest) == 0, _integers(g, 0, v, s, longest),
                          _integers(g, 0, max(1, v // 500), s, longest))
    density = torch.tensor([0.5, 0.02, 0.9], device="cuda")[torch.arange(case["masks"], device="cuda") % 3]
    words = -(-v // 32)
    bits = torch.rand(case["masks"], words, 32, device="cuda", generator=g) < density[:, None, None]
    masks = (bits.long() << torch.arange(32, device="cuda")).sum(-1)
    masks = torch.where(masks >= 2 ** 31, masks - 2 ** 32, masks).int()
    sets = min(4, s) if case["biases"] else 0
    bias_tokens = [torch.randperm(v, device="cuda", generator=g)[:case["biases"]].int() for _ in range(sets)]
    bias_values = [_normal(g, case["biases"], scale=4.0) for _ in range(sets)]
    return {"logits": logits, "history": history, "masks": masks, "tokens": _integers(g, 0, v, rows),
            "bias_tokens": bias_tokens, "bias_values": bias_values}


def _logit_rows(case: dict) -> list[dict]:
    """What each row's logits are changed by, but for its token."""
    rows, new = [], case["new"]
    for s in range(case["sequences"]):
        parents = _parents(case, s) if new > 1 else [-1]
        for j, p in enumerate(parents):
            r = len(rows)
            mask = r % (case["masks"] + 1) - 1 if case["masks"] > 1 else case["masks"] - 1
            rows.append({"repetition": (1.0, 1.1, 1.3)[s % 3], "presence": (0.5, 0.0)[s % 2], "frequency": (0.25, 0.0, 0.1)[s % 3],
                         "history": s, "parent": s * new + p if p >= 0 else -1, "drafted": new > 1,
                         "biases": s % 5 % min(4, case["sequences"]) if case["biases"] and s % 5 < 4 else -1, "mask": mask})
    return rows


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


def _plan(state, pool: torch.Tensor, layers: int, heads: int):
    """A cache over the pool with the case's sequences, the pages of _tables(case), and the plan of its trees."""
    import satori_amd as S
    from satori_amd.cache import CacheLayout, ElementType, PagedCache

    case = state.case
    layout = CacheLayout(layers=layers, kv_heads=case["kv_heads"], head_dim=case["head_dim"], page_tokens=PAGE,
                         type=ElementType[case["type"].upper()])
    cache = state.hold(PagedCache(S.default_context(), layout, pool.shape[0], pool.data_ptr()))
    contexts, shared = _contexts(case), _shared_pages(case) * PAGE
    first = cache.open()
    cache.extend([first], [shared])
    state.sequences = [first] + cache.fork(first, len(contexts) - 1)
    for s, c in zip(state.sequences, contexts):
        cache.extend([s], [c - shared + case["new"]])
    plan = state.hold(cache.plan(heads))
    trees = [_parents(case, s) if "tree" in case else range(-1, case["new"] - 1) for s in range(case["sequences"])]
    plan.set_tree(state.sequences, trees)
    return plan


def _rotation(state, positions: int):
    import satori_amd as S
    from satori_amd.rotary import Rotation, RotaryLayout, RotaryScaling, rotary_frequencies

    case = state.case
    turns = TURNS if case["scaling"] == "yarn" else (1.0, 4.0)
    frequencies, magnitude = rotary_frequencies(case["rotary"], case["base"], RotaryScaling[case["scaling"].upper()],
                                                case["factor"], case["original"], *turns)
    return state.hold(Rotation(S.default_context(), frequencies, magnitude, RotaryLayout[case["layout"].upper()], positions))


def _angles(case: dict, positions: int) -> tuple[torch.Tensor, torch.Tensor]:
    """Sines and cosines of every position's angles, made in 64 bits."""
    frequencies, magnitude = _frequencies(case)
    angle = torch.arange(positions, device="cuda", dtype=torch.float64)[:, None] * torch.tensor(frequencies, device="cuda", dtype=torch.float64)
    return (angle.sin() * magnitude).float(), (angle.cos() * magnitude).float()


def prepare(case: dict, seed: int):
    state = _State(case)
    kind = case["kind"]
    if kind == "rotate":
        state.x, state.positions = _rotate_inputs(case, seed)
        state.out = torch.zeros(case["rows"], case["heads"] * case["head_dim"], device="cuda", dtype=state.x.dtype)
        if own:
            state.rotation = _rotation(state, case["longest"])
        else:
            state.sines, state.cosines = _angles(case, case["longest"])
    elif kind == "logits":
        state.given = given = _logit_inputs(case, seed)
        rows, n = _logit_rows(case), case["sequences"] * case["new"]
        state.logits = given["logits"]
        state.lengths = torch.tensor(_history(case), device="cuda", dtype=torch.int32)
        state.out = torch.zeros_like(state.logits) if case["written"] else None
        state.best = torch.zeros(n, device="cuda", dtype=torch.int32)
        if own:
            import satori_amd as S
            from satori_amd.logits import LOGIT_ROW, LogitBatch, LogitRules

            state.rules = state.hold(LogitRules(S.default_context(), case["vocabulary"], len(given["bias_tokens"]), case["biases"]))
            for i, (tokens, values) in enumerate(zip(given["bias_tokens"], given["bias_values"])):
                state.rules.set_biases(i, tokens.cpu().numpy(), values.cpu().numpy())
            tokens = given["tokens"].tolist()
            table = np.array([(r["repetition"], r["presence"], r["frequency"], r["history"], r["parent"], t if r["drafted"] else -1,
                               r["biases"], r["mask"]) for r, t in zip(rows, tokens)], LOGIT_ROW)
            state.rows = torch.from_numpy(table.view(np.int32)).cuda()
            state.batch = LogitBatch(
                rows=state.rows.data_ptr(), count=n, logits=state.logits.data_ptr(), logits_stride=case["vocabulary"],
                output=state.out.data_ptr() if case["written"] else 0, output_stride=case["vocabulary"], best=state.best.data_ptr(),
                history=given["history"].data_ptr(), history_stride=given["history"].shape[1], histories=case["sequences"],
                lengths=state.lengths.data_ptr(), masks=given["masks"].data_ptr() if case["masks"] else 0,
                mask_count=case["masks"], mask_stride=given["masks"].shape[1])
        else:
            f = lambda name: torch.tensor([r[name] for r in rows], device="cuda")[:, None]  # noqa: E731
            state.repetition, state.presence, state.frequency = f("repetition"), f("presence"), f("frequency")
            state.owner, state.mask = f("history")[:, 0], f("mask")[:, 0]
            branches = [_branch([r["parent"] for r in rows], i) if r["drafted"] else [] for i, r in enumerate(rows)]
            most = max(map(len, branches))
            state.branches = torch.tensor([b + [n] * (most - len(b)) for b in branches], device="cuda", dtype=torch.long).view(n, most)
            biased = [(i, r["biases"]) for i, r in enumerate(rows) if r["biases"] >= 0]
            state.biased = torch.tensor([i for i, _ in biased], device="cuda", dtype=torch.long)
            state.bias_set = torch.tensor([b for _, b in biased], device="cuda", dtype=torch.long)
            if case["biases"]:
                state.bias_tokens, state.bias_values = torch.stack(given["bias_tokens"]).long(), torch.stack(given["bias_values"])
    else:
        contexts, n = _contexts(case), case["sequences"] * case["new"]
        if kind == "keep":
            state.pool = _pool(_generator(seed), case, sum(map(len, _tables(case))), case["layers"])
        elif kind == "append":
            state.q, state.k, state.v, state.biases, state.pool = _append_inputs(case, seed)
            state.out = torch.zeros_like(state.q)
        else:
            state.q, state.pool = _attention_inputs(case, seed)
            state.out = torch.zeros_like(state.q)
        kept = [_kept(case, s) for s in range(case["sequences"])] if kind == "keep" else None
        if own:
            state.kept = kept
            state.plan = _plan(state, state.pool, case["layers"] if kind == "keep" else 1, case.get("heads", case["kv_heads"]))
            if kind == "append":
                state.rotation = _rotation(state, max(contexts) + case["new"])
        else:
            tables = _tables(case)
            place = lambda s, p: tables[s][p // PAGE] * PAGE + p % PAGE  # noqa: E731
            if kind == "keep":
                state.sources = torch.tensor([place(s, contexts[s] + j) for s, rows in enumerate(kept) for j in rows], device="cuda")
                state.destinations = torch.tensor([place(s, contexts[s] + i) for s, rows in enumerate(kept) for i in range(len(rows))],
                                                  device="cuda")
            else:
                trees = [_parents(case, s) for s in range(case["sequences"])]
                state.places = torch.tensor([place(s, c + j) for s, c in enumerate(contexts) for j in range(case["new"])], device="cuda")
                state.positions = torch.tensor([c + d for c, t in zip(contexts, trees) for d in _depths(t)], device="cuda")
            if kind == "append":
                state.sines, state.cosines = _angles(case, max(contexts) + case["new"])
            if kind == "attention":
                most = max(map(len, tables))
                state.table = torch.tensor([t + [0] * (most - len(t)) for t in tables], device="cuda")
                seen = np.zeros((case["sequences"], case["new"], most * PAGE), bool)
                for s, (c, t) in enumerate(zip(contexts, trees)):
                    for j in range(case["new"]):
                        seen[s, j, :c] = True
                        seen[s, j, [c + a for a in _branch(t, j)]] = True
                state.seen = torch.from_numpy(seen).cuda()
    torch.cuda.synchronize()  # the package's calls run on another stream
    return state


# ---- one pass ----

def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(state):
    case = state.case
    if case["kind"] == "rotate":
        state.rotation.apply(state.x.data_ptr(), state.positions.data_ptr(), case["rows"], case["heads"], case["head_dim"],
                             out=state.out.data_ptr(), stride=state.x.shape[1], type=0 if case["type"] == "f32" else 1)
        return state.out
    if case["kind"] == "append":
        state.plan.append_rotated(0, state.q.data_ptr(), state.biases[0].data_ptr(), state.out.data_ptr(), state.k.data_ptr(),
                                  state.biases[1].data_ptr(), state.v.data_ptr(), state.biases[2].data_ptr(), state.rotation)
        return {"q": state.out, "pool": state.pool}
    if case["kind"] == "attention":
        state.plan.attention(0, state.q.data_ptr(), state.out.data_ptr())
        return state.out
    if case["kind"] == "keep":
        state.plan.keep(state.kept)
        return state.pool
    state.rules.apply(state.batch)
    return {"logits": state.out, "best": state.best} if case["written"] else state.best


def _turn(case: dict, x: torch.Tensor, sines: torch.Tensor, cosines: torch.Tensor) -> torch.Tensor:
    """[rows][heads][head_dim] by each row's angles."""
    r = case["rotary"]
    sn, cs = sines[:, None], cosines[:, None]
    if case["layout"] == "half":
        a, b = x[..., :r // 2], x[..., r // 2:r]
        return torch.cat([a * cs - b * sn, a * sn + b * cs, x[..., r:]], dim=-1)
    a, b = x[..., 0:r:2], x[..., 1:r:2]
    return torch.cat([torch.stack([a * cs - b * sn, a * sn + b * cs], dim=-1).flatten(-2), x[..., r:]], dim=-1)


def _run_plain(state):
    case = state.case
    if case["kind"] == "rotate":
        x = state.x[:, :case["heads"] * case["head_dim"]].float().view(case["rows"], case["heads"], case["head_dim"])
        at = state.positions.long()
        state.out.copy_(_turn(case, x, state.sines[at], state.cosines[at]).flatten(1))
        return state.out
    if case["kind"] == "append":
        sines, cosines = state.sines[state.positions], state.cosines[state.positions]
        state.out.copy_(_turn(case, state.q + state.biases[0], sines, cosines))
        pages, offsets = state.places // PAGE, state.places % PAGE
        _keys(state.pool, case)[pages, 0, :, offsets] = _turn(case, state.k + state.biases[1], sines, cosines).to(state.pool.dtype)
        _values(state.pool, case)[pages, 0, :, :, offsets] = (state.v + state.biases[2]).to(state.pool.dtype)
        return {"q": state.out, "pool": state.pool}
    if case["kind"] == "attention":
        return _attention_plain(state)
    if case["kind"] == "keep":
        keys, values = _keys(state.pool, case), _values(state.pool, case)
        to, of = state.destinations, state.sources
        moved = keys[of // PAGE, :, :, of % PAGE], values[of // PAGE, :, :, :, of % PAGE]
        keys[to // PAGE, :, :, to % PAGE], values[to // PAGE, :, :, :, to % PAGE] = moved
        return state.pool
    return _logits_plain(state)


def _attention_plain(state):
    case = state.case
    b, new, kv, d = case["sequences"], case["new"], case["kv_heads"], case["head_dim"]
    group = case["heads"] // kv
    tokens = state.table.shape[1] * PAGE
    k = _keys(state.pool, case)[state.table, 0].permute(0, 2, 1, 3, 4).reshape(b * kv, tokens, d).float()
    v = _values(state.pool, case)[state.table, 0].permute(0, 2, 1, 4, 3).reshape(b * kv, tokens, d).float()
    q = state.q.view(b, new, kv, group, d).permute(0, 2, 1, 3, 4).reshape(b * kv, new * group, d)
    scores = (torch.bmm(q, k.transpose(1, 2).contiguous()) / math.sqrt(d)).view(b, kv, new, group, tokens)
    scores = scores.masked_fill(~state.seen.view(b, 1, new, 1, tokens), -math.inf)
    p = (scores - scores.amax(-1, keepdim=True)).exp()
    p = (p / p.sum(-1, keepdim=True)).view(b * kv, new * group, tokens)
    out = torch.bmm(p, v).view(b, kv, new, group, d)
    state.out.copy_(out.permute(0, 2, 1, 3, 4).reshape(state.out.shape))
    return state.out


def _logits_plain(state):
    case, given = state.case, state.given
    n, v = state.logits.shape
    # What each row has had: its request's history (what lies behind its end counts as token v) and its branch.
    history = torch.where(torch.arange(given["history"].shape[1], device="cuda") < state.lengths[:, None], given["history"], v)
    tokens = torch.cat([given["tokens"], given["tokens"].new_full((1,), v)])
    counts = torch.zeros(case["sequences"], v + 1, device="cuda")
    counts.scatter_add_(1, history.long(), torch.ones_like(history, dtype=torch.float32))
    counts = counts[state.owner]
    branch = tokens[state.branches].long()
    counts = counts.scatter_add_(1, branch, torch.ones_like(branch, dtype=torch.float32))[:, :v]
    x = state.logits
    penalised = torch.where(x > 0, x / state.repetition, x * state.repetition) - (state.presence + state.frequency * counts)
    x = torch.where(counts > 0, penalised, x)
    if case["biases"]:
        x[state.biased[:, None], state.bias_tokens[state.bias_set]] += state.bias_values[state.bias_set]
    if case["masks"]:
        allowed = ((given["masks"][:, :, None] >> torch.arange(32, device="cuda", dtype=torch.int32)) & 1).flatten(1)[:, :v] != 0
        x = x.masked_fill(~allowed[state.mask] & (state.mask >= 0)[:, None], -math.inf)
    top = x.amax(1, keepdim=True)
    first = torch.where(x == top, torch.arange(v, device="cuda"), v).amin(1)
    state.best.copy_(torch.where(top[:, 0] > -math.inf, first, -1))
    if not case["written"]:
        return state.best
    state.out.copy_(x)
    return {"logits": state.out, "best": state.best}


# ---- the outputs in 64 bits ----

def _turned(case: dict, x: torch.Tensor, positions: list[int]) -> torch.Tensor:
    """[rows][heads][head_dim] in 64 bits: complex numbers turned by their row's position."""
    r = case["rotary"]
    frequencies, magnitude = _frequencies(case)
    angle = torch.tensor(positions, device="cuda", dtype=torch.float64)[:, None, None] * torch.tensor(frequencies, device="cuda", dtype=torch.float64)
    turn = torch.polar(torch.full_like(angle, magnitude), angle)
    out = x.clone()
    first, second = (slice(0, r // 2), slice(r // 2, r)) if case["layout"] == "half" else (slice(0, r, 2), slice(1, r, 2))
    z = torch.complex(x[..., first].contiguous(), x[..., second].contiguous()) * turn
    out[..., first], out[..., second] = z.real, z.imag
    return out


def exact(case: dict, seed: int):
    kind = case["kind"]
    if kind == "rotate":
        x, positions = _rotate_inputs(case, seed)
        x = x[:, :case["heads"] * case["head_dim"]].double().reshape(case["rows"], case["heads"], case["head_dim"])
        return _turned(case, x, positions.tolist()).flatten(1)
    if kind == "logits":
        return _logits_exact(case, seed)
    contexts, tables = _contexts(case), _tables(case)
    if kind == "keep":
        pool = _pool(_generator(seed), case, sum(map(len, tables)), case["layers"])
        before, after = pool.clone(), pool
        for s, (c, table) in enumerate(zip(contexts, tables)):
            for i, j in enumerate(_kept(case, s)):
                to, of = divmod(c + i, PAGE), divmod(c + j, PAGE)
                _keys(after, case)[table[to[0]], :, :, to[1]] = _keys(before, case)[table[of[0]], :, :, of[1]]
                _values(after, case)[table[to[0]], :, :, :, to[1]] = _values(before, case)[table[of[0]], :, :, :, of[1]]
        return after
    new = case["new"]
    trees = [_parents(case, s) for s in range(case["sequences"])]
    if kind == "append":
        q, k, v, (bq, bk, bv), pool = _append_inputs(case, seed)
        positions = [c + d for c, t in zip(contexts, trees) for d in _depths(t)]
        pool = pool.double()
        k, v = _turned(case, k.double() + bk.double(), positions), v.double() + bv.double()
        for s, (c, table) in enumerate(zip(contexts, tables)):
            for j in range(new):
                page, offset = divmod(c + j, PAGE)
                _keys(pool, case)[table[page], 0, :, offset] = k[s * new + j]
                _values(pool, case)[table[page], 0, :, :, offset] = v[s * new + j]
        return {"q": _turned(case, q.double() + bq.double(), positions), "pool": pool}
    q, pool = _attention_inputs(case, seed)
    q, kv, d = q.double(), case["kv_heads"], case["head_dim"]
    out = torch.zeros_like(q)
    keys, values = _keys(pool, case), _values(pool, case)
    for s, (c, table, tree) in enumerate(zip(contexts, tables, trees)):
        at = torch.tensor(table, device="cuda")
        hidden = torch.ones(new, new, dtype=torch.bool)
        for j in range(new):
            hidden[j, _branch(tree, j)] = False
        hidden = torch.cat([torch.zeros(new, c, dtype=torch.bool), hidden], dim=1).cuda()
        for h in range(kv):
            k = keys[at, 0, h].reshape(-1, d)[:c + new].double()
            v = values[at, 0, h].transpose(1, 2).reshape(-1, d)[:c + new].double()
            for head in range(h * (case["heads"] // kv), (h + 1) * (case["heads"] // kv)):
                scores = (q[s * new:(s + 1) * new, head] @ k.T * d ** -0.5).masked_fill(hidden, -math.inf)
                out[s * new:(s + 1) * new, head] = torch.softmax(scores, dim=-1) @ v
    return out


def _logits_exact(case: dict, seed: int):
    given = _logit_inputs(case, seed)
    rows, v, lengths = _logit_rows(case), case["vocabulary"], _history(case)
    x = given["logits"].double()
    shifts = torch.arange(32, device="cuda")
    for i, r in enumerate(rows):
        had = given["history"][r["history"], :lengths[r["history"]]]
        if r["drafted"]:
            had = torch.cat([had, given["tokens"][_branch([q["parent"] for q in rows], i)]])
        count = torch.bincount(had, minlength=v).double()
        # (the parameters as the call has them: 32-bit numbers)
        repetition, presence, frequency = (float(np.float32(r[name])) for name in ("repetition", "presence", "frequency"))
        factor = torch.where(x[i] > 0, 1 / repetition, repetition)
        x[i] = torch.where(count > 0, x[i] * factor - presence - frequency * count, x[i])
        if r["biases"] >= 0:
            x[i, given["bias_tokens"][r["biases"]].long()] += given["bias_values"][r["biases"]].double()
        if r["mask"] >= 0:
            bits = (given["masks"][r["mask"]].long()[:, None] >> shifts) & 1
            x[i, bits.flatten()[:v] == 0] = -math.inf
    best = torch.tensor([int((row == row.max()).nonzero()[0]) if row.max() > -math.inf else -1 for row in x], dtype=torch.int32, device="cuda")
    return {"logits": x, "best": best} if case["written"] else best
