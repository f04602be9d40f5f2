"""The operators for several sequences together, as a host that answers several requests uses them: a prompt in chunks, forks
of it, decode steps of the whole batch with an adapter per request over K-quantized projections, eagerly and as one
captured step that is replayed while the sequences grow. Every attention, cache row and adapted projection of every layer is
checked against 64 bits on the device's own inputs, and the replayed steps bit for bit against the eager ones."""
from __future__ import annotations

import numpy as np
import pytest

import satori_amd as S
from helpers import rng
from satori_amd.adapters import LowRankAdapters
from satori_amd.cache import CacheLayout, ElementType
from test_gpu_cache import E, NUMPY, Device, Pool, check_attention

pytestmark = pytest.mark.gpu

HIDDEN, HEADS, KV_HEADS, HEAD_DIM, FFN, LAYERS = 512, 8, 2, 64, 768, 2
Q, KV = HEADS * HEAD_DIM, KV_HEADS * HEAD_DIM
ROPE_BASE, EPSILON, MOST = 1e6, 1e-6, 80
SHAPES = {"q": (Q, HIDDEN), "k": (KV, HIDDEN), "v": (KV, HIDDEN), "o": (HIDDEN, Q), "gate": (FFN, HIDDEN),
          "up": (FFN, HIDDEN), "down": (HIDDEN, FFN)}


class Model:
    """Two layers with their weights, adapters of q and the buffers of a step of up to MOST rows."""

    def __init__(self, context, device):
        g = rng(2024)
        self.context, self.ops = context, S.DeviceOps(context)
        self.layers, self.owned = [], []
        zeros = lambda n: device(np.zeros((MOST, n), np.float32))  # noqa: E731
        self.x, self.normed, self.projected = zeros(HIDDEN), zeros(HIDDEN), zeros(HIDDEN)
        self.q, self.adapted, self.turned, self.attended = zeros(Q), zeros(Q), zeros(Q), zeros(Q)
        self.k, self.v = zeros(KV), zeros(KV)
        self.gate, self.up, self.activated = zeros(FFN), zeros(FFN), zeros(FFN)
        for _ in range(LAYERS):
            m = {}
            for name, (rows, columns) in SHAPES.items():
                w = (g.standard_normal((rows, columns)) * columns ** -0.5).astype(np.float32)
                payload = S.quantize_weights(w, rows, columns, S.BlockQuantization.Q4_K)
                m[name] = self.own(context.create(payload, S.QuantizedMatrixShape(rows, columns, S.BlockQuantization.Q4_K)))
            layer = {"m": m}
            layer["qkv"] = self.own(S.HipGroup(context, [m["q"], m["k"], m["v"]], [self.normed] * 3,
                                               [self.q, self.k, self.v], True))
            layer["gateup"] = self.own(S.HipGroup(context, [m["gate"], m["up"]], [self.normed] * 2, [self.gate, self.up],
                                                  True))
            for name, n in (("attn_norm", HIDDEN), ("ffn_norm", HIDDEN), ("q_bias", Q), ("k_bias", KV), ("v_bias", KV)):
                layer[name] = device((g.random(n) + 0.5 if "norm" in name else g.standard_normal(n) * 0.1).astype(np.float32))
            down = [(g.standard_normal((r, HIDDEN)) * HIDDEN ** -0.5).astype(np.float16) for r in (8, 16, 5)]
            up = [(g.standard_normal((Q, r)) * r ** -0.5).astype(np.float16) for r in (8, 16, 5)]
            scales = [2.0, 1.0, 0.5]
            layer["weights"] = list(zip(down, up, scales))
            layer["adapters"] = self.own(LowRankAdapters(
                context, Q, HIDDEN, [(device(a), device(b), a.shape[0], s) for a, b, s in layer["weights"]]))
            self.layers.append(layer)
        self.table = device(np.zeros(2000 * HEAD_DIM))
        self.ops.rope_table(2000, HEAD_DIM, ROPE_BASE, self.table)

    def own(self, thing):
        self.owned.append(thing)
        return thing

    def read(self, p, rows, width):
        return self.context.download(np.zeros((rows, width), np.float32), p)

    def step(self, plan, rows, selection, check=None):
        """One pass of `rows` rows from self.x, in place."""
        ops = self.ops
        for n, layer in enumerate(self.layers):
            ops.rms_norm(self.x, layer["attn_norm"], EPSILON, HIDDEN, self.normed, rows)
            layer["qkv"].execute_batch(rows)
            layer["adapters"].apply(selection, self.normed, self.q, self.adapted)
            plan.append(n, self.adapted, layer["q_bias"], self.turned, self.k, layer["k_bias"], self.v, layer["v_bias"],
                        ROPE_BASE, HEAD_DIM, self.table, 2000)
            plan.attention(n, self.turned, self.attended)
            if check:
                check(n, layer)
            layer["m"]["o"].execute_batch_device(self.attended, rows, self.projected)
            ops.add(self.x, self.projected, rows * HIDDEN, self.x)
            ops.rms_norm(self.x, layer["ffn_norm"], EPSILON, HIDDEN, self.normed, rows)
            layer["gateup"].execute_batch(rows)
            ops.swiglu(self.gate, self.up, rows * FFN, self.activated)
            layer["m"]["down"].execute_batch_device(self.activated, rows, self.projected)
            ops.add(self.x, self.projected, rows * HIDDEN, self.x)

    def dispose(self):
        while self.owned:
            self.owned.pop().dispose()


@pytest.fixture
def device(context):
    d = Device(context)
    yield d
    d.close()


@pytest.mark.parametrize("type_", [ElementType.F16, ElementType.F32])
def test_prompt_forks_and_decode_steps(context, device, type_):
    g = rng(7)
    model = Model(context, device)
    layout = CacheLayout(LAYERS, KV_HEADS, HEAD_DIM, 32, type_)
    pools = [Pool(context, device, layout, 60) for _ in range(2)]  # the second follows by replays
    plans = [p.cache.plan(HEADS) for p in pools]

    def checked(pool, sequences, new, selection):
        rows = sum(new)

        def check(n, layer):
            x, base, got = model.read(model.normed, rows, HIDDEN), model.read(model.q, rows, Q), model.read(model.adapted, rows, Q)
            for r, a in enumerate(selection):
                if a < 0:
                    assert np.array_equal(got[r], base[r])
                    continue
                down, up, scale = (np.asarray(w, np.float64) for w in layer["weights"][a])
                y = base[r] + scale * (up @ (down @ x[r].astype(np.float64)))
                most = scale * (np.abs(up) @ (np.abs(down) @ np.abs(x[r].astype(np.float64))))
                assert np.all(np.abs(got[r] - y) <= (HIDDEN + 24) * E * most + E * (np.abs(base[r]) + np.abs(y)))
            pool.download()
            values, bias, row = model.read(model.v, rows, KV), np.zeros(KV, np.float32), 0
            context.download(bias, layer["v_bias"])
            for s, count in zip(sequences, new):
                _, v = pool.of(s, n)
                if count:
                    want = (values[row:row + count] + bias).astype(NUMPY[type_]).astype(np.float64)
                    assert np.array_equal(v[-count:].reshape(count, KV), want), "the rows' values are in their pages"
                row += count
            check_attention(pool, sequences, new, HEADS, model.read(model.turned, rows, Q).reshape(rows, HEADS, HEAD_DIM),
                            model.read(model.attended, rows, Q).reshape(rows, HEADS, HEAD_DIM), n, f"layer {n}")
        return check

    def run(which, sequences, new, selection, x, check=True):
        pool, plan = pools[which], plans[which]
        pool.cache.extend(sequences, new)
        plan.set(sequences, new)
        context.upload(model.x, x)
        model.step(plan, sum(new), selection, checked(pool, sequences, new, selection) if check else None)
        return model.read(model.x, sum(new), HIDDEN)

    embed = lambda rows: g.standard_normal((rows, HIDDEN)).astype(np.float32)  # noqa: E731
    firsts = [p.cache.open() for p in pools]
    for chunk in (70, 61):  # a prompt of 131 tokens, none of its chunks on a page's border
        x = embed(chunk)
        results = [run(w, [firsts[w]], [chunk], [2] * chunk, x, check=w == 0) for w in range(2)]
        assert np.array_equal(*results)
    forks = [p.cache.fork(f, 3) for p, f in zip(pools, firsts)]
    assert forks[0] == forks[1]
    sequences = [firsts[0]] + forks[0]
    selection = [0, 1, -1, 2]
    # One eager step of each cache (also the first run of every workspace), then the second cache's steps are replays.
    x = embed(4)
    results = [run(w, sequences, [1] * 4, selection, x, check=w == 0) for w in range(2)]
    assert np.array_equal(*results)
    context.capture_begin()
    model.step(plans[1], 4, selection)
    step = context.capture_end()
    for turn in range(40):  # past the end of a page, twice
        x = embed(4)
        eager = run(0, sequences, [1] * 4, selection, x, check=turn in (0, 1, 27, 28, 29, 39))
        pools[1].cache.extend(sequences, [1] * 4)
        plans[1].set(sequences, [1] * 4)
        context.upload(model.x, x)
        step.execute()
        assert np.array_equal(model.read(model.x, 4, HIDDEN), eager), f"step {turn}"
        if turn == 20:  # a request ends, another takes its place from the prompt of a third; the pages close up
            for p in pools:
                p.cache.free([sequences[1]])
                p.cache.compact()
                assert p.cache.fork(sequences[2]) == [sequences[1]]
                p.cache.truncate(sequences[1], 131)
    step.dispose()
    for p in plans:
        p.dispose()
    model.dispose()
