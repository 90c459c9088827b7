"""One layer's verification step of drafted tokens as a decoder runs it: INT8
projections, INT8 cache, attention over the tree, INT8 output projection and
vocabulary, rules and greedy tokens, the accepted path kept, and the next
token decoded on what is left, captured in a graph where positions change.
Every operator's output is checked against its formula on the very values
that the GPU handed it (the operators' own tests say how near)."""
from __future__ import annotations

import numpy as np
import pytest

import test_hip_attention_q8 as A
import test_hip_logits_rules as R
import test_hip_qmm_a8 as Q
from test_hip_kv_q8 import Cache, assert_equal, dev, expect_append, same

pytestmark = pytest.mark.gpu

HEADS, HK, D, HIDDEN, VOCAB, MAX_SEQ = 8, 2, 64, 512, 3001, 700
WIDTH = (HEADS + 2 * HK) * D


class Layer:
    """The layer's weights, its buffers for `rows` tokens of `seqs` sequences, and its launches."""

    def __init__(self, hip, seqs, rows, cache, tree, rules):
        self.hip, self.seqs, self.rows, self.cache, self.n = hip, seqs, rows, cache, seqs * rows
        self.weights = {}
        for name, (k, n) in {"qkv": (HIDDEN, WIDTH), "o": (HEADS * D, HIDDEN), "lm": (HIDDEN, VOCAB)}.items():
            codes, scale = Q.weights(k, n, n)
            scale *= np.float32(0.05)
            packed, dcodes = hip.DeviceBuffer(hip.a8_weights_bytes(k, n)), dev(hip, codes)
            hip.a8_pack(dcodes.addr, k, n, packed.addr)
            hip.synchronize()
            ws = dev(hip, np.zeros(max(1, hip.qmm_a8_workspace_bytes(self.n, k, n)), np.uint8))
            self.weights[name] = (codes, scale, packed, dev(hip, scale), ws, k, n)
        angle = np.arange(MAX_SEQ)[:, None] * 10000.0 ** (-np.arange(D // 2) / (D // 2))[None, :]
        self.cos, self.sin = np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)
        f = lambda *s: dev(hip, np.zeros(s, np.float32))  # noqa: E731
        self.x, self.qkv, self.q = f(self.n, HIDDEN), f(self.n, WIDTH), f(seqs, HEADS, rows, D)
        self.ctx, self.h, self.logits, self.ruled = f(self.n, HEADS * D), f(self.n, HIDDEN), f(self.n, VOCAB), f(self.n, VOCAB)
        self.tokens = dev(hip, np.zeros((seqs, rows), np.int32))
        self.pos, self.counts = dev(hip, np.zeros(seqs, np.int32)), dev(hip, np.zeros(seqs, np.int32))
        self.depths = dev(hip, np.zeros((seqs, rows), np.int32))
        self.dcos, self.dsin = dev(hip, self.cos), dev(hip, self.sin)
        self.staged = hip.DeviceBuffer(hip.a8_stage_bytes(self.n, HIDDEN))
        self.tree = dev(hip, A.words_of(tree)) if tree is not None else None
        self.attention_ws = dev(hip, np.zeros(max(1, hip.attention_q8_workspace_bytes(seqs, rows, HEADS, HK, D, MAX_SEQ)), np.uint8))
        self.logits_ws = dev(hip, np.zeros(hip.logits_rules_workspace_bytes(seqs, rows, VOCAB), np.uint8))
        self.rules = rules

    def product(self, name, a, c, stream):
        _, _, packed, scale, ws, k, n = self.weights[name]
        self.hip.a8_stage(a.addr, 0, self.n, k, self.staged.addr, stream)
        self.hip.qmm_a8(self.staged.addr, packed.addr, scale.addr, c.addr, 0, self.n, k, n, ws.addr, ws.nbytes, stream)

    def launch(self, stream):
        hip, c = self.hip, self.cache.q8
        self.product("qkv", self.x, self.qkv, stream)
        hip.kv_q8_append(c, self.qkv.addr, 0, self.rows, HEADS, self.dcos.addr, self.dsin.addr, self.pos.addr, self.counts.addr,
                         self.depths.addr, self.q.addr, stream)
        hip.attention_q8(c, self.q.addr, self.ctx.addr, 0, self.rows, HEADS, self.pos.addr, self.counts.addr,
                         self.tree.addr if self.tree else None, 0.0, self.attention_ws.addr, self.attention_ws.nbytes, stream)
        self.product("o", self.ctx, self.h, stream)
        self.product("lm", self.h, self.logits, stream)
        hip.logits_rules(self.rules, self.logits.addr, self.ruled.addr, 0, self.tokens.addr, self.seqs, self.rows, VOCAB,
                         self.counts.addr, self.logits_ws.addr, self.logits_ws.nbytes, stream)

    def upload(self, x, pos, counts, depths, stream):
        for buf, a in ((self.x, x), (self.pos, np.asarray(pos, np.int32)), (self.counts, np.asarray(counts, np.int32)),
                       (self.depths, np.asarray(depths, np.int32))):
            buf.upload(a, stream.handle)

    def check(self, x, pos, counts, depths, sees, rules_input, use):
        """Every stage against its formula; the cache's host copy is brought up to date."""
        s, r = self.seqs, self.rows
        get = lambda b, *shape: b.download(np.float32, shape)  # noqa: E731
        qkv = get(self.qkv, self.n, WIDTH)
        assert_equal(qkv, Q.expect(x, *self.weights["qkv"][:2], 0))
        want, q = expect_append(self.cache, qkv.reshape(s, r, WIDTH), 0, HEADS, self.cos, self.sin, pos, counts, depths,
                                get(self.q, s, HEADS, r, D))
        got = self.cache.download()
        same(got, want)
        assert_equal(get(self.q, s, HEADS, r, D), q)
        self.cache.host = got
        ref, bound, written = A.reference(self.cache, q, 0, pos, counts, sees, D ** -0.5)
        ctx = get(self.ctx, s, r, HEADS, D)
        assert np.all(np.abs(ctx - ref)[written] <= bound[written])
        real = written.reshape(-1)
        h = get(self.h, self.n, HIDDEN)
        assert_equal(h[real], Q.expect(ctx.reshape(self.n, -1), *self.weights["o"][:2], 0)[real])
        logits = get(self.logits, self.n, VOCAB)
        assert_equal(logits[real], Q.expect(h, *self.weights["lm"][:2], 0)[real])
        want, tokens = R.expect(dict(rules_input, logits=logits.reshape(s, r, VOCAB), sees=sees), use, 0)
        assert_equal(get(self.ruled, s, r, VOCAB)[written], want[written])
        assert_equal(self.tokens.download(np.int32, (s, r))[written], tokens[written])
        return qkv.reshape(s, r, WIDTH)


def test_tree_step_keep_and_next_token(hip):
    seqs, rows = 2, 14
    r = np.random.default_rng(3)
    embed = r.standard_normal((VOCAB, HIDDEN)).astype(np.float32)
    cache = Cache(hip, seqs, HK, MAX_SEQ, D, 1)
    sees = A.tree_of(seqs, rows, 4)
    sees[:, :, 0] = True   # one root
    depths = sees.sum(2) - 1
    use = ("history", "repetition", "frequency", "presence", "bias", "allowed", "drafted", "tree")
    rin = R.inputs(seqs, rows, VOCAB, 60, 6, 0, 5)
    rin["tree"] = A.words_of(sees)
    rules = R.Rules(hip, rin, use)
    layer = Layer(hip, seqs, rows, cache, sees, rules.rules)
    stream = hip.Stream()
    graph = hip.Graph(stream)
    graph.begin()
    layer.launch(stream)
    graph.end()
    pos = np.array([500, 33], np.int32)
    for counts in ([14, 14], [9, 0], [14, 11]):
        drafted = r.integers(0, VOCAB, (seqs, rows)).astype(np.int32)
        rin["drafted"] = drafted
        rules.bufs["drafted"].upload(drafted, stream.handle)
        x = embed[drafted].reshape(seqs * rows, HIDDEN)
        layer.upload(x, pos, counts, depths, stream)
        print(f"case verify step counts={counts}", flush=True)
        graph.launch()
        stream.synchronize()
        qkv = layer.check(x, pos, counts, depths, sees, rin, use)

    # the longest path of each tree is accepted: its rows move together, and
    # are what decoding its tokens one by one writes
    kept = np.zeros((seqs, rows), np.int32)
    n = np.zeros(seqs, np.int32)
    for s in range(seqs):
        path = np.flatnonzero(sees[s, int(np.argmax(depths[s, :11]))])
        kept[s, :len(path)], n[s] = path, len(path)
    bufs = [dev(hip, a) for a in (pos, kept, n)]
    hip.kv_q8_keep(cache.q8, *[b.addr for b in bufs], rows, stream)
    stream.synchronize()
    got = cache.download()
    single = Cache(hip, seqs, HK, MAX_SEQ, D, 1)
    single.host = {k: v.copy() for k, v in cache.host.items()}
    for i in range(int(n.max())):
        one = np.stack([qkv[s, kept[s, i]] for s in range(seqs)])[:, None]
        single.host, _ = expect_append(single, one, 0, HEADS, layer.cos, layer.sin, pos + i, (i < n).astype(int), None,
                                       np.zeros((seqs, HEADS, 1, D), np.float32))
    for s in range(seqs):
        for k in got:
            assert np.array_equal(got[k][s, :, :pos[s] + n[s]], single.host[k][s, :, :pos[s] + n[s]]), k

    # the next token, decoded alone behind the kept path
    cache.host = got
    rin1 = R.inputs(seqs, 1, VOCAB, 60, 6, 0, 6)
    use1 = ("history", "repetition", "presence")
    rules1 = R.Rules(hip, rin1, use1)
    step = Layer(hip, seqs, 1, cache, None, rules1.rules)
    x = embed[r.integers(0, VOCAB, seqs)]
    step.upload(x, pos + n, [1, 1], np.zeros((seqs, 1)), stream)
    print("case verify step, the next token", flush=True)
    step.launch(stream)
    stream.synchronize()
    step.check(x, pos + n, [1, 1], np.zeros((seqs, 1), int), None, rin1, use1)
