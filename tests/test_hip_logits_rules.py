"""Penalties, biases, grammar masks and the greedy token on the GPU against
numpy's fp32, step by step, bit for bit."""
from __future__ import annotations

import numpy as np
import pytest

from test_hip_attention_q8 import tree_of, words_of
from test_hip_kv_q8 import assert_equal, dev, dev_typed, host_typed, narrow

pytestmark = pytest.mark.gpu

ALL = ("history", "repetition", "frequency", "presence", "bias", "allowed", "drafted", "tree")


def inputs(seqs, rows, vocab, hist, nb, dtype, seed):
    r = np.random.default_rng(seed)
    a = dict(logits=narrow(r.standard_normal((seqs, rows, vocab)) * 3, dtype))
    a["history"] = r.integers(0, max(1, min(vocab, 40)), (seqs, hist)).astype(np.int32)
    if hist > 4:
        a["history"][:, 3] = -1
        a["history"][:, 4] = vocab
    a["history_lengths"] = r.integers(0, hist + 1, seqs).astype(np.int32)
    a["history_lengths"][0] = hist + 5   # clamped
    a["repetition"] = r.uniform(0.8, 1.6, seqs).astype(np.float32)
    a["frequency"] = r.uniform(-0.2, 0.5, seqs).astype(np.float32)
    a["presence"] = r.uniform(0, 0.5, seqs).astype(np.float32)
    a["bias_tokens"] = r.integers(0, max(1, vocab // 2), (seqs, nb)).astype(np.int32)
    if nb > 3:
        a["bias_tokens"][:, 1] = a["bias_tokens"][:, 3]   # the same token twice
        a["bias_tokens"][:, 2] = -7
    a["bias_values"] = (r.standard_normal((seqs, nb)) * 4).astype(np.float32)
    a["bias_lengths"] = r.integers(0, nb + 1, seqs).astype(np.int32)
    a["bias_lengths"][0] = nb + 1
    may = r.random((seqs, rows, vocab)) < 0.3
    may[0, 0] = False
    a["may"] = may
    words = -(-vocab // 32)
    bits = np.ones((seqs, rows, words * 32), np.uint8)   # bits past vocab mean nothing
    bits[..., :vocab] = may
    a["allowed"] = np.packbits(bits, axis=-1, bitorder="little").view(np.uint32)
    a["drafted"] = r.integers(0, vocab, (seqs, rows)).astype(np.int32)
    a["sees"] = tree_of(seqs, rows, seed)
    a["tree"] = words_of(a["sees"])
    return a


def expect(a, use, dtype):
    x = a["logits"].astype(np.float32).copy()
    seqs, rows, vocab = x.shape
    tokens = np.full((seqs, rows), -1, np.int32)
    f = np.float32
    for s in range(seqs):
        seen = np.zeros(vocab, np.int64)
        if "history" in use:
            h = a["history"][s, :max(0, min(a["history"].shape[1], a["history_lengths"][s]))]
            seen += np.bincount(h[(h >= 0) & (h < vocab)], minlength=vocab)
        bias = np.zeros(vocab, f)
        listed = np.zeros(vocab, bool)
        if "bias" in use:
            for e in range(max(0, min(a["bias_tokens"].shape[1], a["bias_lengths"][s]))):
                if 0 <= a["bias_tokens"][s, e] < vocab:
                    bias[a["bias_tokens"][s, e]] = a["bias_values"][s, e]
                    listed[a["bias_tokens"][s, e]] = True
        for t in range(rows):
            n = seen.copy()
            if "drafted" in use:
                for j in range(rows):
                    if (a["sees"][s, t, j] if "tree" in use else j <= t) and 0 <= a["drafted"][s, j] < vocab:
                        n[a["drafted"][s, j]] += 1
            y, hit = x[s, t], n > 0
            with np.errstate(all="ignore"):
                if "repetition" in use:
                    y = np.where(hit, np.where(y > 0, y / a["repetition"][s], y * a["repetition"][s]), y).astype(f)
                if "frequency" in use:
                    y = np.where(hit, y - n.astype(f) * a["frequency"][s], y).astype(f)
                if "presence" in use:
                    y = np.where(hit, y - a["presence"][s], y).astype(f)
                y = np.where(listed, y + bias, y).astype(f)
            if "allowed" in use:
                y = np.where(a["may"][s, t], y, f(-np.inf))
            x[s, t] = y
            z = np.where(np.isnan(y), -np.inf, y)
            if z.max() > -np.inf:
                tokens[s, t] = int(np.argmax(z))
    return narrow(x, dtype), tokens


class Rules:
    def __init__(self, hip, a, use):
        self.bufs = {}
        fields = {}
        for name in use:
            for key in {"history": ("history", "history_lengths"), "bias": ("bias_tokens", "bias_values", "bias_lengths")}.get(name, (name,)):
                self.bufs[key] = dev(hip, a[key] if a[key].size else np.zeros(1, a[key].dtype))
                fields[key] = self.bufs[key].addr
        if "history" in use:
            fields["history_stride"] = a["history"].shape[1]
        if "bias" in use:
            fields["bias_stride"] = a["bias_tokens"].shape[1]
        self.rules = hip.LogitsRules(**fields)


def run(hip, a, use, dtype, counts=None, in_place=False, ws=None, stream=None):
    seqs, rows, vocab = a["logits"].shape
    r = Rules(hip, a, use)
    x = dev_typed(hip, a["logits"], dtype)
    out = x if in_place else dev_typed(hip, np.full(a["logits"].shape, 7.0), dtype)
    tokens = dev(hip, np.full((seqs, rows), 77, np.int32))
    dc = dev(hip, np.asarray(counts, np.int32)) if counts is not None else None
    ws = dev(hip, np.zeros(hip.logits_rules_workspace_bytes(seqs, rows, vocab), np.uint8)) if ws is None else ws
    hip.logits_rules(r.rules, x.addr, out.addr, dtype, tokens.addr, seqs, rows, vocab, dc.addr if dc else None, ws.addr, ws.nbytes, stream)
    if stream is not None:
        stream.synchronize()
    assert (ws.download(np.uint8, (ws.nbytes,)) == 0).all(), "the workspace is not zero again"
    return host_typed(out, a["logits"].shape, dtype), tokens.download(np.int32, (seqs, rows))


def check(hip, a, use, dtype, **kw):
    got, tokens = run(hip, a, use, dtype, **kw)
    want, wt = expect(a, use, dtype)
    assert_equal(got, want)
    assert_equal(tokens, wt)


@pytest.mark.parametrize("seqs,rows,vocab,hist,nb", [
    (1, 1, 1, 1, 1), (1, 1, 32000, 700, 16), (2, 3, 1023, 50, 5), (1, 2, 1024, 0, 0), (3, 1, 1025, 300, 9), (2, 70, 333, 2000, 400),
    (4, 16, 128256, 999, 30), (130, 4, 4097, 64, 4), (1, 1, 2, 6, 4),
])
@pytest.mark.parametrize("dtype", [0, 4, 5])
def test_all_rules(hip, seqs, rows, vocab, hist, nb, dtype):
    print(f"case logits s={seqs} rows={rows} v={vocab} dtype={dtype}", flush=True)
    check(hip, inputs(seqs, rows, vocab, hist, nb, dtype, vocab), ALL, dtype)


@pytest.mark.parametrize("use", [(), ("history",), ("history", "repetition"), ("history", "frequency"), ("history", "presence"), ("bias",),
                                 ("allowed",), ("drafted", "repetition", "presence"), ("drafted", "tree", "frequency"),
                                 ("history", "repetition", "frequency", "presence", "bias"), ("repetition", "frequency")], ids="+".join)
def test_rules_left_out(hip, use):
    print(f"case logits rules {use}", flush=True)
    check(hip, inputs(3, 9, 5000, 100, 20, 0, 1), use, 0)


def test_in_place_outputs_left_out_and_ties(hip):
    a = inputs(2, 4, 9000, 100, 20, 0, 2)
    a["logits"] = np.round(a["logits"])   # many equal largest values
    check(hip, a, ("allowed",), 0)
    check(hip, a, (), 0)
    check(hip, a, ALL, 0, in_place=True)
    want, wt = expect(a, ALL, 0)
    r = Rules(hip, a, ALL)
    x, out, tokens = dev(hip, a["logits"]), dev(hip, np.zeros_like(a["logits"])), dev(hip, np.zeros((2, 4), np.int32))
    ws = dev(hip, np.zeros(hip.logits_rules_workspace_bytes(2, 4, 9000), np.uint8))
    hip.logits_rules(r.rules, x.addr, out.addr, 0, None, 2, 4, 9000, None, None, 0)
    assert np.array_equal(out.download(np.float32, want.shape), want)
    hip.logits_rules(r.rules, x.addr, None, 0, tokens.addr, 2, 4, 9000, None, ws.addr, ws.nbytes)
    assert np.array_equal(tokens.download(np.int32, (2, 4)), wt)
    assert np.array_equal(x.download(np.float32, want.shape), a["logits"])


@pytest.mark.parametrize("dtype", [0, 4])
def test_special_values(hip, dtype):
    # infinities and NaN in logits and biases, under the mask and outside it;
    # rows without any token left; a repetition of 0
    a = inputs(3, 3, 3000, 200, 12, dtype, 3)
    a["logits"][0, 1, 5:9] = [np.inf, -np.inf, np.nan, np.inf]
    a["logits"][1, 0] = np.nan
    a["logits"][1, 1] = -np.inf
    a["logits"][1, 2, 100:] = np.nan
    a["bias_values"][0, 0], a["bias_values"][0, 5] = np.inf, -np.inf
    a["repetition"][2] = 0.0
    print(f"case logits specials dtype={dtype}", flush=True)
    check(hip, a, ALL, dtype)
    check(hip, a, ("history", "repetition", "bias"), dtype)


def test_padding(hip):
    a = inputs(5, 6, 2500, 100, 8, 0, 4)
    counts = [6, 0, -3, 2, 99]
    print("case logits padding", flush=True)
    got, tokens = run(hip, a, ALL, 0, counts=counts)
    want, wt = expect(a, ALL, 0)
    for s, c in enumerate(counts):
        c = max(0, min(6, c))
        assert np.array_equal(got[s, :c], want[s, :c]) and np.array_equal(tokens[s, :c], wt[s, :c])
        assert (got[s, c:] == 7.0).all() and (tokens[s, c:] == 77).all()


def test_one_workspace_for_several_shapes_and_replays(hip):
    shapes = [(1, 1, 32000), (2, 5, 3000), (600, 1, 5000), (1, 1, 32000)]
    ws = dev(hip, np.zeros(max(hip.logits_rules_workspace_bytes(*s) for s in shapes), np.uint8))
    for s, r, v in shapes:
        print(f"case logits shared workspace {s} {r} {v}", flush=True)
        check(hip, inputs(s, r, v, 30, 4, 0, s), ALL, 0, ws=ws)
    stream = hip.Stream()
    a = inputs(2, 2, 20000, 60, 6, 0, 9)
    r = Rules(hip, a, ALL)
    x, out, tokens = dev(hip, a["logits"]), dev(hip, np.zeros_like(a["logits"])), dev(hip, np.zeros((2, 2), np.int32))
    graph = hip.Graph(stream)
    graph.begin()
    hip.logits_rules(r.rules, x.addr, out.addr, 0, tokens.addr, 2, 2, 20000, None, ws.addr, ws.nbytes, stream)
    graph.end()
    for n in (60, 0, 31):
        a["history_lengths"][:] = n
        r.bufs["history_lengths"].upload(a["history_lengths"], stream.handle)
        for _ in range(3):
            graph.launch()
        stream.synchronize()
        want, wt = expect(a, ALL, 0)
        assert np.array_equal(out.download(np.float32, want.shape), want)
        assert np.array_equal(tokens.download(np.int32, (2, 2)), wt)


def test_two_streams(hip):
    sets = []
    for i in range(2):
        a = inputs(2, 3, 30000, 50, 6, 0, 20 + i)
        sets.append((a, Rules(hip, a, ALL), dev(hip, a["logits"]), dev(hip, np.zeros_like(a["logits"])), dev(hip, np.zeros((2, 3), np.int32)),
                     dev(hip, np.zeros(hip.logits_rules_workspace_bytes(2, 3, 30000), np.uint8)), hip.Stream()))
    hip.synchronize()
    print("case logits two streams", flush=True)
    for _ in range(20):
        for a, r, x, out, tokens, ws, s in sets:
            hip.logits_rules(r.rules, x.addr, out.addr, 0, tokens.addr, 2, 3, 30000, None, ws.addr, ws.nbytes, s)
    for a, r, x, out, tokens, ws, s in sets:
        s.synchronize()
        want, wt = expect(a, ALL, 0)
        assert_equal(out.download(np.float32, want.shape), want)
        assert_equal(tokens.download(np.int32, (2, 3)), wt)


def test_long_histories(hip):
    # histories longer than a workgroup holds in registers, for
    # several chunks of the vocabulary and rows
    print("case logits long histories", flush=True)
    a = inputs(2, 5, 5000, 13001, 1500, 0, 30)
    a["history_lengths"][:] = [13001, 9000]
    check(hip, a, ALL, 0)
    a = inputs(1, 1, 2000000, 9000, 3, 5, 31)
    check(hip, a, ALL, 5)
