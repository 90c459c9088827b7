"""Attention over the INT8 cache against the formula in 64 bits: single
tokens, prompts, trees of drafted tokens, padded batches, tiles' and blocks'
edges, key ranges shared by several workgroups.

Bound.  With a query row's largest magnitude a and codes of a key at most c
times its scale k: the query's two fp16 parts hold 22 bits of a
(|dq| <= 2^-22 a each), the fp32 sum of d products of codes and parts adds
(d + 4) 2^-24 sum |q k|, and the score's few further roundings (scales, log2 e,
the difference from the maximum, exp2) 8 |s| 2^-24, so a score is off by
  ds <= 2^-22 a sum_d |k| + ((d + 4) sum_d |q k| + 8 |s|) 2^-24     (natural units).
A weight is off by that much relatively, plus 2^-21 of its own for its fp16
parts and exp2, and the sums over n keys add n 2^-24 and the rescalings of
(n / 32) blocks 2^-23 each; both of numerator and denominator:
  |err| <= 2 (max ds + 2^-20 + n 2^-23) sum p |v| / sum p.
With 16-bit queries the weights of the numerator are rounded to fp16: 2^-11
sum p |v| / sum p more (half a step, 2^-12, doubled for the scale's own
rounding), and the output to its type: eps / 2 |o|, and half the smallest
subnormal of fp16 (2^-25)."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from test_hip_kv_q8 import Cache, dev, dev_typed, host_typed, narrow

pytestmark = pytest.mark.gpu

HALF_EPS = {0: 0.0, 4: 2.0 ** -11, 5: 2.0 ** -8}
SENTINEL = 7.0


def words_of(sees):
    """bool [batch, rows, rows] as uint64 words [batch, rows, ceil(rows / 64)]."""
    b, rows, _ = sees.shape
    w = -(-rows // 64)
    bits = np.zeros((b, rows, w * 64), np.uint8)
    bits[:, :, :rows] = sees
    return np.packbits(bits, axis=-1, bitorder="little").view(np.uint64)


def tree_of(batch, rows, seed):
    """Ancestors (and itself) of random trees' nodes."""
    r = np.random.default_rng(seed)
    sees = np.zeros((batch, rows, rows), bool)
    for b in range(batch):
        for t in range(rows):
            sees[b, t, t] = True
            if t and r.random() < 0.9:
                sees[b, t] |= sees[b, r.integers(max(0, t - 6), t)]
    return sees


def reference(cache, q, dtype, pos, counts, sees, scale):
    """(out [batch, rows, heads, d], bound, rows that are written)."""
    batch, hk, max_seq, d = cache.shape
    heads, rows = q.shape[1], q.shape[2]
    g = heads // hk
    out, bound = np.zeros((batch, rows, heads, d)), np.zeros((batch, rows, heads, d))
    written = np.zeros((batch, rows), bool)
    n = np.arange(max_seq)
    for b in range(batch):
        real = rows if counts is None else max(0, min(rows, int(counts[b])))
        written[b, :real] = True
        node = n - int(pos[b])
        for t in range(real):
            if sees is None:
                see = node <= t
            else:
                see = (node < 0) | (np.where((node >= 0) & (node < rows), sees[b, t][np.clip(node, 0, rows - 1)], False))
            see &= node < real
            if not see.any():
                continue
            for h in range(heads):
                kc = cache.host["k_codes"][b, h // g][see].astype(np.float64) * cache.host["k_scales"][b, h // g][see].astype(np.float64)[:, None]
                vc = cache.host["v_codes"][b, h // g][see].astype(np.float64) * cache.host["v_scales"][b, h // g][see].astype(np.float64)[:, None]
                x = q[b, h, t].astype(np.float64)
                with np.errstate(all="ignore"):
                    s = scale * (kc @ x)
                    ds = scale * (np.abs(x).max() * np.abs(kc).sum(1) * 2.0 ** -22 + (d + 4) * (np.abs(kc) @ np.abs(x)) * 2.0 ** -24) + 8 * np.abs(s) * 2.0 ** -24
                    p = np.exp(s - s.max())
                    p /= p.sum()
                    out[b, t, h] = p @ vc
                    size = p @ np.abs(vc)
                    bound[b, t, h] = 2 * (ds.max() + 2.0 ** -20 + see.sum() * 2.0 ** -23) * size
                    if dtype:
                        bound[b, t, h] += 2.0 ** -11 * size + HALF_EPS[dtype] * (np.abs(out[b, t, h]) + bound[b, t, h]) + 2.0 ** -25
    return out, bound, written


def run(hip, cache, q, dtype, pos, counts, sees, scale, ws=None, stream=None):
    batch, hk, max_seq, d = cache.shape
    heads, rows = q.shape[1], q.shape[2]
    dq = dev_typed(hip, q, dtype)
    do = dev_typed(hip, np.full((batch, rows, heads, d), SENTINEL), dtype)
    dp = dev(hip, np.asarray(pos, np.int32))
    dc = dev(hip, np.asarray(counts, np.int32)) if counts is not None else None
    dt = dev(hip, words_of(sees)) if sees is not None else None
    need = hip.attention_q8_workspace_bytes(batch, rows, heads, hk, d, max_seq)
    if ws is None:
        ws = dev(hip, np.zeros(max(need, 1), np.uint8))
    hip.attention_q8(cache.q8, dq.addr, do.addr, dtype, rows, heads, dp.addr, dc.addr if dc else None, dt.addr if dt else None,
                     scale, ws.addr, ws.nbytes, stream)
    if stream is not None:
        stream.synchronize()
    out = host_typed(do, (batch, rows, heads, d), dtype)
    if need:
        assert (ws.download(np.uint32, (1024,)) == 0).all(), "tickets left behind"
    return out


def check(hip, cache, q, dtype, pos, counts=None, sees=None, scale=0.0, **kw):
    got = run(hip, cache, q, dtype, pos, counts, sees, scale, **kw).astype(np.float64)
    ref, bound, written = reference(cache, q, dtype, pos, counts, sees, scale if scale > 0 else cache.shape[3] ** -0.5)
    assert (got[~written] == SENTINEL).all(), "a padding row was written"
    got, ref, bound = got[written], ref[written], bound[written]
    assert np.array_equal(np.isnan(got), np.isnan(ref))
    fine = ~np.isnan(ref)
    err = np.abs(got - ref)[fine]
    assert np.all(err <= bound[fine]), (err.max(), np.max(err / np.maximum(bound[fine], 1e-300)))
    return got


def queries(batch, heads, rows, d, dtype, seed):
    return narrow(np.random.default_rng(seed).standard_normal((batch, heads, rows, d)), dtype)


@pytest.mark.parametrize("heads,hk,pos,max_seq", [
    (1, 1, [0], 1), (4, 4, [31], 32), (32, 4, [32], 40), (16, 1, [255], 300), (17, 1, [256], 300), (40, 2, [511, 3, 100], 512),
    (8, 1, [0, 699, 63, 64], 700), (15, 5, [2500], 2600), (100, 1, [1000], 1001),
])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", [0, 4, 5])
def test_single_tokens(hip, heads, hk, pos, max_seq, d, dtype):
    print(f"case attention_q8 token h={heads}/{hk} pos={pos} d={d} dtype={dtype}", flush=True)
    cache = Cache(hip, len(pos), hk, max_seq, d, max_seq)
    check(hip, cache, queries(len(pos), heads, 1, d, dtype, 1), dtype, pos)


@pytest.mark.parametrize("heads,hk,rows,pos,max_seq", [
    (4, 1, 16, [100], 200), (4, 4, 2, [0, 31], 64), (8, 2, 9, [500, 33, 0], 520), (6, 2, 24, [1000], 1024), (3, 3, 65, [70], 140),
    (2, 1, 130, [5], 140), (32, 4, 7, [2000], 2048), (1, 1, 70, [1300], 1400),
])
@pytest.mark.parametrize("d,dtype", [(64, 0), (64, 4), (128, 0), (128, 5)])
def test_trees(hip, heads, hk, rows, pos, max_seq, d, dtype):
    print(f"case attention_q8 tree h={heads}/{hk} rows={rows} pos={pos} d={d} dtype={dtype}", flush=True)
    cache = Cache(hip, len(pos), hk, max_seq, d, rows)
    check(hip, cache, queries(len(pos), heads, rows, d, dtype, 2), dtype, pos, sees=tree_of(len(pos), rows, rows), scale=0.15)


@pytest.mark.parametrize("heads,hk,rows,pos,max_seq", [
    (2, 1, 17, [0], 17), (4, 2, 100, [0, 50], 150), (3, 1, 64, [33], 97), (8, 8, 130, [300], 500),
])
@pytest.mark.parametrize("d,dtype", [(64, 0), (64, 5), (128, 0), (128, 4)])
def test_prompts(hip, heads, hk, rows, pos, max_seq, d, dtype):
    print(f"case attention_q8 prompt h={heads}/{hk} rows={rows} pos={pos} d={d} dtype={dtype}", flush=True)
    cache = Cache(hip, len(pos), hk, max_seq, d, rows)
    check(hip, cache, queries(len(pos), heads, rows, d, dtype, 3), dtype, pos)


def test_a_chain_is_the_tree_of_a_chain(hip):
    cache = Cache(hip, 2, 2, 300, 64, 4)
    q = queries(2, 4, 20, 64, 0, 4)
    print("case attention_q8 chain", flush=True)
    a = run(hip, cache, q, 0, [100, 7], None, None, 0.0)
    b = run(hip, cache, q, 0, [100, 7], None, np.broadcast_to(np.tri(20, dtype=bool), (2, 20, 20)), 0.0)
    assert np.allclose(a, b, rtol=0, atol=4e-6)   # (a chain's tile may share its keys out differently)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", [0, 4])
def test_padding_empty_rows_and_positions_outside(hip, d, dtype):
    # counts below, at and past rows and negative; a position before row 0
    # (its nodes below row 0 do not exist), at max_seq and past it; tokens
    # whose words are zero, with and without cached tokens in front; words
    # with every bit set (bits past the count and the rows are ignored)
    rows, pos = 10, [0, 40, 100, -3, 95, 100, 2**31 - 5, -2**31, 12]
    counts = [10, 4, 0, 10, 10, 10, 10, 10, -7]
    cache = Cache(hip, len(pos), 2, 100, d, 5)
    sees = tree_of(len(pos), rows, 6)
    sees[0, 3] = sees[0, 9] = sees[1, 1] = False
    sees[1, 2] = sees[4, 0] = True
    print(f"case attention_q8 padding d={d} dtype={dtype}", flush=True)
    q = queries(len(pos), 6, rows, d, dtype, 5)
    got = check(hip, cache, q, dtype, pos, counts, sees)
    assert (got[3] == 0).all() and (got[9] == 0).all()   # sequence 0's tokens 3 and 9 see nothing
    check(hip, cache, q, dtype, pos, counts)
    check(hip, cache, q, dtype, pos)


def test_bits_past_the_rows_are_ignored(hip):
    cache = Cache(hip, 1, 1, 100, 64, 5)
    q = queries(1, 2, 10, 64, 0, 5)
    sees = tree_of(1, 10, 6)
    wide = np.ones((1, 10, 64), bool)
    wide[:, :, :10] = sees
    print("case attention_q8 bits past the rows", flush=True)
    a = run(hip, cache, q, 0, [50], None, sees, 0.0)
    dq, dp, do = dev(hip, q), dev(hip, np.array([50], np.int32)), dev(hip, np.zeros((1, 10, 2, 64), np.float32))
    dt = dev(hip, np.packbits(wide, axis=-1, bitorder="little").view(np.uint64))
    ws = dev(hip, np.zeros(1 << 20, np.uint8))
    hip.attention_q8(cache.q8, dq.addr, do.addr, 0, 10, 2, dp.addr, None, dt.addr, 0.0, ws.addr, ws.nbytes)
    assert np.array_equal(do.download(np.float32, (1, 10, 2, 64)), a)


@pytest.mark.parametrize("d,dtype", [(64, 0), (128, 5)])
def test_stale_rows_nan_and_extreme_scales(hip, d, dtype):
    # rows past the call's and masked nodes hold NaN scales (a failed or
    # unused write): nothing reaches the output; a NaN that is seen does;
    # value scales over 30 powers of ten
    rows, pos, max_seq = 12, [200, 64], 600
    cache = Cache(hip, 2, 2, max_seq, d, 8)
    sees = tree_of(2, rows, 9)
    sees[0, :, 5] = False   # node 5 is seen by nobody, not by itself either
    for kv in "kv":
        s = cache.host[kv + "_scales"]
        s[0, :, 212:], s[1, :, 76:] = np.nan, np.nan
        s[0, :, 205] = np.nan
        cache.dev[kv + "_scales"].upload(s)
    cache.host["v_scales"][0, 0, :200] *= np.float32(10.0) ** np.random.default_rng(1).integers(-15, 15, 200).astype(np.float32)
    cache.dev["v_scales"].upload(cache.host["v_scales"])
    q = queries(2, 4, rows, d, dtype, 9) * np.float32(0.25)
    print(f"case attention_q8 stale rows d={d} dtype={dtype}", flush=True)
    got = check(hip, cache, q, dtype, pos, None, sees)
    assert np.isfinite(got).all()
    for kv in "kv":
        s = cache.host[kv + "_scales"].copy()
        s[1, 1, 3] = np.nan
        cache.dev[kv + "_scales"].upload(s)
        old, cache.host[kv + "_scales"] = cache.host[kv + "_scales"], s
        got = check(hip, cache, q, dtype, pos, None, sees)
        assert np.isnan(got[rows:, 2:]).all() and np.isfinite(got[:rows]).all() and np.isfinite(got[rows:, :2]).all()
        cache.host[kv + "_scales"] = old
        cache.dev[kv + "_scales"].upload(old)


def test_queries_with_infinities_give_nan_in_their_own_rows(hip):
    cache = Cache(hip, 1, 1, 90, 64, 3)
    q = queries(1, 3, 8, 64, 0, 3)
    q[0, 1, 4, 7], q[0, 2, 0, 0] = np.inf, np.nan
    q[0, 0, 2] = 0.0          # a row of zeros: the values' mean
    q[0, 0, 3] *= 1e30        # one key takes it all
    q[0, 0, 5] *= 1e-30
    print("case attention_q8 special queries", flush=True)
    got = run(hip, cache, q, 0, [60], None, None, 0.0)
    ref, bound, _ = reference(cache, q, 0, [60], None, None, 64 ** -0.5)
    assert np.isnan(got[0, 4, 1]).all() and np.isnan(got[0, 0, 2]).all()
    ok = ~np.isnan(got)
    assert (~ok).sum() == 2 * 64
    rest = ok.copy()
    rest[0, 3, 0] = False
    assert np.all(np.abs(got - ref)[rest] <= bound[rest])
    # with scores of 1e30 apart the largest one's value, to a weight of one
    s = cache.host["k_codes"][0, 0, :64].astype(np.float64) @ q[0, 0, 3].astype(np.float64) * cache.host["k_scales"][0, 0, :64]
    top = int(np.argmax(s))
    v = cache.host["v_codes"][0, 0, top].astype(np.float64) * cache.host["v_scales"][0, 0, top]
    assert np.all(np.abs(got[0, 3, 0] - v) <= np.abs(v) * 2.0 ** -20)


@pytest.mark.parametrize("d,dtype", [(64, 0), (128, 5)])
def test_long_caches(hip, d, dtype):
    # the third sequence's codes start past 2^32 bytes; keys shared by as many
    # workgroups as there may be
    max_seq = 0x7fffffff // d
    n = 3 * max_seq
    big = [hip.DeviceBuffer(n * d), hip.DeviceBuffer(n * 4), hip.DeviceBuffer(n * d), hip.DeviceBuffer(n * 4)]
    rows, past, heads = 3, 30000, 4
    cache = Cache(hip, 3, 1, past + rows, d, 4)
    lib = hip.open_library()
    for k, buf in zip(("k_codes", "k_scales", "v_codes", "v_scales"), big):
        row = d if k.endswith("codes") else 4
        for b in range(3):
            hip.check(lib.vm_hip_memcpy_d2d(buf.addr + b * max_seq * row, cache.dev[k].addr + b * (past + rows) * row,
                                            (past + rows) * row, None))
    small, cache.q8 = cache.q8, hip.KvQ8(*[b.addr for b in big], 3, 1, max_seq, d)
    cache.shape = (3, 1, max_seq, d)
    q = queries(3, heads, rows, d, dtype, 4)
    pos = [past, 5, past - 5]
    print(f"case attention_q8 long d={d} dtype={dtype}", flush=True)
    got = run(hip, cache, q, dtype, pos, None, None, 0.0)
    cache.q8, cache.shape = small, (3, 1, past + rows, d)
    ref, bound, _ = reference(cache, q, dtype, pos, None, None, d ** -0.5)
    assert np.all(np.abs(got - ref) <= bound), np.max(np.abs(got - ref) / bound)


def test_two_streams_and_shared_workspace_sizes(hip):
    # workspaces of their own on two streams; one workspace for calls of
    # several shapes in turn
    caches = [Cache(hip, 1, 2, 3000, 64, i) for i in range(2)]
    qs = [queries(1, 8, 4, 64, 0, i) for i in range(2)]
    streams = [hip.Stream() for _ in range(2)]
    print("case attention_q8 two streams", flush=True)
    alone = [run(hip, c, q, 0, [2900], None, None, 0.0) for c, q in zip(caches, qs)]
    need = hip.attention_q8_workspace_bytes(1, 4, 8, 2, 64, 3000)
    sets = []
    for c, q, s in zip(caches, qs, streams):
        sets.append((c, dev(hip, q), dev(hip, np.zeros((1, 4, 8, 64), np.float32)), dev(hip, np.array([2900], np.int32)),
                     dev(hip, np.zeros(need, np.uint8)), s))
    hip.synchronize()   # the uploads are in place before other streams read them
    for _ in range(20):
        for c, q, o, p, w, s in sets:
            hip.attention_q8(c.q8, q.addr, o.addr, 0, 4, 8, p.addr, None, None, 0.0, w.addr, need, s)
    for (c, q, o, p, w, s), want in zip(sets, alone):
        s.synchronize()
        assert np.array_equal(o.download(np.float32, (1, 4, 8, 64)), want)
    ws = dev(hip, np.zeros(max(need, hip.attention_q8_workspace_bytes(1, 40, 8, 2, 64, 3000)), np.uint8))
    for rows in (4, 1, 40, 4, 9):
        check(hip, caches[0], queries(1, 8, rows, 64, 0, rows), 0, [2900], ws=ws)


def test_captured_and_replayed(hip):
    # positions and counts change between replays of one graph
    cache = Cache(hip, 2, 2, 2000, 64, 6)
    q = queries(2, 8, 5, 64, 0, 6)
    need = hip.attention_q8_workspace_bytes(2, 5, 8, 2, 64, 2000)
    stream = hip.Stream()
    dq, do, ws = dev(hip, q), dev(hip, np.zeros((2, 5, 8, 64), np.float32)), dev(hip, np.zeros(need, np.uint8))
    dp, dc = dev(hip, np.zeros(2, np.int32)), dev(hip, np.zeros(2, np.int32))
    graph = hip.Graph(stream)
    graph.begin()
    hip.attention_q8(cache.q8, dq.addr, do.addr, 0, 5, 8, dp.addr, dc.addr, None, 0.0, ws.addr, need, stream)
    graph.end()
    for pos, counts in (([0, 1990], [5, 5]), ([1500, 3], [2, 5]), ([700, 700], [0, 1])):
        do.upload(np.full((2, 5, 8, 64), SENTINEL, np.float32), stream.handle)
        dp.upload(np.array(pos, np.int32), stream.handle)
        dc.upload(np.array(counts, np.int32), stream.handle)
        print(f"case attention_q8 replay {pos} {counts}", flush=True)
        for _ in range(3):
            graph.launch()
        stream.synchronize()
        eager = run(hip, cache, q, 0, pos, counts, None, 0.0)
        assert np.array_equal(do.download(np.float32, (2, 5, 8, 64)), eager)
