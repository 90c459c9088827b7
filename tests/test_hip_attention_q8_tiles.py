"""Attention over the INT8 cache with several row tiles a wave (32 or 64 query
rows of a KV head a workgroup): what prompts and large trees run, with keys
shared by several workgroups and without.  The launch plan is written down
here a second time, so that a case cannot change its kernel unnoticed.

Bound as in test_hip_attention_q8.py."""
from __future__ import annotations

import numpy as np
import pytest

from test_hip_attention_q8 import HALF_EPS, SENTINEL, queries, tree_of, words_of
from test_hip_kv_q8 import Cache, dev, dev_typed, host_typed

pytestmark = pytest.mark.gpu

TYPES = [(64, 0), (64, 4), (64, 5), (128, 0), (128, 4), (128, 5)]
TICKETS = 512 * 16   # words


def plan(batch, rows, heads, hk, d, max_seq, dtype):
    """(16-row tiles of a wave, workgroups that share a tile's keys, workspace bytes)."""
    r, most = rows * (heads // hk), min(-(-max_seq // 256), 64)
    rt = 4 if d == 64 and dtype else 2
    while rt > 1 and (r <= 8 * rt or batch * hk * -(-r // (16 * rt)) * most < 512):
        rt //= 2
    units = batch * hk * -(-r // (16 * rt))
    splits = max(1, min(512 // units if units < 512 else 1, most))
    return rt, splits, TICKETS * 4 + units * splits * 16 * rt * (d + 2) * 4 if splits > 1 else 0


def reference(cache, q, dtype, pos, counts, sees, scale):
    """(out [batch, rows, heads, d], bound, rows that are written), in 64 bits."""
    batch, hk, max_seq, d = cache.shape
    heads, rows = q.shape[1], q.shape[2]
    g = heads // hk
    out, bound = np.zeros((batch, rows, heads, d)), np.zeros((batch, rows, heads, d))
    written = np.zeros((batch, rows), bool)
    for b in range(batch):
        real = rows if counts is None else max(0, min(rows, counts[b]))
        written[b, :real] = True
        n = min(pos[b] + real, max_seq)
        see = np.ones((rows, n), bool)
        see[:, pos[b]:] = (np.tri(rows, dtype=bool) if sees is None else sees[b])[:, :n - pos[b]]
        for h in range(heads):
            kc, vc = (cache.host[x + "_codes"][b, h // g, :n].astype(np.float64) for x in "kv")
            sk, sv = (cache.host[x + "_scales"][b, h // g, :n].astype(np.float64) for x in "kv")
            x, k = q[b, h].astype(np.float64), kc * np.where(np.isnan(sk), 0, sk)[:, None]
            s = scale * (x @ k.T)
            ds = scale * (np.abs(x).max(1)[:, None] * np.abs(k).sum(1) * 2.0 ** -22 + (d + 4) * (np.abs(x) @ np.abs(k).T) * 2.0 ** -24) + 8 * np.abs(s) * 2.0 ** -24
            s, ds = np.where(see, s, -np.inf), np.where(see, ds, 0)
            some = see.any(1)
            p = np.exp(s - np.where(some, s.max(1), 0)[:, None])
            w = np.where(see, p / np.where(some, p.sum(1), 1)[:, None] * np.where(np.isnan(sv), 0, sv), 0)
            o, size = w @ vc, w @ np.abs(vc)
            e = 2 * (ds.max(1) + 2.0 ** -20 + see.sum(1) * 2.0 ** -23)[:, None] * size
            if dtype:
                e += 2.0 ** -11 * size
                e += HALF_EPS[dtype] * (np.abs(o) + e) + 2.0 ** -25
            out[b, :, h], bound[b, :, h] = o, e
            lost = (see & (np.isnan(sk) | np.isnan(sv))).any(1)
            out[b, lost, h] = np.nan
    return out, bound, written


def launch(hip, cache, q, dtype, pos, counts, sees, scale):
    batch, hk, max_seq, d = cache.shape
    heads, rows = q.shape[1], q.shape[2]
    dq, do = dev_typed(hip, q, dtype), dev_typed(hip, np.full((batch, rows, heads, d), SENTINEL), dtype)
    dp = dev(hip, np.asarray(pos, np.int32))
    dc = dev(hip, np.asarray(counts, np.int32)) if counts is not None else None
    dt = dev(hip, words_of(sees)) if sees is not None else None
    need = hip.attention_q8_workspace_bytes(batch, rows, heads, hk, d, max_seq)
    ws = dev(hip, np.zeros(max(need, 1), np.uint8))
    hip.attention_q8(cache.q8, dq.addr, do.addr, dtype, rows, heads, dp.addr, dc.addr if dc else None, dt.addr if dt else None,
                     scale, ws.addr, ws.nbytes)
    out = host_typed(do, (batch, rows, heads, d), dtype)
    if need:
        assert (ws.download(np.uint32, (TICKETS,)) == 0).all(), "tickets left behind"
    return out


def check(hip, cache, q, dtype, pos, counts, sees, splits, scale=0.12):
    batch, hk, max_seq, d = cache.shape
    heads, rows = q.shape[1], q.shape[2]
    rt, got_splits, _ = plan(batch, rows, heads, hk, d, max_seq, dtype)
    assert rt == (4 if d == 64 and dtype else 2) and (got_splits > 1) == splits
    assert hip.attention_q8_workspace_bytes(batch, rows, heads, hk, d, max_seq) == max(
        plan(batch, rows, heads, hk, d, max_seq, t)[2] for t in (0, 4))
    got = launch(hip, cache, q, dtype, pos, counts, sees, scale).astype(np.float64)
    ref, bound, written = reference(cache, q, dtype, pos, counts, sees, scale)
    assert (got[~written] == SENTINEL).all(), "a padding row was written"
    got, ref, bound = got[written], ref[written], bound[written]
    assert np.array_equal(np.isnan(got), np.isnan(ref))
    fine = ~np.isnan(ref)
    err = np.abs(got - ref)[fine]
    assert np.all(err <= bound[fine]), (err.max(), np.max(err / np.maximum(bound[fine], 1e-300)))
    return got


# (batch, kv heads, heads of a group, rows, pos, max_seq, counts, keys are shared)
CASES = [
    (1, 4, 8, 24, [3000], 12000, None, True), (2, 3, 5, 17, [2500, 40], 12000, [17, 9], True), (40, 2, 2, 40, None, 1000, None, True),
    (1, 8, 8, 24, [700], 6100, [23], True), (1, 4, 8, 1000, [301], 1301, None, False), (2, 9, 3, 345, [0, 77], 430, [345, 200], False),
    (1, 2, 64, 11, [5000], 16384, None, True),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "x".join(map(str, c[:4])))
@pytest.mark.parametrize("tree", [False, True], ids=["chain", "tree"])
@pytest.mark.parametrize("d,dtype", TYPES)
def test_many_rows(hip, case, tree, d, dtype):
    batch, hk, g, rows, pos, max_seq, counts, splits = case
    if pos is None:
        pos = np.random.default_rng(1).integers(0, max_seq - rows + 1, batch).tolist()
    print(f"case attention_q8 tiles {case[:4]} pos={pos[:3]} tree={tree} d={d} dtype={dtype}", flush=True)
    cache = Cache(hip, batch, hk, max_seq, d, rows)
    check(hip, cache, queries(batch, hk * g, rows, d, dtype, rows), dtype, pos, counts, tree_of(batch, rows, rows) if tree else None, splits)


@pytest.mark.parametrize("d,dtype", TYPES)
def test_masks_that_leave_nothing_stale_rows_and_nan(hip, d, dtype):
    # nodes that see nothing, with and without cached tokens in front; NaN
    # scales of nodes that nobody sees and past the call's rows; one that is
    # seen reaches those who see it and nobody else; counts below the rows
    batch, hk, g, rows, pos, max_seq, counts = 2, 3, 5, 17, [0, 333], 12000, [17, 12]
    cache = Cache(hip, batch, hk, max_seq, d, 11)
    sees = tree_of(batch, rows, 12)
    sees[0, 3] = sees[0, 16] = sees[1, 1] = False
    sees[:, :, 6] = False
    sees[1, 5, 7] = True
    for kv in "kv":
        s = cache.host[kv + "_scales"]
        for b in range(batch):
            s[b, :, pos[b] + counts[b]:] = np.nan
            s[b, :, pos[b] + 6] = np.nan
    cache.host["v_scales"][1, 1, pos[1] + 2] = np.nan
    cache.host["k_scales"][0, 2, 4] = np.nan
    for name, buf in cache.dev.items():
        buf.upload(cache.host[name])
    print(f"case attention_q8 tiles masks d={d} dtype={dtype}", flush=True)
    got = check(hip, cache, queries(batch, hk * g, rows, d, dtype, 13), dtype, pos, counts, sees, True)
    assert (got[3] == 0).all() and (got[16] == 0).all() and np.isnan(got).any()


@pytest.mark.parametrize("d,dtype", [(64, 5), (128, 0)])
def test_replayed_with_other_positions_beside_another_stream(hip, d, dtype):
    batch, hk, g, rows, max_seq = 1, 4, 8, 24, 12000
    cache = Cache(hip, batch, hk, max_seq, d, 14)
    q = queries(batch, hk * g, rows, d, dtype, 15)
    assert plan(batch, rows, hk * g, hk, d, max_seq, dtype)[:2] == ((4, 42) if d == 64 else (2, 21))
    need = hip.attention_q8_workspace_bytes(batch, rows, hk * g, hk, d, max_seq)
    sets = []
    for _ in range(2):
        stream = hip.Stream()
        bufs = [dev_typed(hip, q, dtype), dev_typed(hip, np.zeros((batch, rows, hk * g, d)), dtype), dev(hip, np.zeros(batch, np.int32)),
                dev(hip, np.zeros(need, np.uint8))]
        hip.synchronize()
        graph = hip.Graph(stream)
        graph.begin()
        hip.attention_q8(cache.q8, bufs[0].addr, bufs[1].addr, dtype, rows, hk * g, bufs[2].addr, None, None, 0.12, bufs[3].addr, need, stream)
        graph.end()
        sets.append((stream, graph, bufs))
    for pos in ([9000], [0], [2222]):
        print(f"case attention_q8 tiles replay {pos} d={d} dtype={dtype}", flush=True)
        for stream, _, bufs in sets:
            bufs[2].upload(np.array(pos, np.int32), stream.handle)
        for _ in range(4):
            for _, graph, _ in sets:
                graph.launch()
        want = launch(hip, cache, q, dtype, pos, None, None, 0.12)
        for stream, _, bufs in sets:
            stream.synchronize()
            assert np.array_equal(host_typed(bufs[1], (batch, rows, hk * g, d), dtype), want)
