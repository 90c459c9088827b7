"""Attention over the INT8 cache where value scales lie far apart: rows of
zeros (stored with scale 1) beside small values, keys that a row does not see,
keys whose weight is next to nothing, scales that grow from token to token.
What a row gets depends on the keys that it sees and their weights alone.

Bound.  Scores, sums and outputs as in test_hip_attention_q8.py:
  2 (max ds + 2^-20 + n 2^-23) sum p |v|,   and for 16-bit queries 2^-11 sum p |v|
and the output's own rounding.  Beside it a product of a weight and its value
scale is fp16 in a unit where the row's largest such product (of keys whose
codes are not all zero) is 2^3 at least, so below fp16's normal range it is
off by half the smallest step, 2^-25, that is 2^-28 of the row's largest:
  2^-28 max(p sv) sum |cv|."""
from __future__ import annotations

import numpy as np
import pytest

from test_hip_attention_q8 import HALF_EPS, queries, run, tree_of
from test_hip_kv_q8 import Cache

pytestmark = pytest.mark.gpu

# (batch, kv heads, heads of a group, rows, pos, max_seq): one row tile a wave; several (two or four) with padding rows
# and an odd tail; keys shared by several workgroups
SHAPES = [(1, 2, 2, 12, [200], 600), (2, 4, 8, 9, [300, 45], 8192), (1, 1, 4, 6, [3000], 3100)]
TYPES = [(64, 0), (64, 4), (64, 5), (128, 0), (128, 4), (128, 5)]


def reference(cache, q, dtype, pos, sees, scale):
    """(out [batch, rows, heads, d], bound), in 64 bits."""
    batch, hk, max_seq, d = cache.shape
    heads, rows = q.shape[1], q.shape[2]
    g = heads // hk
    out, bound = np.zeros((batch, rows, heads, d)), np.zeros((batch, rows, heads, d))
    for b in range(batch):
        n = min(pos[b] + rows, max_seq)
        see = np.ones((rows, n), bool)
        see[:, pos[b]:] = (np.tri(rows, dtype=bool) if sees is None else sees[b])[:, :n - pos[b]]
        for h in range(heads):
            kc, vc = (cache.host[x + "_codes"][b, h // g, :n].astype(np.float64) for x in "kv")
            sk, sv = (cache.host[x + "_scales"][b, h // g, :n].astype(np.float64) for x in "kv")
            x, k = q[b, h].astype(np.float64), kc * sk[:, None]
            s = scale * (x @ k.T)
            ds = scale * (np.abs(x).max(1)[:, None] * np.abs(k).sum(1) * 2.0 ** -22 + (d + 4) * (np.abs(x) @ np.abs(k).T) * 2.0 ** -24) + 8 * np.abs(s) * 2.0 ** -24
            s = np.where(see, s, -np.inf)
            ds = np.where(see, ds, 0)
            with np.errstate(all="ignore"):
                p = np.where(see, np.exp(s - s.max(1, keepdims=True)), 0)
                p = np.where(see.any(1)[:, None], p / p.sum(1, keepdims=True), 0)
            w = p * sv
            o, size = w @ vc, w @ np.abs(vc)
            most = np.where((vc != 0).any(1), w, 0).max(1)
            e = 2 * (ds.max(1) + 2.0 ** -20 + see.sum(1) * 2.0 ** -23)[:, None] * size
            e += 2.0 ** -28 * most[:, None] * (see.astype(np.float64) @ np.abs(vc))
            if dtype:
                e += 2.0 ** -11 * size
                e += HALF_EPS[dtype] * (np.abs(o) + e) + (2.0 ** -25 if dtype == 4 else 0)
            out[b, :, h], bound[b, :, h] = o, e
    return out, bound


def check(hip, cache, q, dtype, pos, sees, scale):
    for name, buf in cache.dev.items():
        buf.upload(cache.host[name])
    got = run(hip, cache, q, dtype, pos, None, sees, scale).astype(np.float64)
    ref, bound = reference(cache, q, dtype, pos, sees, scale)
    fits = np.abs(ref) + bound < (65504 if dtype == 4 else 3e38)
    assert fits.mean() > 0.3
    with np.errstate(invalid="ignore"):
        err = np.abs(got - ref)[fits]
    assert np.all(err <= bound[fits]), (err.max(), np.nanmax(err / np.maximum(bound[fits], 1e-300)), int((~(err <= bound[fits])).sum()))
    return got


def make(hip, shape, d, dtype, seed):
    batch, hk, g, rows, pos, max_seq = shape
    cache = Cache(hip, batch, hk, max_seq, d, seed)
    return cache, queries(batch, hk * g, rows, d, dtype, seed)


@pytest.mark.parametrize("size", [1e2, 1e-2, 1e-4, 1e-6, 1e-8, 1e-30])
@pytest.mark.parametrize("d,dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_rows_of_zeros_beside_small_values(hip, shape, d, dtype, size):
    # a fifth of the cached rows, a whole block of them and two of the call's
    # own rows (a batch padded with zeros) are zeros with scale 1
    batch, hk, _, rows, pos, max_seq = shape
    cache, q = make(hip, shape, d, dtype, 21)
    cache.host["v_scales"] *= np.float32(size)
    zero = np.random.default_rng(3).random((batch, hk, max_seq)) < 0.2
    zero[:, :, :32] = True
    for b in range(batch):
        zero[b, :, pos[b] + rows - 2:] = True
    cache.host["v_codes"][zero], cache.host["v_scales"][zero] = 0, 1.0
    print(f"case attention_q8 zeros {shape} d={d} dtype={dtype} size={size}", flush=True)
    for sees in (None, tree_of(batch, rows, 4)):
        check(hip, cache, q, dtype, pos, sees, 0.1)


@pytest.mark.parametrize("d,dtype", TYPES)
def test_values_of_zeros_only(hip, d, dtype):
    shape = SHAPES[0]
    cache, q = make(hip, shape, d, dtype, 22)
    cache.host["v_codes"][:], cache.host["v_scales"][:] = 0, 1.0
    print(f"case attention_q8 only zeros d={d} dtype={dtype}", flush=True)
    assert (check(hip, cache, q, dtype, shape[4], None, 0.1) == 0).all()


@pytest.mark.parametrize("ratio", [20, 26, 50, 100])
@pytest.mark.parametrize("d,dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_large_values_of_nodes_that_are_not_seen(hip, shape, d, dtype, ratio):
    # node 2 is seen by nobody, node 3 by itself and its descendants: both
    # hold values 2^ratio times the others'
    batch, _, _, rows, pos, _ = shape
    cache, q = make(hip, shape, d, dtype, 23)
    sees = tree_of(batch, rows, 5)
    sees[:, :, 2] = False
    sees[:, 4, 3] = False   # (an aunt)
    for b in range(batch):
        for node in (2, 3):
            cache.host["v_scales"][b, :, pos[b] + node] *= np.float32(2.0) ** ratio
    print(f"case attention_q8 unseen values {shape} d={d} dtype={dtype} 2^{ratio}", flush=True)
    check(hip, cache, q, dtype, pos, sees, 0.1)


@pytest.mark.parametrize("step", [1, 4, 12])
@pytest.mark.parametrize("d,dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_values_that_grow_from_token_to_token(hip, shape, d, dtype, step):
    # a prompt whose every token's values are 2^step times the one's before:
    # what comes later is not seen, what came before hardly counts
    batch, _, _, rows, pos, max_seq = shape
    cache, q = make(hip, shape, d, dtype, 24)
    scales = cache.host["v_scales"]
    first = -round(0.6 * step * rows)   # (fp16 outputs hold the first half)
    for b in range(batch):
        token = np.clip(np.arange(max_seq) - pos[b], 0, rows - 1)
        scales[b] = np.ldexp(scales[b], first + step * token)
    print(f"case attention_q8 growing values {shape} d={d} dtype={dtype} 2^{step}", flush=True)
    check(hip, cache, q, dtype, pos, None, 0.1)


@pytest.mark.parametrize("ratio", [20, 40, 60])
@pytest.mark.parametrize("d,dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_large_values_that_weigh_next_to_nothing(hip, shape, d, dtype, ratio):
    # key 7's score is 60 below 0 in the rows whose query starts with 4 and
    # 60 above it in those that start with -4: of its values, 2^ratio times
    # the others', the former see about 2^(ratio - 86), the latter all
    batch, _, _, rows, pos, _ = shape
    cache, q = make(hip, shape, d, dtype, 25)
    q[..., 0] = np.where(np.arange(rows) % 3 == 0, -4.0, 4.0)
    cache.host["k_codes"][:, :, 7] = 0
    cache.host["k_codes"][:, :, 7, 0] = -127
    cache.host["k_scales"][:, :, 7] = np.float32(60 / (127 * 4 * 0.1))
    cache.host["v_scales"][:, :, 7] *= np.float32(2.0) ** ratio
    print(f"case attention_q8 weightless values {shape} d={d} dtype={dtype} 2^{ratio}", flush=True)
    check(hip, cache, q, dtype, pos, None, 0.1)


@pytest.mark.parametrize("size", [1e2, 1.0, 1e-6])
@pytest.mark.parametrize("d,dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_rows_of_zeros_that_take_nearly_all_the_weight(hip, shape, d, dtype, size):
    # key 7 holds zeros (scale 1); its score is 30 above the others' size in
    # every third row, 30 below it in the others
    batch, _, _, rows, pos, _ = shape
    cache, q = make(hip, shape, d, dtype, 26)
    q[..., 0] = np.where(np.arange(rows) % 3 == 0, -4.0, 4.0)
    cache.host["k_codes"][:, :, 7] = 0
    cache.host["k_codes"][:, :, 7, 0] = -127
    cache.host["k_scales"][:, :, 7] = np.float32(30 / (127 * 4 * 0.1))
    cache.host["v_scales"] *= np.float32(size)
    cache.host["v_codes"][:, :, 7], cache.host["v_scales"][:, :, 7] = 0, 1.0
    print(f"case attention_q8 zeros' weight {shape} d={d} dtype={dtype} size={size}", flush=True)
    check(hip, cache, q, dtype, pos, None, 0.1)


@pytest.mark.parametrize("d,dtype", [(64, 0), (64, 5), (128, 0), (128, 5)])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_largest_scales(hip, shape, d, dtype):
    # keys' scales up to 2^98 under queries so small that scores are ordinary
    # ones, values' scales up to 2^88
    cache, q = make(hip, shape, d, dtype, 27)
    cache.host["k_scales"] = np.ldexp(np.minimum(cache.host["k_scales"] * 50, np.float32(0.999)), 98)
    cache.host["v_scales"] = np.ldexp(np.minimum(cache.host["v_scales"] * 50, np.float32(0.999)), 88)
    q = np.ldexp(q, -105)
    print(f"case attention_q8 largest scales {shape} d={d} dtype={dtype}", flush=True)
    check(hip, cache, q, dtype, shape[4], None, 0.1)
