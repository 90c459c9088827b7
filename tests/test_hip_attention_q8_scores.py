"""Attention over the INT8 cache with 16-bit queries: scores that lie close to
one another and far from zero, over keys whose scale one channel sets.

Every sum of products is exact here: a query's values are multiples of 2^-11
below 2 and codes whole numbers, so any partial sum of at most 128 products is
a multiple of 2^-11 below 2^13 (at most 24 bits).  What is left of the bound of
test_hip_attention_q8.py are a score's further roundings, 8 |s| 2^-24 in all,
so for fp16 weights and the output's own rounding (HALF_EPS of its size)
  |err| <= (2 (8 max|s| 2^-24 + 2^-20 + n 2^-23) + 2^-11) sum p |v|."""
from __future__ import annotations

import numpy as np
import pytest

from test_hip_attention_q8 import HALF_EPS, run
from test_hip_kv_q8 import Cache

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("batch,hk,g,rows,pos,max_seq", [(1, 1, 8, 4, [20], 32), (2, 4, 8, 9, [20, 11], 8192)])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", [4, 5])
def test_close_scores_far_from_zero(hip, batch, hk, g, rows, pos, max_seq, d, dtype):
    r = np.random.default_rng(d)
    q = r.integers(4, 8, (batch, hk * g, rows, d)).astype(np.float32) / 4
    q[..., 0] = 0
    q[..., 1:9] = r.integers(-8, 9, q[..., 1:9].shape).astype(np.float32) / 2048
    cache = Cache(hip, batch, hk, max_seq, d, 7)
    codes = cache.host["k_codes"]
    codes[..., 9:] = 2
    codes[..., 0] = 127   # (the channel that sets the scale, where the queries are 0)
    scale = 0.125
    cache.host["k_scales"][:] = np.float32(1000 / (scale * 1.4 * 2 * (d - 9)))
    for name, buf in cache.dev.items():
        buf.upload(cache.host[name])
    print(f"case attention_q8 close scores batch={batch} d={d} dtype={dtype}", flush=True)
    got = run(hip, cache, q, dtype, pos, None, None, scale).astype(np.float64)
    for b in range(batch):
        for h in range(hk * g):
            kc, vc = (cache.host[x + "_codes"][b, h // g].astype(np.float64) for x in "kv")
            sk, sv = (cache.host[x + "_scales"][b, h // g].astype(np.float64) for x in "kv")
            for t in range(rows):
                n = pos[b] + t + 1
                s = scale * (kc[:n] @ q[b, h, t].astype(np.float64)) * sk[:n]
                p = np.exp(s - s.max())
                w = p / p.sum() * sv[:n]
                o, size = w @ vc[:n], w @ np.abs(vc[:n])
                bound = (2 * (8 * np.abs(s).max() * 2.0 ** -24 + 2.0 ** -20 + n * 2.0 ** -23) + 2.0 ** -11) * size
                bound += HALF_EPS[dtype] * (np.abs(o) + bound) + 2.0 ** -25
                err = np.abs(got[b, t, h] - o)
                assert np.all(err <= bound), (b, h, t, float((err / bound).max()))
