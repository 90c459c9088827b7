"""Small weights and large scores in the attention over cache pages and of
packed prompts, on the GPU, against the formula in 64 bits.

Scores here are exact, so a weight is off by what the roundings of its
exponent (log2 units below 32: the reference, its part's reference and the factor 1 /
ln 2, 2^-20 each, so 2^-18 of the weight with exp2 itself) and the 16 bits that it is
rounded to make of it: half a step of the rows' type, and with F16 at least 2^-33 of
the row's largest weight.  Sums of n weights add n 2^-24, once above and once
below the line; the result is rounded by half a step."""
from __future__ import annotations

import numpy as np
import pytest

from test_hip_attention_paged import STEP, TYPES, WEIGHT, Packed, Paged, close, held

pytestmark = pytest.mark.gpu


def small(values, scores, dtype):
    """(outputs [d], tolerances) of one row over values [keys, d] with these scores."""
    p = np.exp(scores - scores.max())
    l = p.sum()
    out = p @ values / l
    a = np.abs(values)
    each = p * (WEIGHT[dtype] + 2.0 ** -18) + (2.0 ** -33 if dtype == 4 else 0)
    tol = each @ a / l + (p @ a / l) * (len(p) * 2.0 ** -23 + 2.0 ** -18) + np.abs(out) * STEP[dtype]
    return out, tol + (2.0 ** -25 if dtype == 4 else 0)


@TYPES
@pytest.mark.parametrize("low", [15.0, 17.0, 17.5])
@pytest.mark.parametrize("n,length,heads,hk,d", [(1, 700, 4, 4, 64), (1, 300, 16, 2, 128), (1, 9000, 8, 1, 64),
                                                 (40, 2000, 16, 2, 128), (150, 150, 8, 2, 64), (40, 9000, 8, 8, 64)],
                         ids=str)
def test_many_small_weights_behind_large_ones(hip, dtype, low, n, length, heads, hk, d):
    """A few keys that every row weighs 1 and whose values are 0, and all others
    `low` below them: the outputs are theirs alone.  16 bits keep e^-17."""
    c = Paged(hip, dtype, [n], [length], heads, hk, d, 16, 41)
    c.scale = 1.0
    c.q[:] = c.k[:] = 0
    c.q[:, :, 0] = 1
    values = np.random.default_rng(42).choice([256.0, 512.0, 1024.0], (length, d))
    large = np.zeros(length, bool)
    large[:128:32] = True    # the first key of every wave
    values[large] = 0
    t = np.arange(length)
    c.k[c.tables[0, t // 16], :, t % 16, 0] = np.where(large, low, 0)[:, None]
    c.v[c.tables[0, t // 16], :, t % 16] = values[:, None]
    c.upload().call()
    got = c.result()
    for i in {0, n // 2, n - 1}:
        seen = length - n + i + 1
        want, tol = small(values[:seen], np.where(large[:seen], low, 0), dtype)
        close(got[i], np.broadcast_to(want, (heads, d)), np.broadcast_to(tol, (heads, d)))


@TYPES
@pytest.mark.parametrize("d", [64, 128])
def test_many_small_weights_in_a_prompt(hip, dtype, d):
    """The same in packed prompts, with as many rows as need no sharing of keys."""
    heads, hk, low, n = 32, 4, 17.25, [1500, 33]
    c = Packed(hip, dtype, n, heads, hk, d, 43)
    c.scale = 1.0
    c.qkv[:] = 0
    c.qkv[:, :heads, 0] = 1
    values = np.random.default_rng(44).choice([256.0, 512.0, 1024.0], (sum(n), d))
    values[0] = values[n[0]] = 0
    c.qkv[0, heads:heads + hk, 0] = c.qkv[n[0], heads:heads + hk, 0] = low
    c.qkv[:, heads + hk:] = values[:, None]
    c.upload().call()
    got = c.result()
    for i in (1, 31, 700, 1499, 1501, 1532):
        first = 0 if i < n[0] else n[0]
        scores = np.zeros(i + 1 - first)
        scores[0] = low
        want, tol = small(values[first:i + 1], scores, dtype)
        close(got[i], np.broadcast_to(want, (heads, d)), np.broadcast_to(tol, (heads, d)))


# A reference near 2^k has a step of 2^(k - 23): what its rounding adds to every exponent
# (0.43 steps with queries of 167, -0.22 with 131) passes what F16 holds from 2^28 on,
# and fp32 from 2^32.
@TYPES
@pytest.mark.parametrize("n,length,heads,hk,d", [(1, 700, 4, 4, 64), (3, 300, 16, 2, 128), (1, 9000, 8, 1, 64),
                                                 (40, 2000, 16, 2, 128), (150, 150, 8, 2, 64), (40, 6000, 8, 8, 64)],
                         ids=str)
@pytest.mark.parametrize("power", [14, 17, 22, 28, 30, 34, 60, 99])
@pytest.mark.parametrize("query", [167.0, 131.0])
@pytest.mark.parametrize("sign", [1, -1], ids=["positive", "negative"])
def test_large_scores(hip, dtype, n, length, heads, hk, d, power, query, sign):
    """Scores of about 2^power, and half or twice that: some keys weigh 1, all others
    nothing, and the outputs are means of the values of the first."""
    c = Paged(hip, dtype, [n], [length], heads, hk, d, 16, 45)
    c.scale = float(np.float32(2.0) ** (power - 14) * np.float32(1.1))
    c.q[:] = c.k[:] = 0
    c.q[:, :, 1] = query
    t = np.arange(length)
    large = np.random.default_rng(46).random(length) < 0.4
    large[0] = True
    key = np.where(large, 93.0, 46.5) if sign > 0 else np.where(large, -46.5, -93.0)
    c.k[c.tables[0, t // 16], :, t % 16, 1] = key[:, None]
    c.upload().call()
    got = c.result()
    _, values, _ = c.keys(0)
    for i in {0, n // 2, n - 1}:
        seen = np.flatnonzero(large[:length - n + i + 1])
        for h in range(heads):
            v = values[seen][:, h // (heads // hk)]
            mean = v.mean(0)
            # weights are alike, but not 1: at 2^14 167 adds 0.43 2^-9 to their exponents, so that
            # 16 bits round each (1.0006, half a step of the rows' type, WEIGHT), their sum not
            tol = np.abs(v).mean(0) * (len(seen) * 2.0 ** -23 + 2.0 ** -22 + WEIGHT[dtype]) + np.abs(mean) * STEP[dtype]
            close(got[i, h], mean, tol + (2.0 ** -25 if dtype == 4 else 0))
