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
