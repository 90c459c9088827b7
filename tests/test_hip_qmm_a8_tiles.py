"""The INT8 x INT8 product's 128 x 128 tiles, bit for bit: eight waves a tile
(160 to 255 tiles) and four (256 and more), over few and many stages of 64 k
and every remainder of them, with ragged rows and columns."""
from __future__ import annotations

import numpy as np
import pytest

from test_hip_kv_q8 import assert_equal, narrow
from test_hip_qmm_a8 import expect, run, weights

pytestmark = pytest.mark.gpu


def check(hip, m, k, n, dtype, least, most):
    tiles = -(-m // 128) * -(-n // 128)
    assert m > 128 and least <= tiles < most
    print(f"case qmm_a8 tiles m={m} k={k} n={n} dtype={dtype}", flush=True)
    a = narrow(np.random.default_rng(m + k).standard_normal((m, k)), dtype)
    codes, scale = weights(k, n, k + n)
    assert_equal(run(hip, a, codes, scale, dtype), expect(a, codes, scale, dtype))


@pytest.mark.parametrize("m,n", [(500, 5600), (1290, 2050), (200, 10309), (129, 10241), (512, 5632)])
@pytest.mark.parametrize("k", [64, 100, 192, 255, 320, 321, 448, 512, 570])   # one to nine stages
@pytest.mark.parametrize("dtype", [0, 4, 5])
def test_eight_waves(hip, m, n, k, dtype):
    check(hip, m, k, n, dtype, 160, 256)


@pytest.mark.parametrize("m,n,k", [(500, 5600, 2048), (1290, 2050, 2100), (512, 5632, 2048)])
def test_eight_waves_many_stages(hip, m, n, k):
    check(hip, m, k, n, 0, 160, 256)


@pytest.mark.parametrize("m,n", [(1100, 4000), (2049, 2049)])
@pytest.mark.parametrize("k", [64, 100, 192, 256, 300, 384, 448])   # one to seven stages
@pytest.mark.parametrize("dtype", [0, 4, 5])
def test_four_waves(hip, m, n, k, dtype):
    check(hip, m, k, n, dtype, 256, 1 << 20)
