"""Row offsets that fall, are negative or lie past the rows, in the attention over
cache pages and of packed prompts, on the GPU: they are held to [0, rows] and to the
largest before them, every row is one request's, and nothing but its rows is
written, behind and in front of the output neither.  Tolerances are those of the
formula's test."""
from __future__ import annotations

import numpy as np
import pytest

from test_hip_attention_paged import SIZE, TYPES, Packed, Paged

pytestmark = pytest.mark.gpu

GUARD = 1 << 16


class Guarded:
    """A device buffer of 0x5b bytes with as many in front of it and behind it as GUARD says."""

    def __init__(self, hip, nbytes):
        self.nbytes = nbytes
        self.buf = hip.DeviceBuffer.from_array(np.full(nbytes + 2 * GUARD, 0x5b, np.uint8))
        self.addr = self.buf.addr + GUARD

    def bytes(self):
        return self.buf.download(np.uint8, (self.nbytes + 2 * GUARD,))

    def download(self, dtype, shape):
        return self.bytes()[GUARD:GUARD + self.nbytes].view(dtype).reshape(shape)

    def check(self):
        b = self.bytes()
        assert (b[:GUARD] == 0x5b).all() and (b[-GUARD:] == 0x5b).all(), "written outside the output"


def rising(start, rows):
    return np.maximum.accumulate(np.clip(np.asarray(start, np.int64), 0, rows))


def given(c, start):
    """Call c (uploaded) with these offsets, and check it."""
    c.start = rising(start, c.rows)
    c.n = np.diff(c.start)
    c.ds = c.hip.DeviceBuffer.from_array(np.asarray(start, np.int32))
    c.out = Guarded(c.hip, c.rows * c.heads * c.d * SIZE[c.dtype])
    for _ in range(2):   # the workspace is left ready
        c.call()
    c.check()
    left = c.out.download(np.uint8, (c.rows, c.heads * c.d * SIZE[c.dtype]))
    assert (left[:c.start[0]] == 0x5b).all() and (left[c.start[-1]:] == 0x5b).all()
    c.out.check()


STARTS = [[0, 30, 10, 30], [5, 3, 9, 40], [-4, 10, 10 ** 9, 20], [0, 2 ** 31 - 1, -2 ** 31, 30], [30, 20, 10, 0],
          [0, 25, 3, 28], [7, 7, 2, 7], [-9, -8, -7, -6], [31, 40, 50, 60], [2 ** 31 - 1, 0, 2 ** 31 - 1, 0], [4, 9, 9, 3]]


@TYPES
@pytest.mark.parametrize("start", STARTS, ids=str)
def test_three_requests(hip, dtype, start):
    given(Packed(hip, dtype, [10, 10, 10], 4, 2, 64, 51).upload(), start)
    n = np.diff(rising(start, 30))
    for max_rows in (0, max(1, int(n.max()))):
        c = Paged(hip, dtype, [10, 10, 10], [30, 300, 50], 4, 2, 64, 16, 52, max_rows=max_rows)
        given(c.upload(), start)


@pytest.mark.parametrize("batch,rows", [(2, 200), (60, 400), (300, 500), (2000, 700)], ids=str)
@pytest.mark.parametrize("dtype", [0, 4], ids=["f32", "f16"])
def test_many_requests(hip, dtype, batch, rows):
    """Offsets that go up and down, of more requests than threads too."""
    r = np.random.default_rng(batch)
    start = (np.linspace(0, rows, batch + 1) + r.normal(0, 12, batch + 1)).astype(np.int64)
    c = Packed(hip, dtype, [rows] + [0] * (batch - 1), 4, 2, 64, 53)
    given(c.upload(), start)
    n = np.diff(rising(start, rows))
    lengths = n + r.integers(0, 90, batch)
    c = Paged(hip, dtype, [rows] + [0] * (batch - 1), lengths, 4, 2, 64, 16, 54, max_rows=int(n.max()))
    given(c.upload(), start)


def test_tiles_of_many_sizes(hip):
    """Enough tiles that each has a workgroup of its own, sorted by length and not."""
    for n, heads, hk, d in [(2200, 32, 8, 128), (1500, 64, 8, 64)]:
        c = Packed(hip, 5, [n, 0, 0, 0, 0], heads, hk, d, 55).upload()
        given(c, [3, n // 2, 70, n // 3, 2 * n, n // 4])
