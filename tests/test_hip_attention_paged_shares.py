"""Every key of a long context counts once, whichever workgroups take it, and the
kernel of two row tiles a wave over pages, on the GPU.

Keys of zeros weigh alike, so an output is the mean of the values that its row sees,
and a value is not 0 only in the element that its 16 tokens have: lost or repeated
ones change that element by several per cent.  Weights are powers of two and sums
of whole numbers exact (below 2^24); a part's factor, the sum's reciprocal and the
product with it are off by 2^-22 in all, and the result is rounded by half a step."""
from __future__ import annotations

import numpy as np
import pytest

from test_hip_attention_paged import SIZE, STEP, TYPES, Packed, Paged, close, held, reference

pytestmark = pytest.mark.gpu

BLOCK = 16


def marked(length, d, seed):
    """Values [length, d]: 1, 2 or 3 in one element of each token, the same of 16 tokens."""
    r = np.random.default_rng(seed)
    blocks = -(-length // BLOCK)
    v = np.zeros((length, d))
    t = np.arange(length)
    v[t, (t // BLOCK) % d] = r.choice([1.0, 2.0, 3.0], blocks)[t // BLOCK]
    return v


def check(got, v, first, dtype):
    """got [rows, heads, d] against means over the values [keys, d] up to each row's own."""
    sums = np.cumsum(v, 0)
    for i in range(got.shape[0]):
        seen = first + i + 1
        want = sums[seen - 1] / seen
        tol = want * (STEP[dtype] + 2.0 ** -22)
        # a block less changes its element by its own share, and all by the smaller count
        whole = seen // BLOCK
        at = np.arange(whole) % v.shape[1]
        lost = v[np.arange(whole) * BLOCK, at] * BLOCK / seen
        assert (lost > 2 * tol[at] + 2 * want[at] * BLOCK / seen).all() or whole < 2, "a lost block would not show"
        close(got[i], np.broadcast_to(want, got[i].shape), np.broadcast_to(tol, got[i].shape))


SHAPES = [(1, 20000), (2, 9000), (4, 20000), (40, 6000), (130, 5000), (7, 33000)]


@TYPES
@pytest.mark.parametrize("heads,hk,d", [(32, 4, 64), (8, 1, 128), (16, 16, 64), (40, 1, 128)], ids=str)
@pytest.mark.parametrize("n,length", SHAPES, ids=str)
@pytest.mark.parametrize("beside", [False, True], ids=["alone", "beside others"])
def test_every_key_once(hip, dtype, heads, hk, d, n, length, beside):
    if beside:
        c = Paged(hip, dtype, [1, n, 1, 3], [3000, length, 77, 1500], heads, hk, d, 16, 71)
    else:
        c = Paged(hip, dtype, [n], [length], heads, hk, d, 64, 72)
    c.k[:] = 0
    values = [marked(int(total), d, 73 + b) for b, total in enumerate(c.lengths)]
    for b, v in enumerate(values):
        t = np.arange(len(v))
        c.v[c.tables[b, t // c.page], :, t % c.page] = v[:, None]
    c.upload().call()
    got = c.result()
    for b, v in enumerate(values):
        check(got[c.start[b]:c.start[b + 1]], v, len(v) - int(c.n[b]), dtype)


@TYPES
@pytest.mark.parametrize("heads,hk,d", [(32, 4, 64), (8, 2, 128)], ids=str)
@pytest.mark.parametrize("n", [[5000], [100, 3000, 7], [700] * 6], ids=str)
def test_every_key_of_prompts_once(hip, dtype, heads, hk, d, n):
    c = Packed(hip, dtype, n, heads, hk, d, 74)
    c.qkv[:, heads:heads + hk] = 0
    values = [marked(x, d, 75 + b) for b, x in enumerate(n)]
    c.qkv[:, heads + hk:] = np.concatenate(values)[:, None]
    c.upload().call()
    got = c.result()
    for b, v in enumerate(values):
        rows = got[c.start[b]:c.start[b + 1]]
        for i in sorted({0, 15, 16, 127, 128, len(v) // 2, len(v) - 129, len(v) - 1} & set(range(len(v)))):
            check(rows[i:i + 1], v, i, dtype)


# Steps of 2048 rows and more of 64-wide 16-bit heads in groups of 4 and more: two row
# tiles a wave.  Offsets that leave most of the rows to padding, as a captured step's
# are, have their keys shared out and parts of 256 rows joined.
@pytest.mark.parametrize("dtype", [4, 5], ids=["f16", "bf16"])
@pytest.mark.parametrize("n,lengths,pad,max_rows", [([2100], [3500], 0, None), ([900, 1, 1200, 40], [2000, 700, 1200, 900], 3, None),
                                                    ([40, 1, 300, 2], [9000, 4000, 333, 60], 2000, 0),
                                                    ([1, 1, 1], [5000, 1, 77], 2200, 0), ([33], [6000], 2048, 0),
                                                    ([0, 600, 0, 1], [9, 8000, 3, 130], 1600, 700)], ids=str)
@pytest.mark.parametrize("heads,hk", [(64, 8), (80, 5), (64, 16)], ids=str)
@pytest.mark.parametrize("page", [16, 128])
def test_two_row_tiles_a_wave(hip, dtype, n, lengths, pad, max_rows, heads, hk, page):
    c = Paged(hip, dtype, n, lengths, heads, hk, 64, page, 76, max_rows=max_rows, pad=pad).upload()
    g = heads // hk
    assert g >= 4 and c.rows * g // 256 * hk >= 512
    c.call()
    got, q = c.result(), held(c.q, dtype)
    for b in range(len(n)):
        k, v, _ = c.keys(b)
        rows = slice(int(c.start[b]), int(c.start[b + 1]))
        for h in (0, hk - 1):
            u = [h * g, h * g + g - 1]
            want, tol = reference(q[rows][:, u], k[:, [h]], v[:, [h]], lengths[b] - n[b], 64 ** -0.5, dtype)
            close(got[rows][:, u], want, tol)
    left = c.out.download(np.uint8, (c.rows, heads * 64 * SIZE[dtype]))[c.start[-1]:]
    assert (left == 0x5b).all()
    for _ in range(2):
        c.call()
        assert np.array_equal(got, c.result())


@pytest.mark.parametrize("dtype", [4, 5], ids=["f16", "bf16"])
def test_two_row_tiles_a_wave_count_every_key_once(hip, dtype):
    for n, length, pad in [(40, 9000, 2050), (300, 4100, 2000), (2100, 2500, 0)]:
        c = Paged(hip, dtype, [n, 1], [length, 2000], 64, 8, 64, 16, 77, pad=pad, max_rows=0)
        c.k[:] = 0
        values = [marked(length, 64, 78), marked(2000, 64, 79)]
        for b, v in enumerate(values):
            t = np.arange(len(v))
            c.v[c.tables[b, t // 16], :, t % 16] = v[:, None]
        c.upload().call()
        got = c.result()
        for i in (0, 31, n // 2, n - 1):
            check(got[i:i + 1], values[0], length - n + i, dtype)
        check(got[n:n + 1], values[1], 1999, dtype)
