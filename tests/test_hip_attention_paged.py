"""Attention over cache pages and of packed prompts on the GPU, against the
formula in 64 bits.

Tolerance of an element: with p_j the formula's weights (largest 1), l their
sum and D the head's size, a score's relative effect on its weight is at most
  e_j = scale (D + 4) 2^-24 sum_d |q_d k_jd| + |s_j| 2^-22 + 2^-20
(fp32 sums of D products; the scaled score and the reference, each rounded and
subtracted; exp2), twice for a sum in another order.  A weight's own rounding is
w = 2^-8 (bf16), 2^-11 (fp16) or nothing (fp32), below 2^-14 2^-25 absolute
(fp16); sums of n terms add n 2^-24, once above and once below the line; the
result is rounded by half a step r."""
from __future__ import annotations

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

TORCH = {0: torch.float32, 4: torch.float16, 5: torch.bfloat16}
SIZE = {0: 4, 4: 2, 5: 2}
STEP = {0: 2.0 ** -24, 4: 2.0 ** -11, 5: 2.0 ** -8}
WEIGHT = {0: 0.0, 4: 2.0 ** -11, 5: 2.0 ** -8}


def held(x, dtype):
    """x rounded to dtype, in 64 bits."""
    return torch.from_numpy(np.ascontiguousarray(x, np.float32)).to(TORCH[dtype]).double().numpy()


def raw(x, dtype):
    """The bytes of x in dtype."""
    t = torch.from_numpy(np.ascontiguousarray(x, np.float32)).to(TORCH[dtype])
    return t.numpy() if dtype == 0 else t.view(torch.int16).numpy()


def back(buf, shape, dtype):
    if dtype == 0:
        return buf.download(np.float32, shape).astype(np.float64)
    return torch.from_numpy(buf.download(np.int16, shape)).view(TORCH[dtype]).double().numpy()


def reference(q, k, v, first, scale, dtype):
    """(outputs, tolerances) of q [n, heads, d] over k, v [keys, hk, d]: row i
    sees keys up to first + i."""
    n, heads, d = q.shape
    hk = k.shape[1]
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    sees = np.arange(k.shape[0])[None, :] <= first + np.arange(n)[:, None]
    with np.errstate(all="ignore"):
        for h in range(heads):
            kh, vh = k[:, h // (heads // hk)], v[:, h // (heads // hk)]
            s = np.where(sees, scale * (q[:, h] @ np.where(np.isfinite(kh), kh, 0).T), -np.inf)
            size = scale * (np.abs(q[:, h]) @ np.abs(np.where(np.isfinite(kh), kh, 0)).T)
            top = s.max(1, keepdims=True, initial=-np.inf)
            p = np.where(sees, np.exp(s - np.where(np.isfinite(top), top, 0)), 0)
            l = np.maximum(p.sum(1, keepdims=True), 1e-300)
            e = 2 * (size * (d + 4) * 2.0 ** -24 + np.where(sees, np.abs(s), 0) * 2.0 ** -22 + 2.0 ** -20)
            a = np.abs(np.where(np.isfinite(vh), vh, 0))
            out[:, h] = (p @ np.where(np.isfinite(vh), vh, 0)) / l
            mean = (p @ a) / l
            part = (p * e) @ a / l + mean * ((p * e).sum(1, keepdims=True) / l)
            rounded = WEIGHT[dtype] * mean + (2.0 ** -25 * (sees @ a) / l if dtype == 4 else 0)
            tol[:, h] = part + rounded + mean * k.shape[0] * 2.0 ** -23 + np.abs(out[:, h]) * STEP[dtype] + 1e-37
            if dtype == 4:
                tol[:, h] += 2.0 ** -25   # a subnormal result
    return out, tol


def close(got, want, tol):
    assert got.shape == want.shape
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (f"{bad.sum()} of {bad.size}, first at {np.argwhere(bad)[0]}: {got[bad][0]!r}, not "
                           f"{want[bad][0]!r} +- {tol[bad][0]!r}")


class Paged:
    """A cache in pages with requests in it, and a call over its last rows."""

    def __init__(self, hip, dtype, n, lengths, heads, hk, d, page, seed, spare=3, max_rows=None, pad=0, fill=None):
        r = np.random.default_rng(seed)
        self.hip, self.dtype, self.n, self.lengths = hip, dtype, np.asarray(n), np.asarray(lengths)
        self.heads, self.hk, self.d, self.page = heads, hk, d, page
        self.rows = int(self.n.sum()) + pad
        need = -(-self.lengths // page)
        self.pages = int(need.sum()) + spare
        order = r.permutation(self.pages)
        self.max_pages = max(1, int(need.max()) + 1)
        self.tables = np.full((len(need), self.max_pages), -7, np.int32)
        at = 0
        for b, c in enumerate(need):
            self.tables[b, :c] = order[at:at + c]
            at += c
        shape = (self.pages, hk, page, d)
        big = np.where(np.arange(d) % 17 == 3, 3.0, 1.0)
        self.k, self.v = r.standard_normal(shape) * big, r.standard_normal(shape)
        if fill is not None:   # whatever lies behind a request's tokens and in free pages
            used = np.zeros((self.pages, page), bool)
            for b, length in enumerate(self.lengths):
                for t in range(int(length)):
                    used[self.tables[b, t // page], t % page] = True
            self.k[~used.repeat(hk, 0).reshape(self.pages, hk, page)] = fill
            self.v[~used.repeat(hk, 0).reshape(self.pages, hk, page)] = fill
        self.q = r.standard_normal((self.rows, heads, d))
        self.start = np.concatenate([[0], np.cumsum(self.n)]).astype(np.int32)
        self.max_rows = int(self.n.max()) if max_rows is None else max_rows
        self.scale = 0.0

    def upload(self):
        dev = self.hip.DeviceBuffer.from_array
        self.dk, self.dv, self.dq = (dev(raw(x, self.dtype)) for x in (self.k, self.v, self.q))
        self.dt, self.ds = dev(self.tables), dev(self.start)
        self.dl = dev(self.lengths.astype(np.int32))
        self.out = dev(np.full(self.rows * self.heads * self.d * SIZE[self.dtype], 0x5b, np.uint8))
        self.cache = self.hip.KvPaged(self.dk.addr, self.dv.addr, self.dtype, self.pages, self.page, self.hk, self.d)
        size = self.hip.attention_paged_workspace_bytes(len(self.n), self.rows, self.max_rows, self.heads, self.hk,
                                                        self.d, self.max_pages * self.page)
        self.ws = dev(np.zeros(max(1, size), np.uint8))
        return self

    def call(self, stream=None, ws=None):
        ws = ws or self.ws
        self.hip.attention_paged(self.cache, self.dt.addr, self.max_pages, self.dq.addr, self.out.addr, len(self.n),
                                 self.rows, self.max_rows, self.heads, self.ds.addr, self.dl.addr, self.scale, ws.addr,
                                 ws.nbytes, stream)

    def result(self):
        return back(self.out, (self.rows, self.heads, self.d), self.dtype)

    def keys(self, b):
        """(k, v) [tokens, hk, d] of request b, as held."""
        t = np.arange(int(self.lengths[b]))
        ids = self.tables[b, t // self.page]
        there = (ids >= 0) & (ids < self.pages)
        ids = np.where(there, ids, 0)
        k, v = (held(x[ids, :, t % self.page], self.dtype) for x in (self.k, self.v))
        return k, v, there

    def want(self):
        q = held(self.q, self.dtype)
        out = np.full(q.shape, np.nan)
        tol = np.full(q.shape, np.nan)
        scale = self.scale if self.scale > 0 else self.d ** -0.5
        for b, n in enumerate(self.n):
            if n == 0:
                continue
            a = int(self.start[b])
            todo = min(int(n), self.max_rows) if self.max_rows else int(n)
            k, v, there = self.keys(b)
            if not there.all():
                assert todo == 1
                k, v = k[there], v[there]
                first = len(k) - 1
            else:
                first = len(k) - n
            out[a:a + todo], tol[a:a + todo] = reference(q[a:a + todo], k, v, first, scale, self.dtype)
        return out, tol

    def check(self):
        want, tol = self.want()
        got = self.result()
        rows = ~np.isnan(want[:, 0, 0])
        close(got[rows], want[rows], tol[rows])
        left = self.out.download(np.uint8, (self.rows, self.heads * self.d * SIZE[self.dtype]))[~rows]
        assert (left == 0x5b).all(), "rows behind the last one were written"


TYPES = pytest.mark.parametrize("dtype", [0, 4, 5], ids=["f32", "f16", "bf16"])
HEADS = pytest.mark.parametrize("heads,hk,d", [(4, 4, 64), (32, 4, 64), (15, 5, 64), (16, 2, 128), (3, 1, 128)], ids=str)


@TYPES
@HEADS
@pytest.mark.parametrize("page", [16, 64, 256])
def test_single_tokens(hip, dtype, heads, hk, d, page):
    """Decoding: every length around blocks, rounds and pages."""
    lengths = [1, 2, 15, 16, 17, 31, 32, 33, 127, 128, 129, 255, 257, 300, 1000]
    c = Paged(hip, dtype, [1] * len(lengths), lengths, heads, hk, d, page, 1, pad=2).upload()
    c.call()
    c.check()


@TYPES
@HEADS
@pytest.mark.parametrize("n,before", [(2, 0), (3, 30), (5, 123), (17, 0), (33, 100), (64, 64), (70, 1), (150, 333),
                                      (300, 0)], ids=str)
def test_chunks(hip, dtype, heads, hk, d, n, before):
    """One request's chunk, and the same beside decoding ones."""
    c = Paged(hip, dtype, [n], [n + before], heads, hk, d, 32, 2).upload()
    c.call()
    c.check()
    c = Paged(hip, dtype, [1, n, 0, 1, 4], [40, n + before, 9, 513, 130], heads, hk, d, 16, 3, pad=5).upload()
    c.call()
    c.check()


@TYPES
@pytest.mark.parametrize("heads,hk,d", [(32, 4, 64), (8, 1, 128)], ids=str)
@pytest.mark.parametrize("n,length", [(1, 20000), (2, 9000), (4, 20000), (40, 6000), (130, 5000)], ids=str)
def test_long_contexts(hip, dtype, heads, hk, d, n, length):
    """Keys shared out to many workgroups, and the parts joined."""
    c = Paged(hip, dtype, [n], [length], heads, hk, d, 16, 4).upload()
    c.call()
    c.check()
    first = c.result()
    for _ in range(3):   # tickets are left ready, and nothing depends on who is last
        c.call()
        assert np.array_equal(first, c.result())


@TYPES
@pytest.mark.parametrize("heads,hk,d", [(32, 8, 128), (32, 8, 64), (40, 5, 64)], ids=str)
@pytest.mark.parametrize("known", [True, False], ids=["most rows known", "unknown"])
@pytest.mark.parametrize("n,lengths", [([60, 1, 1, 3], [2060, 1500, 300, 40]), ([1, 10, 1], [1900, 1510, 1]),
                                       ([1, 1, 33, 20], [700, 2600, 633, 2500])], ids=str)
def test_chunks_beside_decoded_tokens(hip, dtype, heads, hk, d, known, n, lengths):
    """Row tiles of which some waves have no rows, alone and joined from two to
    many workgroups' parts."""
    c = Paged(hip, dtype, n, lengths, heads, hk, d, 16, 31, max_rows=None if known else 0, pad=2).upload()
    c.call()
    c.check()
    first = c.result()
    c.call()
    assert np.array_equal(first, c.result())


@TYPES
def test_one_workspace_for_many_shapes(hip, dtype):
    shapes = [([1] * 40, [700 + 13 * i for i in range(40)]), ([200, 1], [3000, 5000]), ([1], [9000]),
              ([3, 3, 3], [2000, 2500, 100]), ([90], [4000]), ([1, 2], [6000, 10])]
    calls = [Paged(hip, dtype, n, length, 16, 4, 64, 16, 5 + i).upload() for i, (n, length) in enumerate(shapes)]
    ws = max((c.ws for c in calls), key=lambda w: w.nbytes)
    for _ in range(2):
        for c in calls:
            c.call(ws=ws)
    for c in calls:
        c.check()


@TYPES
def test_more_requests_than_threads(hip, dtype):
    r = np.random.default_rng(6)
    n = r.choice([0, 1, 1, 1, 2, 6], 700)
    c = Paged(hip, dtype, n, n + r.integers(0, 60, 700), 8, 2, 64, 16, 7, pad=3).upload()
    c.call()
    c.check()


@TYPES
@pytest.mark.parametrize("n", [1, 3, 40])
def test_rows_without_tokens(hip, dtype, n):
    """Lengths shorter than the rows: the first rows see nothing and give zeros."""
    c = Paged(hip, dtype, [n, 2, 1], [n, 2, 5], 8, 2, 64, 16, 8).upload()
    short = np.asarray([n // 2, 0, 5], np.int32)
    c.dl.upload(short)
    c.call()
    got = c.result()
    for b, (rows, length) in enumerate(zip([n, 2, 1], short)):
        k, v, _ = c.keys(b)
        a = c.start[b]
        want, tol = reference(held(c.q, dtype)[a:a + rows], k[:length], v[:length], length - rows, 64 ** -0.5, dtype)
        close(got[a:a + rows], want, tol)


@TYPES
@pytest.mark.parametrize("n,length", [(1, 77), (2, 77), (5, 200), (70, 100), (33, 530)], ids=str)
@pytest.mark.parametrize("fill", [np.nan, np.inf, -np.inf], ids=str)
@pytest.mark.parametrize("d", [64, 128])
def test_what_is_not_seen_counts_for_nothing(hip, dtype, n, length, fill, d):
    """Infinities and NaN behind the last token, in free pages, and in later
    tokens of the chunk."""
    c = Paged(hip, dtype, [n, 1], [length, 19], 8, 2, d, 16, 9, fill=fill).upload()
    c.call()
    c.check()
    if n > 1:
        t = length - 1   # the last row's own token: no other row sees it
        c.k[c.tables[0, t // 16], :, t % 16] = fill
        c.v[c.tables[0, t // 16], :, t % 16] = fill
        c.dk.upload(raw(c.k, dtype))
        c.dv.upload(raw(c.v, dtype))
        c.call()
        want, tol = c.want()
        got = c.result()
        rows = np.r_[0:n - 1, n:n + 1]
        close(got[rows], want[rows], tol[rows])
        assert not np.isfinite(got[n - 1]).any()


@TYPES
@pytest.mark.parametrize("n,length", [(1, 300), (4, 300), (60, 300)], ids=str)
def test_values_that_are_not_finite(hip, dtype, n, length):
    """A value's infinity reaches its element of the rows that see it."""
    c = Paged(hip, dtype, [n], [length], 8, 2, 64, 16, 10)
    at = {3: np.inf, 150: -np.inf, length - 1: np.nan, max(length - n // 2 - 1, 0): np.inf}
    for i, (t, x) in enumerate(at.items()):
        c.v[c.tables[0, t // 16], 1, t % 16, 7 + i] = x
    c.upload().call()
    got = c.result()
    want, tol = c.want()
    odd = np.zeros(want.shape, bool)
    for i, t in enumerate(at):
        odd[[j for j in range(n) if length - n + j >= t], 4:, 7 + i] = True
    close(got[~odd], want[~odd], tol[~odd])
    assert not np.isfinite(got[odd]).any()


@TYPES
def test_entries_that_are_no_page(hip, dtype):
    """Tokens in them do not exist, and nothing is read there."""
    for bad in (-1, 10 ** 9, -2 ** 31):
        c = Paged(hip, dtype, [1, 1, 1, 1], [200, 48, 16, 500], 8, 2, 64, 16, 11)
        c.tables[0, 3] = c.tables[0, 4] = c.tables[1, 0] = c.tables[3, 31] = c.tables[3, 10] = bad
        c.upload().call()
        c.check()
        c.tables[2, 0] = bad   # nothing is left: zeros
        c.dt.upload(c.tables)
        c.call()
        assert (c.result()[2] == 0).all()
    c = Paged(hip, dtype, [40], [200], 8, 2, 64, 16, 12)
    c.tables[0, 2] = c.pages
    c.upload().call()
    k, v, there = c.keys(0)
    gone = np.concatenate([k[:32], k[48:]]), np.concatenate([v[:32], v[48:]])
    want, tol = reference(held(c.q, dtype), *gone, 144, 64 ** -0.5, dtype)
    close(c.result(), want, tol)


@TYPES
def test_most_rows(hip, dtype):
    """Rows past max_rows are left as they were; 0: not known."""
    for max_rows in (1, 2, 30, 0):
        c = Paged(hip, dtype, [1, 33, 2, 1], [20, 50, 300, 129], 8, 2, 64, 16, 13, max_rows=max_rows).upload()
        c.call()
        c.check()


@TYPES
@pytest.mark.parametrize("heads,hk", [(40, 1), (17, 1), (64, 2)], ids=str)
@pytest.mark.parametrize("d", [64, 128])
def test_wide_groups(hip, dtype, heads, hk, d):
    """More query heads for a KV head than the small kernel's tiles take."""
    c = Paged(hip, dtype, [1, 1, 3], [5, 700, 90], heads, hk, d, 16, 14).upload()
    c.call()
    c.check()


@TYPES
@pytest.mark.parametrize("scale", [1e-3, 1.0, 4.0])
def test_scales(hip, dtype, scale):
    """Flat and very sharp weights."""
    for n in (1, 50):
        c = Paged(hip, dtype, [n, 1], [n + 90, 400], 8, 2, 64, 16, 15)
        c.scale = scale
        c.upload().call()
        c.check()


@TYPES
def test_rising_scores(hip, dtype):
    """Every block holds a larger score than all before it."""
    for n in (1, 40):
        c = Paged(hip, dtype, [n], [1500], 4, 2, 64, 16, 16)
        c.q[:] = np.abs(c.q)
        for t in range(1500):
            c.k[c.tables[0, t // 16], :, t % 16] = t / 400
        c.upload().call()
        c.check()


def test_offsets_past_32_bits(hip):
    """Pages more than 4 GiB behind the cache's first byte."""
    page, hk, d = 256, 8, 128
    page_bytes = hk * page * d * 2
    pages = (5 << 30) // page_bytes
    c = Paged(hip, 5, [1, 20], [400, 300], 16, hk, d, page, 17)
    far = np.arange(pages - c.pages, pages)
    small = c.upload()
    big = {}
    for name, src in (("k", c.k), ("v", c.v)):
        big[name] = hip.DeviceBuffer(pages * page_bytes)
        host = raw(src, 5)
        hip.check(hip.open_library().vm_hip_memcpy_h2d(big[name].addr + int(far[0]) * page_bytes, host.ctypes.data,
                                                       host.nbytes, None))
    c.dt.upload(np.where(c.tables >= 0, c.tables + far[0], -1).astype(np.int32))
    c.cache = hip.KvPaged(big["k"].addr, big["v"].addr, 5, pages, page, hk, d)
    small.call()
    c.check()


# ---- whole prompts, packed

class Packed:
    def __init__(self, hip, dtype, n, heads, hk, d, seed, pad=0, apart=False):
        r = np.random.default_rng(seed)
        self.hip, self.dtype, self.n, self.heads, self.hk, self.d = hip, dtype, np.asarray(n), heads, hk, d
        self.rows = int(self.n.sum()) + pad
        self.qkv = r.standard_normal((self.rows, heads + 2 * hk, d))
        self.start = np.concatenate([[0], np.cumsum(self.n)]).astype(np.int32)
        self.apart = apart   # q, k and v in buffers of their own, rows further apart than they are long
        self.scale = 0.0

    def upload(self):
        dev = self.hip.DeviceBuffer.from_array
        h, hk, d, size = self.heads, self.hk, self.d, SIZE[self.dtype]
        if self.apart:
            gaps = (8, 16, 40)
            parts = (self.qkv[:, :h], self.qkv[:, h:h + hk], self.qkv[:, h + hk:])
            self.buf = [dev(raw(np.pad(x.reshape(self.rows, -1), ((0, 0), (0, gap)), constant_values=np.nan), self.dtype))
                        for x, gap in zip(parts, gaps)]
            self.at = [b.addr for b in self.buf]
            self.strides = [h * d + 8, hk * d + 16, hk * d + 40]
        else:
            self.buf = [dev(raw(self.qkv, self.dtype))]
            self.at = [self.buf[0].addr + x * d * size for x in (0, h, h + hk)]
            self.strides = [(h + 2 * hk) * d] * 3
        self.ds = dev(self.start)
        self.out = dev(np.full(self.rows * h * d * size, 0x5b, np.uint8))
        self.ws = dev(np.zeros(max(1, self.hip.attention_packed_workspace_bytes(len(self.n), self.rows, h, hk, d)), np.uint8))
        return self

    def call(self, stream=None):
        self.hip.attention_packed(*self.at, self.out.addr, self.dtype, *self.strides, len(self.n), self.rows, self.heads,
                                  self.hk, self.d, self.ds.addr, self.scale, self.ws.addr, self.ws.nbytes, stream)

    def result(self):
        return back(self.out, (self.rows, self.heads, self.d), self.dtype)

    def check(self, rows=None):
        got, x = self.result(), held(self.qkv, self.dtype)
        for a, b in zip(self.start[:-1], self.start[1:]):
            if a == b:
                continue
            q, k, v = x[a:b, :self.heads], x[a:b, self.heads:self.heads + self.hk], x[a:b, self.heads + self.hk:]
            want, tol = reference(q, k, v, 0, self.scale if self.scale > 0 else self.d ** -0.5, self.dtype)
            at = slice(0, b - a) if rows is None else rows
            close(got[a:b][at], want[at], tol[at])
        left = self.out.download(np.uint8, (self.rows, self.heads * self.d * SIZE[self.dtype]))[self.start[-1]:]
        assert (left == 0x5b).all(), "rows behind the last one were written"


@TYPES
@HEADS
@pytest.mark.parametrize("n", [[1], [2], [31], [32, 1], [33, 64], [65, 0, 3], [127, 128, 129], [1] * 9 + [200],
                               [0, 0, 5, 0], [513]], ids=str)
@pytest.mark.parametrize("apart", [False, True], ids=["fused", "apart"])
def test_packed(hip, dtype, heads, hk, d, n, apart):
    c = Packed(hip, dtype, n, heads, hk, d, 20, pad=4, apart=apart).upload()
    c.call()
    c.check()


@TYPES
@pytest.mark.parametrize("d", [64, 128])
def test_packed_longer(hip, dtype, d):
    c = Packed(hip, dtype, [1500, 700], 4, 2, d, 21).upload()
    c.call()
    c.check()
    first = c.result()
    c.call()
    assert np.array_equal(first, c.result())


@TYPES
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("odd", [np.nan, np.inf, -np.inf], ids=str)
def test_packed_later_rows_count_for_nothing(hip, dtype, d, odd):
    """Infinities and NaN in a later row and in the next prompt."""
    for n, t in [(40, 20), (200, 130), (300, 299), (70, 1)]:
        c = Packed(hip, dtype, [n, 5], 8, 2, d, 22)
        c.qkv[t:n + 5] = odd
        c.upload().call()
        got, x = c.result(), held(c.qkv, dtype)
        want, tol = reference(x[:t, :8], x[:t, 8:10], x[:t, 10:], 0, d ** -0.5, dtype)
        close(got[:t], want, tol)
        assert not np.isfinite(got[t:n]).any()


@pytest.mark.parametrize("dtype,heads,hk,d,n", [(4, 64, 8, 64, [2300, 77]), (5, 64, 8, 64, [2100]), (5, 64, 8, 128, [900, 700]),
                                                (4, 48, 16, 64, [1400]), (0, 40, 5, 64, [1300, 1]), (0, 16, 16, 128, [700]),
                                                (4, 32, 32, 128, [1000, 600])], ids=str)
def test_packed_large(hip, dtype, heads, hk, d, n):
    """More row tiles than workgroups run at once, and both tile sizes, by some of the heads."""
    c = Packed(hip, dtype, n, heads, hk, d, 30).upload()
    c.call()
    got, x = c.result(), held(c.qkv, dtype)
    g = heads // hk
    for a, b in zip(c.start[:-1], c.start[1:]):
        for h in (0, hk // 2, hk - 1):
            u = [h * g, h * g + g - 1]
            want, tol = reference(x[a:b, u], x[a:b, [heads + h]], x[a:b, [heads + hk + h]], 0, d ** -0.5, dtype)
            close(got[a:b, u], want, tol)
    first = got
    c.call()
    assert np.array_equal(first, c.result())


@pytest.mark.parametrize("dtype", [0, 5], ids=["f32", "bf16"])
def test_chunks_large(hip, dtype):
    """Chunks whose keys several workgroups share, and chunks that have one each."""
    for n, lengths, heads, hk, d in [([600, 90, 300], [2600, 4000, 300], 16, 4, 64), ([300] * 5, [500] * 5, 32, 8, 128)]:
        c = Paged(hip, dtype, n, lengths, heads, hk, d, 32, 31).upload()
        for _ in range(2):
            c.call()
        c.check()


@TYPES
def test_packed_many_requests(hip, dtype):
    r = np.random.default_rng(23)
    c = Packed(hip, dtype, r.choice([0, 1, 2, 3, 17], 900), 6, 2, 64, 24, pad=1).upload()
    c.call()
    c.check()


def test_row_starts_that_are_wrong_stay_inside(hip):
    """Falling, negative and too large offsets: other rows, never another's memory."""
    for start in ([5, 3, 9, 40], [-4, 10, 10 ** 9, 20], [0, 2 ** 31 - 1, -2 ** 31, 30]):
        c = Packed(hip, 4, [10, 10, 10], 4, 2, 64, 25).upload()
        c.ds.upload(np.asarray(start, np.int32))
        c.call()
        p = Paged(hip, 4, [10, 10, 10], [30, 40, 50], 4, 2, 64, 16, 26).upload()
        p.ds.upload(np.asarray(start, np.int32))
        p.dl.upload(np.asarray([2 ** 31 - 1, -5, 33], np.int32))
        p.call()
        hip.synchronize()


def test_streams_and_graphs(hip):
    """Two streams at once with a workspace each, and a captured call replayed
    with other lengths, rows and tables."""
    a = Paged(hip, 5, [1, 60], [3000, 900], 16, 4, 128, 16, 27).upload()
    b = Paged(hip, 5, [1, 1, 1], [2000, 4000, 100], 16, 4, 128, 32, 28).upload()
    s, t = hip.Stream(), hip.Stream()
    for _ in range(5):
        a.call(stream=s)
        b.call(stream=t)
    s.synchronize()
    t.synchronize()
    a.check()
    b.check()
    c = Paged(hip, 4, [4, 30, 1], [200, 800, 5000], 16, 4, 64, 16, 29, max_rows=30).upload()
    c.call(stream=s)
    s.synchronize()
    graph = hip.Graph(s)
    graph.begin()
    c.call(stream=s)
    graph.end()
    for n, lengths in [([4, 30, 1], [200, 800, 5000]), ([1, 1, 1], [17, 800, 4999]), ([0, 5, 30], [3, 16, 300])]:
        c.n, c.lengths = np.asarray(n), np.asarray(lengths)
        c.start = np.concatenate([[0], np.cumsum(n)]).astype(np.int32)
        c.ds.upload(c.start)
        c.dl.upload(c.lengths.astype(np.int32))
        c.out.upload(np.full(c.out.nbytes, 0x5b, np.uint8))
        graph.launch()
        s.synchronize()
        c.check()
