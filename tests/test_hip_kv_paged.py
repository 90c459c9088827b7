"""A step's plan, pages given back, rotation tables, and norm, rotation and
append on the GPU, against plain Python and numpy in 64 bits.

Whole numbers are equal.  Tables: cosines and sines of 64-bit angles rounded
once, half a step of fp32 and 2^-40.  Append: the norm's factor is off by at
most 12 2^-24 (sums of D / 16 squares in a lane and of 16 lanes, mean, eps, root
and reciprocal), its two products by 2 more, the rotation's sum by 3 of |a cos| +
|b sin|, and the result is rounded by half a step of its type; rows that are
only moved keep their bits."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

TORCH = {0: torch.float32, 4: torch.float16, 5: torch.bfloat16}
STEP = {0: 2.0 ** -24, 4: 2.0 ** -11, 5: 2.0 ** -8}
TYPES = pytest.mark.parametrize("dtype", [0, 4, 5], ids=["f32", "f16", "bf16"])


def i32(hip, a):
    return hip.DeviceBuffer.from_array(np.asarray(a, np.int32))


# ---- plan and release

class Pool:
    """Requests, their tables and a pool of pages, on the host and the GPU."""

    def __init__(self, hip, lengths, page, pages, max_pages, seed, rows):
        r = np.random.default_rng(seed)
        self.hip, self.page, self.pages, self.max_pages, self.rows = hip, page, pages, max_pages, rows
        self.batch = len(lengths)
        self.lengths = np.asarray(lengths, np.int64)
        order = [int(x) for x in r.permutation(pages)]
        self.tables = np.full((self.batch, max_pages), -1, np.int64)
        for b, n in enumerate(self.lengths):
            for j in range(min(max(-(-int(n) // page), 0), max_pages)):
                self.tables[b, j] = order.pop()
        self.free = order
        self.dl, self.dt = i32(hip, self.lengths), i32(hip, self.tables)
        self.df = i32(hip, self.free + [-9] * (pages - len(self.free)))
        self.dn = i32(hip, [len(self.free)])
        self.dc, self.dstart = i32(hip, np.zeros(self.batch)), i32(hip, np.zeros(self.batch + 1))
        self.dp, self.dslots = i32(hip, np.zeros(max(1, rows))), i32(hip, np.zeros(max(1, rows)))
        self.ws = hip.DeviceBuffer.from_array(np.zeros(hip.kv_paged_plan_workspace_bytes(self.batch, rows), np.uint8))
        self.plan = hip.PagePlan(self.batch, rows, max_pages, pages, page, self.dl.addr, self.dc.addr, self.df.addr,
                                 self.dn.addr, self.dt.addr, self.dstart.addr, self.dl.addr, self.dn.addr, self.dp.addr,
                                 self.dslots.addr)

    def launch(self, stream=None):
        self.hip.kv_paged_plan(self.plan, self.ws.addr, self.ws.nbytes, stream)

    def expect(self, counts):
        """What the step leaves, on the host's copies."""
        page = self.page
        used, short_rows, short_pages = 0, False, False
        start, positions, slots = [0], [], []
        for b, c in enumerate(int(x) for x in counts):
            n = int(self.lengths[b])
            took = 0
            if n >= 0 and c >= 0 and n + c <= self.max_pages * page:
                used += c
                short_rows |= used > self.rows
                if not short_rows:
                    held, want = -(-n // page), -(-(n + c) // page) - -(-n // page)
                    if c == 0:
                        want = 0
                    short_pages |= want > 0 and want > len(self.free)
                    if want == 0 or not short_pages:
                        took = c
                        for j in range(want):
                            self.tables[b, held + j] = self.free.pop()
                        for p in range(n, n + c):
                            positions.append(p)
                            id = int(self.tables[b, p // page])
                            slots.append(id * page + p % page if 0 <= id < self.pages else -1)
            start.append(start[-1] + took)
            self.lengths[b] += took
        pad = [-1] * (self.rows - len(positions))
        return start, positions + pad, slots + pad

    def check(self, want):
        start, positions, slots = want
        got = lambda buf, n: buf.download(np.int32, (n,))  # noqa: E731
        assert np.array_equal(got(self.dstart, self.batch + 1), start)
        assert np.array_equal(got(self.dp, self.rows), positions)
        assert np.array_equal(got(self.dslots, self.rows), slots)
        self.check_state()

    def check_state(self):
        assert np.array_equal(self.dl.download(np.int32, (self.batch,)), self.lengths)
        assert np.array_equal(self.dt.download(np.int32, self.tables.shape), self.tables)
        n = int(self.dn.download(np.int32, (1,))[0])
        assert n == len(self.free)
        assert np.array_equal(self.df.download(np.int32, (self.pages,))[:n], self.free)

    def step(self, counts):
        self.dc.upload(np.asarray(counts, np.int32))
        want = self.expect(counts)
        self.launch()
        self.check(want)

    def release(self, finished):
        f = i32(self.hip, finished)
        self.hip.kv_paged_release(self.batch, self.max_pages, self.pages, self.page, f.addr, self.dl.addr, self.dt.addr,
                                  self.df.addr, self.dn.addr)
        for b in np.flatnonzero(finished):
            for j in range(-(-int(self.lengths[b]) // self.page)):
                self.free.append(int(self.tables[b, j]))
                self.tables[b, j] = -1
            self.lengths[b] = 0
        self.check_state()


@pytest.mark.parametrize("batch", [1, 2, 64, 255, 256, 257, 700, 1024, 1025, 2048])
@pytest.mark.parametrize("page", [16, 256])
def test_plan(hip, batch, page):
    """Steps of tokens and chunks, in place; pages run out on the way."""
    r = np.random.default_rng(batch)
    lengths = r.integers(0, 200, batch)
    need = int((-(-lengths // page)).sum())
    p = Pool(hip, lengths, page, need + 5 + batch // 3, 400 // page + 2, 1, 3000)
    for i in range(4):
        p.step(r.integers(0, 3, batch))
        p.step(r.choice([0, 0, 1, 17, 60], batch))
        p.release(r.random(batch) < 0.2)


def test_plan_corners(hip):
    p = Pool(hip, [0, 16, 15, 31, 5, 0, 47, 0], 16, 20, 3, 2, 40)
    p.step([0] * 8)
    p.step([1, 1, 1, 1, 1, 0, 1, 0])                  # new pages at the borders
    p.step([49, 100, 2 ** 31 - 1, 1, -3, 2, 0, -1])   # longer than their tables, or not valid: the others go on
    p.step([20, 0, 0, 0, 21, 1, 0, 0])                # more rows than fit: the later ones wait
    p.step([0, 0, 0, 0, 20, 1, 0, 0])
    p.dl.upload(np.asarray([-5, -2 ** 31, 2 ** 31 - 1, 48, 3, 2, 1, 0], np.int32))
    p.lengths[:] = [-5, -2 ** 31, 2 ** 31 - 1, 48, 3, 2, 1, 0]
    p.tables[4:7, 0] = [3, 20, -1]                    # entries that are no page: no slots
    p.dt.upload(p.tables.astype(np.int32))
    p.step([1, 1, 1, 1, 1, 1, 1, 0])


def test_plan_without_pages_or_rows(hip):
    p = Pool(hip, [10, 16, 3], 16, 2 + 1, 4, 3, 8)
    p.step([1, 1, 1])      # the second one waits, the third goes on
    p = Pool(hip, [10, 0, 3], 16, 4, 4, 3, 0)
    p.step([0, 0, 0])
    p.step([1, 0, 0])
    p = Pool(hip, [5], 16, 3, 4, 4, 8)
    for count, left in ((-4, 0), (99, 3)):   # a count that is wrong is held to the pool
        p.dn.upload(np.asarray([count], np.int32))
        p.dc.upload(np.asarray([8], np.int32))
        p.dl.upload(np.asarray([5], np.int32))
        p.launch()
        assert p.dl.download(np.int32, (1,))[0] == 13
        assert p.dn.download(np.int32, (1,))[0] == left


def test_plan_many_rows(hip):
    """Several workgroups, in place, the same step over and over."""
    for total in (1024, 1025, 5000, 70000):
        p = Pool(hip, [100] * 30, 32, 6000, 200, 4, total)
        for _ in range(2):
            p.step([total // 30] * 29 + [total // 30 // 2])
            p.release([1] * 30)
            p.lengths[:] = 0


def test_plan_elsewhere(hip):
    """Results beside the inputs leave these as they were."""
    p = Pool(hip, [7, 30, 0], 16, 9, 5, 5, 10)
    out_l, out_n = i32(hip, [0, 0, 0]), i32(hip, [0])
    p.plan.lengths_out, p.plan.free_count_out = out_l.addr, out_n.addr
    p.dc.upload(np.asarray([1, 3, 4], np.int32))
    before, free = p.lengths.copy(), len(p.free)
    want = p.expect([1, 3, 4])
    for _ in range(2):
        p.launch()
    assert np.array_equal(out_l.download(np.int32, (3,)), p.lengths)
    assert out_n.download(np.int32, (1,))[0] == len(p.free)
    assert np.array_equal(p.dl.download(np.int32, (3,)), before)
    assert p.dn.download(np.int32, (1,))[0] == free
    assert np.array_equal(p.dslots.download(np.int32, (10,)), want[2])


def test_plan_captured(hip):
    """A captured plan goes on with each replay."""
    s = hip.Stream()
    p = Pool(hip, [3] * 50, 16, 300, 30, 6, 2500)
    p.dc.upload(np.full(50, 1, np.int32))
    g = hip.Graph(s)
    g.begin()
    p.launch(s)
    g.end()
    for c in (1, 40, 0, 7, 1):
        p.dc.upload(np.full(50, c, np.int32))
        want = p.expect([c] * 50)
        g.launch()
        s.synchronize()
        p.check(want)


def test_release_into_a_full_pool(hip):
    """A pool never holds more than its pages."""
    p = Pool(hip, [40, 40], 16, 6, 3, 7, 4)
    p.dn.upload(np.asarray([4], np.int32))
    f = i32(hip, [1, 1])
    hip.kv_paged_release(2, 3, 6, 16, f.addr, p.dl.addr, p.dt.addr, p.df.addr, p.dn.addr)
    assert p.dn.download(np.int32, (1,))[0] == 6
    assert np.array_equal(p.df.download(np.int32, (6,))[4:], p.tables[0, :2])


# ---- rotation tables

def frequencies(dim, theta, kind, factor, low, high, original):
    f = [theta ** (-2.0 * i / dim) for i in range(dim // 2)]
    if kind == 1:
        f = [x / factor for x in f]
    if kind == 2:
        out = []
        for x in f:
            turns = original * x / (2 * math.pi)
            keep = min(1.0, max(0.0, (turns - low) / (high - low)))
            out.append(x * keep + x / factor * (1 - keep))
        f = out
    if kind == 3:
        at = lambda turns: dim * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(theta))  # noqa: E731
        a, b = max(math.floor(at(high)), 0), min(math.ceil(at(low)), dim - 1)
        f = [x / factor * r + x * (1 - r) for x, r in ((x, min(1.0, max(0.0, (i - a) / max(b - a, 0.001)))) for i, x in enumerate(f))]
    return np.asarray(f)


@pytest.mark.parametrize("kind", [0, 1, 2, 3])
@pytest.mark.parametrize("first,rows,dim", [(0, 1, 64), (0, 7, 2), (5, 100, 18), (0, 2000, 64), (131000, 72, 128),
                                            (2 ** 31 - 3, 3, 128), (7, 40000, 126)], ids=str)
def test_rope_tables(hip, kind, first, rows, dim):
    cos, sin = (hip.DeviceBuffer(rows * dim // 2 * 4) for _ in "cs")
    scaling = hip.RopeScaling(kind, 8.0, 1.0, 32.0 if kind == 3 else 4.0, 4096.0, 1.25)
    hip.rope_tables(cos.addr, sin.addr, first, rows, dim, 10000.0, scaling)
    f = frequencies(dim, 10000.0, kind, 8.0, 1.0, 32.0 if kind == 3 else 4.0, 4096.0)
    angle = (first + np.arange(rows, dtype=np.float64))[:, None] * f
    # the angle itself is rounded to 64 bits, and the frequency by a few steps of them
    slack = 2.0 ** -40 + 1.25 * np.abs(angle) * 2.0 ** -50
    for buf, want in ((cos, 1.25 * np.cos(angle)), (sin, 1.25 * np.sin(angle))):
        got = buf.download(np.float32, angle.shape).astype(np.float64)
        assert (np.abs(got - want) <= np.abs(want) * 2.0 ** -24 + slack).all()
    if kind == 0:
        hip.rope_tables(cos.addr, sin.addr, first, rows, dim, 10000.0)   # the same without a struct
        got = cos.download(np.float32, angle.shape).astype(np.float64)
        assert (np.abs(got - np.cos(angle)) <= np.abs(np.cos(angle)) * 2.0 ** -24 + slack).all()


# ---- append

def bits(x, dtype):
    t = torch.from_numpy(np.ascontiguousarray(x, np.float32)).to(TORCH[dtype])
    return t.numpy() if dtype == 0 else t.view(torch.int16).numpy()


def numbers(a, dtype):
    return a.astype(np.float64) if dtype == 0 else torch.from_numpy(a).view(TORCH[dtype]).double().numpy()


class Rows:
    """A projection's rows and what they are normed and rotated with."""

    def __init__(self, hip, dtype, rows, heads, hk, d, rotary, pairs, norm, seed, table_rows=300):
        r = np.random.default_rng(seed)
        self.hip, self.dtype, self.rows, self.heads, self.hk, self.d = hip, dtype, rows, heads, hk, d
        self.rotary, self.pairs, self.norm, self.table_rows = rotary, pairs, norm, table_rows
        self.x = r.standard_normal((rows, heads + 2 * hk, d)) * 2
        self.positions = r.integers(0, table_rows + 20, rows)
        self.wq, self.wk = (r.uniform(0.5, 1.5, d).astype(np.float32) for _ in "qk")
        angle = np.arange(table_rows)[:, None] * 10000.0 ** (-np.arange(max(rotary // 2, 1)) / max(rotary // 2, 1))
        self.cos, self.sin = np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)
        dev = hip.DeviceBuffer.from_array
        self.dx, self.dp = dev(bits(self.x, dtype)), i32(hip, self.positions)
        self.dw, self.dt = [dev(self.wq), dev(self.wk)], [dev(self.cos), dev(self.sin)]
        self.rope = hip.Rope(self.dt[0].addr, self.dt[1].addr, table_rows, rotary, int(pairs))
        self.head_norm = hip.QkNorm(self.dw[0].addr, self.dw[1].addr, 1e-5) if norm else None
        self.size = 4 if dtype == 0 else 2
        self.q = dev(np.full(rows * heads * d * self.size, 0x5b, np.uint8))

    def want(self):
        """(query and key heads, tolerances) [rows, heads + hk, d]."""
        x = numbers(bits(self.x, self.dtype), self.dtype)[:, :self.heads + self.hk]
        u = 3.0
        if self.norm:
            w = np.concatenate([np.tile(self.wq, (self.heads, 1)), np.tile(self.wk, (self.hk, 1))]).astype(np.float64)
            x = x / np.sqrt((x * x).mean(-1, keepdims=True) + np.float64(np.float32(1e-5))) * w
            u += 14.0
        h = self.rotary // 2
        i = np.arange(h) * (2 if self.pairs else 1)
        j = i + (1 if self.pairs else h)
        at = np.minimum(self.positions, self.table_rows - 1)
        y, size = x.copy(), np.abs(x) * (1 if self.norm else 0)
        if h:
            c, s = (t[at].astype(np.float64)[:, None] for t in (self.cos, self.sin))
            y[..., i], y[..., j] = x[..., i] * c - x[..., j] * s, x[..., j] * c + x[..., i] * s
            size[..., i] = np.abs(x[..., i] * c) + np.abs(x[..., j] * s)
            size[..., j] = np.abs(x[..., j] * c) + np.abs(x[..., i] * s)
        return y, u * 2.0 ** -24 * size + STEP[self.dtype] * np.abs(y) + (2.0 ** -25 if self.dtype == 4 else 1e-37)

    def queries(self):
        kind = np.float32 if self.dtype == 0 else np.int16
        return self.q.download(kind, (self.rows, self.heads, self.d))


def near(got, want, tol):
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), f"{bad.sum()} of {bad.size}, first at {np.argwhere(bad)[0]}: {got[bad][0]!r}, not {want[bad][0]!r} +- {tol[bad][0]!r}"


SHAPES = pytest.mark.parametrize("rows,heads,hk,d", [(1, 32, 4, 64), (7, 15, 5, 64), (33, 4, 4, 128), (3, 64, 8, 128),
                                                     (1500, 3, 1, 64), (5001, 3, 1, 128)], ids=str)


@TYPES
@SHAPES
@pytest.mark.parametrize("rotary", ["all", "half", "odd", "two", "none"])
@pytest.mark.parametrize("pairs", [False, True], ids=["halves", "pairs"])
@pytest.mark.parametrize("norm", [False, True], ids=["bare", "norm"])
def test_append(hip, dtype, rows, heads, hk, d, rotary, pairs, norm):
    rotary = {"all": d, "half": d // 2, "odd": d // 4 + 2, "two": 2, "none": 0}[rotary]
    x = Rows(hip, dtype, rows, heads, hk, d, rotary, pairs, norm, 1)
    r = np.random.default_rng(2)
    page = 16
    pages = rows // page + 3
    slots = r.permutation(pages * page)[:rows]
    padding = np.zeros(rows, bool)
    if rows > 1:
        for at, bad in zip(r.choice(rows, min(rows - 1, 4), replace=False), (-1, pages * page, 2 ** 31 - 1, -2 ** 31)):
            slots[at] = bad
            padding[at] = True
        at = int(np.flatnonzero(~padding)[0])
        if (~padding).sum() > 1:
            x.positions[at] = -1
            x.dp.upload(x.positions.astype(np.int32))
            padding[at] = True
    dev = hip.DeviceBuffer.from_array
    nbytes = pages * hk * page * d * x.size
    dk, dv = dev(np.full(nbytes, 0x31, np.uint8)), dev(np.full(nbytes, 0x32, np.uint8))
    cache = hip.KvPaged(dk.addr, dv.addr, dtype, pages, page, hk, d)
    ds = i32(hip, slots)
    hip.kv_paged_append(cache, x.dx.addr, rows, heads, x.head_norm, x.rope, x.dp.addr, ds.addr, x.q.addr)
    want, tol = x.want()
    q = x.queries()
    near(numbers(q[~padding], dtype), want[~padding, :heads], tol[~padding, :heads])
    assert (np.ascontiguousarray(q[padding]).view(np.uint8) == 0x5b).all()
    kind = np.float32 if dtype == 0 else np.int16
    k, v = (b.download(kind, (pages, hk, page, d)).transpose(0, 2, 1, 3).reshape(pages * page, hk, d) for b in (dk, dv))
    at = slots[~padding]
    near(numbers(np.ascontiguousarray(k[at]), dtype), want[~padding, heads:], tol[~padding, heads:])
    whole = bits(x.x, dtype)
    assert np.array_equal(v[at], whole[~padding, heads + hk:])
    rest = np.ones(pages * page, bool)
    rest[at] = False
    assert (np.ascontiguousarray(k[rest]).view(np.uint8) == 0x31).all()
    assert (np.ascontiguousarray(v[rest]).view(np.uint8) == 0x32).all()
    if not norm and rotary < d:   # what is not rotated keeps its bits
        assert np.array_equal(q[~padding][..., rotary:], whole[~padding, :heads, rotary:])
    # without a cache
    k_out = dev(np.full(rows * hk * d * x.size, 0x5b, np.uint8))
    x.q.upload(np.full(x.q.nbytes, 0x5b, np.uint8))
    hip.qk_norm_rope(x.dx.addr, dtype, rows, heads, hk, d, x.head_norm, x.rope, x.dp.addr, x.q.addr, k_out.addr)
    there = x.positions >= 0
    assert np.array_equal(x.queries()[~padding], q[~padding])
    near(numbers(x.queries()[there], dtype), want[there, :heads], tol[there, :heads])
    got = k_out.download(kind, (rows, hk, d))
    near(numbers(got[there], dtype), want[there, heads:], tol[there, heads:])
    assert (np.ascontiguousarray(got[~there]).view(np.uint8) == 0x5b).all()


@TYPES
def test_append_without_rope(hip, dtype):
    x = Rows(hip, dtype, 5, 4, 2, 64, 0, False, True, 3)
    k_out = hip.DeviceBuffer(5 * 2 * 64 * x.size)
    hip.qk_norm_rope(x.dx.addr, dtype, 5, 4, 2, 64, x.head_norm, None, x.dp.addr, x.q.addr, k_out.addr)
    want, tol = x.want()
    near(numbers(x.queries(), dtype), want[:, :4], tol[:, :4])


@TYPES
@pytest.mark.parametrize("pairs", [False, True])
def test_append_keeps_what_is_not_finite_apart(hip, dtype, pairs):
    """An infinity or NaN reaches its own pair, or with a norm its head, only."""
    for norm in (False, True):
        x = Rows(hip, dtype, 3, 4, 2, 64, 32, pairs, norm, 4)
        want, tol = x.want()
        x.x[1, 2, 40], x.x[2, 5, 3], x.x[0, 0, 6] = np.inf, np.nan, -np.inf
        x.dx.upload(bits(x.x, dtype))
        k_out = hip.DeviceBuffer(3 * 2 * 64 * x.size)
        hip.qk_norm_rope(x.dx.addr, dtype, 3, 4, 2, 64, x.head_norm, x.rope, x.dp.addr, x.q.addr, k_out.addr)
        kind = np.float32 if dtype == 0 else np.int16
        got = np.concatenate([numbers(x.queries(), dtype), numbers(k_out.download(kind, (3, 2, 64)), dtype)], 1)
        odd = np.zeros(got.shape, bool)
        for row, head, e in [(1, 2, 40), (2, 5, 3), (0, 0, 6)]:
            if norm:
                odd[row, head] = True
            else:
                odd[row, head, e] = True
                if e < 32:
                    odd[row, head, (e ^ 1) if pairs else (e + 16) % 32] = True
        near(got[~odd], want[~odd], tol[~odd])
