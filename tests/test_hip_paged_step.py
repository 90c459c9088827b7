"""Steps of a server over a pool of cache pages as they are run: rotation
tables, then for every step the plan, norm, rotation and append of a
projection's rows, and attention over the pages, captured once and replayed with
requests that come, wait for pages, grow and end.  Every operator's output is
checked against its formula on the values that the GPU handed it; and prompts
without a cache give what the pages give."""
from __future__ import annotations

import numpy as np
import pytest

from test_hip_attention_paged import close, held, raw, back, reference
from test_hip_kv_paged import Pool, i32, near, numbers

pytestmark = pytest.mark.gpu

HEADS, HK, D, PAGE, PAGES, WIDTH, ROWS, ROTARY = 8, 2, 64, 16, 40, 12, 96, 48
STEP = {0: 2.0 ** -24, 4: 2.0 ** -11, 5: 2.0 ** -8}


class Server:
    def __init__(self, hip, dtype, batch, pairs):
        self.hip, self.dtype, self.pairs = hip, dtype, pairs
        r = np.random.default_rng(3)
        dev = hip.DeviceBuffer.from_array
        self.pool = Pool(hip, [0] * batch, PAGE, PAGES, WIDTH, 4, ROWS)
        self.size = 4 if dtype == 0 else 2
        shape = (PAGES, HK, PAGE, D)
        self.dk, self.dv = (dev(np.full(int(np.prod(shape)) * self.size, 0xff, np.uint8)) for _ in "kv")   # NaN
        self.cache = hip.KvPaged(self.dk.addr, self.dv.addr, dtype, PAGES, PAGE, HK, D)
        self.cos, self.sin = hip.DeviceBuffer(WIDTH * PAGE * ROTARY * 2), hip.DeviceBuffer(WIDTH * PAGE * ROTARY * 2)
        scaling = hip.RopeScaling(hip.ROPE_RAMP, 4.0, 1.0, 32.0, 64.0, 1.1)
        hip.rope_tables(self.cos.addr, self.sin.addr, 0, WIDTH * PAGE, ROTARY, 10000.0, scaling)
        self.rope = hip.Rope(self.cos.addr, self.sin.addr, WIDTH * PAGE, ROTARY, int(pairs))
        self.wq, self.wk = (r.uniform(0.5, 1.5, D).astype(np.float32) for _ in "qk")
        self.dwq, self.dwk = dev(self.wq), dev(self.wk)
        self.norm = hip.QkNorm(self.dwq.addr, self.dwk.addr, 1e-5)
        self.qkv = dev(np.zeros(ROWS * (HEADS + 2 * HK) * D * self.size, np.uint8))
        self.q = dev(np.zeros(ROWS * HEADS * D * self.size, np.uint8))
        self.out = dev(np.zeros(ROWS * HEADS * D * self.size, np.uint8))
        nbytes = hip.attention_paged_workspace_bytes(batch, ROWS, 0, HEADS, HK, D, WIDTH * PAGE)
        self.ws = dev(np.zeros(nbytes, np.uint8))

    def launch(self, stream):
        p, hip = self.pool, self.hip
        p.launch(stream)
        hip.kv_paged_append(self.cache, self.qkv.addr, ROWS, HEADS, self.norm, self.rope, p.dp.addr, p.dslots.addr,
                            self.q.addr, stream)
        hip.attention_paged(self.cache, p.dt.addr, WIDTH, self.q.addr, self.out.addr, p.batch, ROWS, 0, HEADS,
                            p.dstart.addr, p.dl.addr, 0.0, self.ws.addr, self.ws.nbytes, stream)

    def stored(self, buf):
        """The cache [slots, hk, D]."""
        return back(buf, (PAGES, HK, PAGE, D), self.dtype).transpose(0, 2, 1, 3).reshape(PAGES * PAGE, HK, D)

    def rotated(self, x, positions):
        """(normed and rotated heads in 64 bits, tolerances) of x [rows, HEADS + HK, D], as the append's own test has them."""
        w = np.concatenate([np.tile(self.wq, (HEADS, 1)), np.tile(self.wk, (HK, 1))]).astype(np.float64)
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + np.float64(np.float32(1e-5))) * w
        h = ROTARY // 2
        i = np.arange(h) * (2 if self.pairs else 1)
        j = i + (1 if self.pairs else h)
        tables = [t.download(np.float32, (WIDTH * PAGE, h)).astype(np.float64)[positions][:, None] for t in (self.cos, self.sin)]
        y, size = x.copy(), np.abs(x)
        c, s = tables
        y[..., i], y[..., j] = x[..., i] * c - x[..., j] * s, x[..., j] * c + x[..., i] * s
        size[..., i] = np.abs(x[..., i] * c) + np.abs(x[..., j] * s)
        size[..., j] = np.abs(x[..., j] * c) + np.abs(x[..., i] * s)
        return y, 17 * 2.0 ** -24 * size + STEP[self.dtype] * np.abs(y) + (2.0 ** -25 if self.dtype == 4 else 1e-37)

    def check(self, want, x):
        start, positions, slots = want
        self.pool.check(want)
        rows = start[-1]
        if rows == 0:
            return
        x = held(x[:rows], self.dtype)
        positions, slots = np.asarray(positions[:rows]), np.asarray(slots[:rows])
        y, tol = self.rotated(x[:, :HEADS + HK], positions)
        q = back(self.q, (ROWS, HEADS, D), self.dtype)[:rows]
        near(q, y[:, :HEADS], tol[:, :HEADS])
        k, v = self.stored(self.dk), self.stored(self.dv)
        near(k[slots], y[:, HEADS:], tol[:, HEADS:])
        assert np.array_equal(v[slots], x[:, HEADS + HK:])
        out = back(self.out, (ROWS, HEADS, D), self.dtype)
        for b in range(self.pool.batch):
            a, e = start[b], start[b + 1]
            if a == e:
                continue
            t = np.arange(int(self.pool.lengths[b]))
            at = self.pool.tables[b, t // PAGE] * PAGE + t % PAGE
            close(out[a:e], *reference(q[a:e], k[at], v[at], len(t) - (e - a), D ** -0.5, self.dtype))


@pytest.mark.parametrize("dtype", [0, 4, 5], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("pairs", [False, True], ids=["halves", "pairs"])
def test_steps(hip, dtype, pairs):
    s = Server(hip, dtype, 6, pairs)
    stream = hip.Stream()
    graph = hip.Graph(stream)
    graph.begin()
    s.launch(stream)
    graph.end()
    r = np.random.default_rng(5)
    waited = 0
    steps = [[17, 40, 1, 0, 30, 8], [1, 1, 1, 33, 1, 1], [1] * 6, [60, 1, 0, 1, 30, 4], [1, 90, 90, 90, 1, 1],
             "release", [1, 60, 1, 1, 90, 0], [0] * 6, [3, 1, 1, 1, 50, 40], "release", [90, 1, 1, 1, 1, 1], [1] * 6]
    for n, counts in enumerate(steps):
        if counts == "release":
            s.pool.release((np.arange(6) % 3 == n % 3).astype(np.int32))
            continue
        s.pool.dc.upload(np.asarray(counts, np.int32))
        x = r.standard_normal((ROWS, HEADS + 2 * HK, D))
        s.qkv.upload(raw(x, dtype))
        want = s.pool.expect(counts)
        graph.launch()
        stream.synchronize()
        s.check(want, x)
        waited += want[0][-1] < sum(counts)
    assert waited, "no request waited"


@pytest.mark.parametrize("dtype", [0, 4, 5], ids=["f32", "f16", "bf16"])
def test_prompts_without_a_cache(hip, dtype):
    """vm_hip_qk_norm_rope and vm_hip_attention_packed on the rows of a first step:
    the keys bit for bit, the outputs within both calls' tolerances."""
    s = Server(hip, dtype, 3, False)
    counts = [50, 1, 33]
    s.pool.dc.upload(np.asarray(counts, np.int32))
    x = np.random.default_rng(6).standard_normal((ROWS, HEADS + 2 * HK, D))
    s.qkv.upload(raw(x, dtype))
    want = s.pool.expect(counts)
    s.launch(None)
    rows, size = want[0][-1], s.size
    k_out = hip.DeviceBuffer(ROWS * HK * D * size)
    q_out, out = hip.DeviceBuffer(s.q.nbytes), hip.DeviceBuffer(s.out.nbytes)
    hip.qk_norm_rope(s.qkv.addr, dtype, ROWS, HEADS, HK, D, s.norm, s.rope, s.pool.dp.addr, q_out.addr, k_out.addr)
    width = (HEADS + 2 * HK) * D
    nbytes = hip.attention_packed_workspace_bytes(3, ROWS, HEADS, HK, D)
    ws = hip.DeviceBuffer.from_array(np.zeros(nbytes, np.uint8))
    hip.attention_packed(q_out.addr, k_out.addr, s.qkv.addr + (HEADS + HK) * D * size, out.addr, dtype, HEADS * D, HK * D,
                         width, 3, ROWS, HEADS, HK, D, s.pool.dstart.addr, 0.0, ws.addr, ws.nbytes)
    kind = np.float32 if dtype == 0 else np.int16
    assert np.array_equal(q_out.download(kind, (ROWS, HEADS, D))[:rows], s.q.download(kind, (ROWS, HEADS, D))[:rows])
    slots = np.asarray(want[2][:rows])
    k, v = numbers(k_out.download(kind, (ROWS, HK, D)), dtype), held(x[:, HEADS + HK:], dtype)
    assert np.array_equal(k[:rows], s.stored(s.dk)[slots])
    q = back(s.q, (ROWS, HEADS, D), dtype)
    for buf in (out, s.out):
        got = back(buf, (ROWS, HEADS, D), dtype)
        for a, e in zip(want[0][:-1], want[0][1:]):
            close(got[a:e], *reference(q[a:e], k[a:e], v[a:e], 0, D ** -0.5, dtype))
