"""The INT8 cache on the GPU: rotation and quantization as keys and values are
written, reading back, and moving an accepted path's rows, against numpy.

Codes and scales are defined in fp32 steps (each product, difference and sum
of the rotation rounded; max / 127; the reciprocal; round half away from
zero), so they are compared bit for bit with numpy's fp32.  q is the rotated
row rounded once to its type: fp32 bit for bit, 16 bits equal to numpy's (or
torch's) rounding of the same fp32 value."""
from __future__ import annotations

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

TORCH = {0: torch.float32, 4: torch.float16, 5: torch.bfloat16}


def quantise(x):
    """(codes, scales) of fp32 rows [..., n]."""
    x = np.asarray(x, np.float32)
    amax = np.abs(x).max(-1, keepdims=True)
    with np.errstate(all="ignore"):
        fine = np.isfinite(amax)
        zero = amax < np.float32(2.0 ** -119)
        s = np.where(zero, np.float32(1), amax / np.float32(127)).astype(np.float32)
        y = x * (np.float32(1) / s)
        c = np.clip(np.copysign(np.floor(np.abs(y).astype(np.float64) + 0.5), y), -127, 127)
        c = np.where(fine & ~zero, c, 0)
    return c.astype(np.int8), np.where(fine, s, np.float32(np.nan))[..., 0]


def rotate(x, cos, sin):
    h = x.shape[-1] // 2
    a, b = x[..., :h], x[..., h:]
    return np.concatenate([a * cos - b * sin, b * cos + a * sin], -1)


def narrow(x, dtype):
    """fp32 rounded to dtype, as fp32."""
    return torch.from_numpy(np.ascontiguousarray(x, np.float32)).to(TORCH[dtype]).float().numpy()


class Cache:
    """A cache on the GPU, full of recognisable codes and scales."""

    def __init__(self, hip, batch, kv_heads, max_seq, d, seed):
        r = np.random.default_rng(seed)
        self.shape = (batch, kv_heads, max_seq, d)
        self.host = {}
        for kv in "kv":
            self.host[kv + "_codes"] = r.integers(-127, 128, self.shape).astype(np.int8)
            self.host[kv + "_scales"] = r.uniform(0.005, 0.02, self.shape[:3]).astype(np.float32)
        self.dev = {k: hip.DeviceBuffer.from_array(v) for k, v in self.host.items()}
        self.q8 = hip.KvQ8(self.dev["k_codes"].addr, self.dev["k_scales"].addr, self.dev["v_codes"].addr,
                           self.dev["v_scales"].addr, batch, kv_heads, max_seq, d)

    def download(self):
        return {k: b.download(self.host[k].dtype, self.host[k].shape) for k, b in self.dev.items()}


def same(a, b):
    assert a.keys() == b.keys()
    for k in a:
        assert np.array_equal(a[k].view(np.uint8), b[k].view(np.uint8)), k


def assert_equal(got, want):
    """Bit for bit (any NaN for a NaN), with a short message."""
    assert got.shape == want.shape
    differ = ~((got == want) | (np.isnan(got) & np.isnan(want)))
    assert not differ.any(), f"{differ.sum()} of {differ.size} differ, first at {np.argwhere(differ)[0]}: {got[differ][0]!r}, not {want[differ][0]!r}"


def dev(hip, a):
    return hip.DeviceBuffer.from_array(a)


def dev_typed(hip, x, dtype):
    t = torch.from_numpy(np.ascontiguousarray(x, np.float32)).to(TORCH[dtype])
    return hip.DeviceBuffer.from_array(t.numpy() if dtype == 0 else t.view(torch.int16).numpy())


def host_typed(buf, shape, dtype):
    if dtype == 0:
        return buf.download(np.float32, shape)
    return torch.from_numpy(buf.download(np.int16, shape)).view(TORCH[dtype]).float().numpy()


def expect_append(cache, qkv, dtype, heads, cos, sin, pos, counts, depths, q0):
    """(cache arrays, q) after an append; qkv fp32 holding dtype's values."""
    out, q = {k: v.copy() for k, v in cache.host.items()}, q0.copy()
    batch, hk, max_seq, d = cache.shape
    rows = qkv.shape[1]
    for b in range(batch):
        for t in range(rows if counts is None else max(0, min(rows, counts[b]))):
            p = int(pos[b]) + t
            if not 0 <= p < max_seq:
                continue
            turn = min(max(int(pos[b]) + (t if depths is None else int(depths[b, t])), 0), max_seq - 1)
            x = qkv[b, t].reshape(heads + 2 * hk, d)
            with np.errstate(all="ignore"):
                y = rotate(x[:heads + hk], cos[turn], sin[turn]).astype(np.float32)
            q[b, :, t] = narrow(y[:heads], dtype)
            for kv, z in (("k", y[heads:]), ("v", x[heads + hk:])):
                out[kv + "_codes"][b, :, p], out[kv + "_scales"][b, :, p] = quantise(z)
    return out, q


def run_append(hip, cache, qkv, dtype, heads, cos, sin, pos, counts, depths, q0, stream=None):
    batch, hk, max_seq, d = cache.shape
    rows = qkv.shape[1]
    bufs = [dev_typed(hip, qkv, dtype), dev(hip, cos), dev(hip, sin), dev(hip, np.asarray(pos, np.int32)),
            dev(hip, np.asarray(counts, np.int32)) if counts is not None else None,
            dev(hip, np.asarray(depths, np.int32)) if depths is not None else None, dev_typed(hip, q0, dtype)]
    hip.kv_q8_append(cache.q8, bufs[0].addr, dtype, rows, heads, bufs[1].addr, bufs[2].addr, bufs[3].addr,
                     bufs[4].addr if bufs[4] else None, bufs[5].addr if bufs[5] else None, bufs[6].addr, stream)
    if stream is not None:
        stream.synchronize()
    return host_typed(bufs[6], q0.shape, dtype)


def case(batch, heads, hk, d, rows, max_seq, dtype, seed, special=False):
    r = np.random.default_rng(seed)
    qkv = narrow(r.standard_normal((batch, rows, (heads + 2 * hk) * d)) * 3, dtype)
    if special:
        x = qkv.reshape(batch, rows, heads + 2 * hk, d)
        x[0, 0, heads, 3] = np.inf               # a key
        x[0, 0, heads + hk, d - 1] = np.nan      # a value
        x[-1, -1, heads + hk] = 0.0              # a value of zeros
        x[-1, -1, heads] = 1e-37                 # its key: subnormal products
        x[0, -1, 0, 0] = -np.inf                 # a query
    angle = r.uniform(0, 6.28, (max_seq, d // 2))
    return qkv, np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)


@pytest.mark.parametrize("batch,heads,hk,rows,max_seq,pos", [
    (1, 1, 1, 1, 1, [0]), (1, 32, 4, 1, 77, [76]), (1, 15, 5, 7, 64, [0]), (3, 4, 2, 5, 41, [0, 36, 17]), (2, 8, 1, 33, 100, [3, 60]),
])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", [0, 4, 5])
def test_append(hip, batch, heads, hk, rows, max_seq, pos, d, dtype):
    print(f"case kv_q8_append b={batch} h={heads}/{hk} rows={rows} d={d} dtype={dtype}", flush=True)
    cache = Cache(hip, batch, hk, max_seq, d, rows)
    qkv, cos, sin = case(batch, heads, hk, d, rows, max_seq, dtype, rows + d)
    q0 = narrow(np.full((batch, heads, rows, d), 7.0), dtype)
    want, q = expect_append(cache, qkv, dtype, heads, cos, sin, pos, None, None, q0)
    got_q = run_append(hip, cache, qkv, dtype, heads, cos, sin, pos, None, None, q0)
    same(cache.download(), want)
    assert np.array_equal(got_q, q)


@pytest.mark.parametrize("dtype", [0, 4, 5])
def test_append_of_trees_padding_and_positions_outside(hip, dtype):
    # depths shared by siblings and outside the tables; sequences with fewer
    # tokens than rows, none, and a count past rows; positions before row 0
    # and past max_seq; infinities, NaN, zeros and subnormals
    batch, heads, hk, d, rows, max_seq = 6, 4, 2, 64, 9, 50
    pos = [10, 45, -4, 30, 0, 2**31 - 3]
    counts = [9, 100, 9, 0, 3, 9]
    r = np.random.default_rng(5)
    depths = r.integers(0, 5, (batch, rows)).astype(np.int32)
    depths[0, 3], depths[0, 4] = 1000, -1000
    qkv, cos, sin = case(batch, heads, hk, d, rows, max_seq, dtype, 3, special=True)
    qkv.reshape(batch, rows, heads + 2 * hk, d)[4, 1, heads + hk] = 0.0
    cache = Cache(hip, batch, hk, max_seq, d, 1)
    q0 = narrow(r.standard_normal((batch, heads, rows, d)), dtype)
    print(f"case kv_q8_append tree and padding dtype={dtype}", flush=True)
    want, q = expect_append(cache, qkv, dtype, heads, cos, sin, pos, counts, depths, q0)
    got_q = run_append(hip, cache, qkv, dtype, heads, cos, sin, pos, counts, depths, q0)
    got = cache.download()
    for kv in "kv":   # NaN scales carry no particular bits
        k = kv + "_scales"
        assert np.array_equal(got[k], want[k], equal_nan=True)
        assert np.array_equal(got[kv + "_codes"], want[kv + "_codes"])
    assert np.array_equal(got_q, q, equal_nan=True)
    assert np.isnan(got["k_scales"][0, 0, 10]) and np.isnan(got["v_scales"][0, 0, 10])
    assert got["v_scales"][4, 0, 1] == 1.0


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", [0, 4, 5])
@pytest.mark.parametrize("first,rows", [(0, 37), (36, 1), (5, 20), (3, 0)])
def test_read(hip, d, dtype, first, rows):
    batch, hk, max_seq = 2, 3, 37
    cache = Cache(hip, batch, hk, max_seq, d, 9)
    shape = (batch, hk, max(rows, 1), d)
    k, v = dev_typed(hip, np.full(shape, 5.0), dtype), dev_typed(hip, np.full(shape, 5.0), dtype)
    print(f"case kv_q8_read d={d} dtype={dtype} first={first} rows={rows}", flush=True)
    hip.kv_q8_read(cache.q8, first, rows, k.addr, v.addr, dtype)
    for kv, buf in (("k", k), ("v", v)):
        got = host_typed(buf, shape, dtype)
        if rows == 0:
            assert (got == 5.0).all()
            continue
        x = cache.host[kv + "_codes"].astype(np.float32) * cache.host[kv + "_scales"][..., None]
        assert np.array_equal(got, narrow(x[:, :, first:first + rows], dtype))
    if rows == 20:   # either output alone
        for one, other in ((k, v), (v, k)):
            fresh = dev_typed(hip, np.zeros(shape), dtype)
            hip.kv_q8_read(cache.q8, first, rows, fresh.addr if one is k else None, fresh.addr if one is v else None, dtype)
            assert np.array_equal(host_typed(fresh, shape, dtype), host_typed(one, shape, dtype))


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("width", [1, 7, 256])
def test_keep(hip, d, width):
    # ascending paths, any other order, the same row twice, rows outside
    batch, hk, max_seq = 5, 2, 300
    cache = Cache(hip, batch, hk, max_seq, d, width)
    r = np.random.default_rng(width)
    pos = np.array([20, 0, 290, -3, 17], np.int32)
    kept = np.stack([np.sort(r.choice(280, width, replace=False)), r.integers(0, 300, width), np.arange(width) + 2,
                     r.integers(-5, 10, width), np.zeros(width)]).astype(np.int32)
    counts = np.array([width, width, 999, width, -1], np.int32)
    bufs = [dev(hip, a) for a in (pos, kept, counts)]
    print(f"case kv_q8_keep d={d} width={width}", flush=True)
    hip.kv_q8_keep(cache.q8, *[b.addr for b in bufs], width)
    want = {k: v.copy() for k, v in cache.host.items()}
    for b in range(batch):
        for i in range(min(max(int(counts[b]), 0), width)):
            s, t = int(pos[b]) + int(kept[b, i]), int(pos[b]) + i
            if 0 <= s < max_seq and 0 <= t < max_seq:
                for k in want:
                    want[k][b, :, t] = cache.host[k][b, :, s]
    same(cache.download(), want)


def test_append_captured_and_replayed(hip):
    # the position lives in device memory: each replay writes where it says
    batch, heads, hk, d, rows, max_seq = 2, 4, 2, 64, 3, 60
    qkv, cos, sin = case(batch, heads, hk, d, rows, max_seq, 0, 8)
    cache = Cache(hip, batch, hk, max_seq, d, 2)
    stream = hip.Stream()
    bufs = [dev(hip, a) for a in (qkv.astype(np.float32), cos, sin)]
    dpos, q = dev(hip, np.zeros(batch, np.int32)), dev(hip, np.zeros((batch, heads, rows, d), np.float32))
    graph = hip.Graph(stream)
    graph.begin()
    hip.kv_q8_append(cache.q8, bufs[0].addr, 0, rows, heads, bufs[1].addr, bufs[2].addr, dpos.addr, None, None, q.addr, stream)
    graph.end()
    want = {k: v.copy() for k, v in cache.host.items()}
    for pos in ([0, 7], [20, 3], [57, 58]):
        dpos.upload(np.array(pos, np.int32), stream.handle)
        print(f"case kv_q8_append replay pos={pos}", flush=True)
        graph.launch()
        stream.synchronize()
        cache.host = want
        want, wq = expect_append(cache, qkv, 0, heads, cos, sin, pos, None, None, np.zeros((batch, heads, rows, d), np.float32))
        same(cache.download(), want)
