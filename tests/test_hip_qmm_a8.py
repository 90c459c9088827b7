"""INT8 x INT8 products against numpy, bit for bit: codes and scales are
defined in fp32 steps, the sum is an exact integer (computed here in fp64,
below 2^53), and what follows is one conversion and two fp32 products, rounded
once to the output's type."""
from __future__ import annotations

import numpy as np
import pytest

from test_hip_kv_q8 import assert_equal, dev, dev_typed, host_typed, narrow, quantise

pytestmark = pytest.mark.gpu


def expect(a, codes, scale, dtype):
    ca, sa = quantise(a)
    acc = (ca.astype(np.float64) @ codes.astype(np.float64)).astype(np.float32)
    with np.errstate(all="ignore"):
        return narrow(acc * (sa[:, None] * scale[None, :]), dtype)


def run(hip, a, codes, scale, dtype, out_dtype=None, stream=None, ws=None):
    out_dtype = dtype if out_dtype is None else out_dtype
    (m, k), n = a.shape, codes.shape[1]
    da, dc, ds = dev_typed(hip, a, dtype), dev(hip, codes), dev(hip, scale)
    staged, packed = hip.DeviceBuffer(hip.a8_stage_bytes(m, k)), hip.DeviceBuffer(hip.a8_weights_bytes(k, n))
    # what no call may rely on
    hip.check(hip.open_library().vm_hip_memcpy_h2d(staged.ptr, np.full(staged.nbytes, 0x7f, np.uint8).ctypes.data, staged.nbytes, None))
    out = dev_typed(hip, np.full((m + 1, n), 7.0), out_dtype)
    need = hip.qmm_a8_workspace_bytes(m, k, n)
    ws = dev(hip, np.zeros(max(need, 1), np.uint8)) if ws is None else ws
    hip.a8_pack(dc.addr, k, n, packed.addr, stream)
    hip.a8_stage(da.addr, dtype, m, k, staged.addr, stream)
    hip.qmm_a8(staged.addr, packed.addr, ds.addr, out.addr, out_dtype, m, k, n, ws.addr, ws.nbytes, stream)
    if stream is not None:
        stream.synchronize()
    y = host_typed(out, (m + 1, n), out_dtype)
    assert (y[m] == 7.0).all(), "written past the last row"
    if need:
        assert (ws.download(np.uint32, (4096,)) == 0).all(), "tickets left behind"
    return y[:m]


def weights(k, n, seed):
    r = np.random.default_rng(seed)
    return r.integers(-127, 128, (k, n)).astype(np.int8), r.uniform(0.001, 0.01, n).astype(np.float32)


@pytest.mark.parametrize("m", [1, 5, 32, 33, 65, 129, 300])
@pytest.mark.parametrize("k,n", [(1, 1), (15, 33), (64, 32), (65, 31), (200, 100), (1000, 257), (2048, 96), (4160, 70)])
@pytest.mark.parametrize("dtype", [0, 4, 5])
def test_products(hip, m, k, n, dtype):
    print(f"case qmm_a8 m={m} k={k} n={n} dtype={dtype}", flush=True)
    r = np.random.default_rng(m + k)
    a = narrow(r.standard_normal((m, k)) * 2, dtype)
    codes, scale = weights(k, n, k + n)
    assert_equal(run(hip, a, codes, scale, dtype), expect(a, codes, scale, dtype))


@pytest.mark.parametrize("m,k,n", [(7, 28672, 40), (3, 131072, 33), (40, 20000, 64), (2100, 512, 96), (2049, 100, 33),
                                   (530, 1100, 1030), (1024, 64, 2048), (700, 8192, 600),
                                   (2049, 130, 8200), (4100, 64, 4160), (300, 2500, 16500)])
@pytest.mark.parametrize("dtype", [0, 5])
def test_long_rows_and_large_outputs(hip, m, k, n, dtype):
    print(f"case qmm_a8 large m={m} k={k} n={n} dtype={dtype}", flush=True)
    r = np.random.default_rng(k)
    a = narrow(r.standard_normal((m, k)), dtype)
    codes, scale = weights(k, n, n)
    assert_equal(run(hip, a, codes, scale, dtype), expect(a, codes, scale, dtype))


def test_largest_sums(hip):
    # every product 127 * 127 (or its negative) over the longest row: 2^31 is not reached
    k = 131072
    a = np.ones((2, k), np.float32)
    a[1] = -1
    codes, scale = np.full((k, 8), 127, np.int8), np.ones(8, np.float32)
    print("case qmm_a8 largest sums", flush=True)
    got = run(hip, a, codes, scale, 0)
    assert_equal(got, expect(a, codes, scale, 0))
    assert got[0, 0] > 1.3e5


@pytest.mark.parametrize("dtype,out", [(0, 5), (5, 0), (4, 0), (0, 4)])
def test_output_type_is_its_own(hip, dtype, out):
    a = narrow(np.random.default_rng(1).standard_normal((20, 300)), dtype)
    codes, scale = weights(300, 50, 2)
    ca, sa = quantise(a)
    y = (ca.astype(np.float64) @ codes.astype(np.float64)).astype(np.float32) * (sa[:, None] * scale[None, :])
    print(f"case qmm_a8 {dtype} -> {out}", flush=True)
    assert_equal(run(hip, a, codes, scale, dtype, out), narrow(y, out))


@pytest.mark.parametrize("m", [6, 70])
def test_special_rows(hip, m):
    # zeros, tiny, huge, infinite and NaN rows beside ordinary ones; 16-bit
    # outputs that overflow
    r = np.random.default_rng(3)
    a = r.standard_normal((m, 130)).astype(np.float32)
    a[0] = 0
    a[1] *= np.float32(1e-37)
    a[2] *= np.float32(1e37)
    a[3, 5] = np.inf
    a[4, 129] = np.nan
    codes, scale = weights(130, 40, 5)
    print(f"case qmm_a8 specials m={m}", flush=True)
    for out in (0, 4):
        got, ca = run(hip, a, codes, scale, 0, out), expect(a, codes, scale, 0)
        assert_equal(got, narrow(ca, out))
        assert np.isnan(got[3:5]).all() and np.isfinite(got[5:]).all() and (got[0] == 0).all()


def test_one_staged_buffer_for_siblings_on_a_stream_and_in_a_graph(hip):
    m, k, ns = 19, 700, (96, 33, 200)
    r = np.random.default_rng(4)
    stream = hip.Stream()
    a = dev(hip, np.zeros((m, k), np.float32))
    staged = hip.DeviceBuffer(hip.a8_stage_bytes(m, k))
    members = []
    for n in ns:
        codes, scale = weights(k, n, n)
        packed, out = hip.DeviceBuffer(hip.a8_weights_bytes(k, n)), dev(hip, np.zeros((m, n), np.float32))
        dcodes = dev(hip, codes)
        hip.a8_pack(dcodes.addr, k, n, packed.addr)
        hip.synchronize()
        ws = dev(hip, np.zeros(max(1, hip.qmm_a8_workspace_bytes(m, k, n)), np.uint8))
        members.append((n, codes, scale, packed, dev(hip, scale), out, ws))
    graph = hip.Graph(stream)
    graph.begin()
    hip.a8_stage(a.addr, 0, m, k, staged.addr, stream)
    for n, _, _, packed, ds, out, ws in members:
        hip.qmm_a8(staged.addr, packed.addr, ds.addr, out.addr, 0, m, k, n, ws.addr, ws.nbytes, stream)
    graph.end()
    for i in range(3):
        x = r.standard_normal((m, k)).astype(np.float32)
        a.upload(x, stream.handle)
        print(f"case qmm_a8 replay {i}", flush=True)
        graph.launch()
        stream.synchronize()
        for n, codes, scale, _, _, out, _ in members:
            assert_equal(out.download(np.float32, (m, n)), expect(x, codes, scale, 0))


def test_one_workspace_for_several_shapes(hip):
    shapes = [(3, 4096, 64), (40, 2048, 96), (3, 4096, 64), (100, 1024, 33), (1, 8192, 32)]
    ws = dev(hip, np.zeros(max(hip.qmm_a8_workspace_bytes(*s) for s in shapes), np.uint8))
    for m, k, n in shapes:
        a = np.random.default_rng(k).standard_normal((m, k)).astype(np.float32)
        codes, scale = weights(k, n, n)
        print(f"case qmm_a8 shared workspace m={m} k={k} n={n}", flush=True)
        assert_equal(run(hip, a, codes, scale, 0, ws=ws), expect(a, codes, scale, 0))


def test_packed_int8_weights_of_the_framework(hip):
    # the codes and scales that vm_hip_pack_int8 makes, against the product
    # of the numbers they stand for: a's quantization is off by half a step
    # of amax / 127 per value
    r = np.random.default_rng(6)
    w, a = r.standard_normal((256, 64)).astype(np.float32), r.standard_normal((9, 256)).astype(np.float32)
    codes, scale = hip.run_pack_int8(w)
    got = run(hip, a, codes, scale, 0)
    dense = codes.astype(np.float64) * scale.astype(np.float64)
    bound = (np.abs(a).max(1) / 254 * (1 + 1e-5))[:, None] * np.abs(dense).sum(0)[None, :]
    assert np.all(np.abs(got - a.astype(np.float64) @ dense) <= bound)


def test_two_streams(hip):
    # products that share a staged buffer and its weights, each with its own
    # workspace and output, on two streams at once
    m, k, n = 12, 4096, 96
    a = np.random.default_rng(9).standard_normal((m, k)).astype(np.float32)
    codes, scale = weights(k, n, 9)
    da, dc, ds = dev(hip, a), dev(hip, codes), dev(hip, scale)
    staged, packed = hip.DeviceBuffer(hip.a8_stage_bytes(m, k)), hip.DeviceBuffer(hip.a8_weights_bytes(k, n))
    hip.a8_pack(dc.addr, k, n, packed.addr)
    hip.a8_stage(da.addr, 0, m, k, staged.addr)
    need = hip.qmm_a8_workspace_bytes(m, k, n)
    assert need > 0   # several workgroups share a tile here
    sets = [(hip.Stream(), dev(hip, np.zeros((m, n), np.float32)), dev(hip, np.zeros(need, np.uint8))) for _ in range(2)]
    hip.synchronize()
    print("case qmm_a8 two streams", flush=True)
    for _ in range(30):
        for s, out, ws in sets:
            hip.qmm_a8(staged.addr, packed.addr, ds.addr, out.addr, 0, m, k, n, ws.addr, need, s)
    for s, out, _ in sets:
        s.synchronize()
        assert_equal(out.download(np.float32, (m, n)), expect(a, codes, scale, 0))
