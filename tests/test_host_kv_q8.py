"""What the INT8 cache's entry points and the attention over it refuse, and
the attention's workspace, checked without a GPU: every refusal comes before
anything is launched."""
from __future__ import annotations

import numpy as np
import pytest

import velomind_hip as H

P = 0x1000   # a 16-byte aligned address that is never read here


def _cache(**over):
    a = dict(k_codes=P, k_scales=P, v_codes=P, v_scales=P, batch=2, kv_heads=2, max_seq=100, head_dim=64)
    a.update(over)
    return H.KvQ8(*a.values())


BAD_CACHES = [dict(head_dim=96), dict(head_dim=0), dict(batch=-1), dict(batch=65536), dict(kv_heads=0), dict(max_seq=0),
              dict(max_seq=1 << 25), dict(max_seq=1 << 24, head_dim=128), dict(k_codes=None), dict(v_codes=None),
              dict(k_scales=None), dict(v_scales=None), dict(k_codes=P + 8), dict(v_codes=P + 1), dict(k_scales=P + 2)]


def _refused(call, *args):
    with pytest.raises(H.VmHipError) as e:
        call(*args)
    assert e.value.status == H.EINVAL and str(e.value)


@pytest.mark.parametrize("over", BAD_CACHES, ids=str)
def test_bad_caches(over):
    c = _cache(**over)
    _refused(H.kv_q8_append, c, P, H.DTYPE_F32, 1, 4, P, P, P, None, None, P)
    _refused(H.kv_q8_read, c, 0, 1, P, P, H.DTYPE_F32)
    _refused(H.kv_q8_keep, c, P, P, P, 4)
    _refused(H.attention_q8, c, P, P, H.DTYPE_F32, 1, 4, P, None, None, 1.0, None, 0)


def test_append_arguments():
    c, ok = _cache(), [P, H.DTYPE_F32, 1, 4, P, P, P, None, None, P]
    for at, bad in [(0, None), (0, P + 4), (1, 1), (1, -1), (2, -1), (2, (1 << 20) + 1), (3, 3), (3, 0), (4, None), (5, None),
                    (6, None), (9, None), (9, P + 8)]:
        args = list(ok)
        args[at] = bad
        _refused(H.kv_q8_append, c, *args)
    H.kv_q8_append(c, None, H.DTYPE_F32, 0, 4, None, None, None, None, None, None)   # nothing to do
    H.kv_q8_append(_cache(batch=0), None, H.DTYPE_F32, 3, 4, None, None, None, None, None, None)


def test_read_arguments():
    c, ok = _cache(), [0, 1, P, P, H.DTYPE_F32]
    for at, bad in [(0, -1), (0, 100), (0, 101), (1, -1), (1, 101), (1, 1 << 62), (2, P + 4), (3, P + 4), (4, 3)]:
        args = list(ok)
        args[at] = bad
        _refused(H.kv_q8_read, c, *args)
    _refused(H.kv_q8_read, c, 0, 1, None, None, H.DTYPE_F32)
    H.kv_q8_read(c, 100, 0, None, None, H.DTYPE_F32)


def test_keep_arguments():
    c, ok = _cache(), [P, P, P, 4]
    for at, bad in [(0, None), (1, None), (2, None), (3, -1), (3, 257)]:
        args = list(ok)
        args[at] = bad
        _refused(H.kv_q8_keep, c, *args)
    H.kv_q8_keep(c, None, None, None, 0)


def test_attention_arguments():
    c = _cache(max_seq=4096)
    need = H.attention_q8_workspace_bytes(2, 1, 4, 2, 64, 4096)
    assert need > 0
    ok = [P, P, H.DTYPE_F32, 1, 4, P, None, None, 1.0, P, need]
    for at, bad in [(0, None), (0, P + 4), (1, None), (1, P + 8), (2, 2), (3, -1), (3, (1 << 20) + 1), (4, 5), (4, 0), (5, None),
                    (8, np.inf), (8, np.nan), (9, None), (9, P + 4), (10, need - 1), (10, 0)]:
        args = list(ok)
        args[at] = bad
        _refused(H.attention_q8, c, *args)
    H.attention_q8(c, None, None, H.DTYPE_F32, 0, 4, None, None, None, 1.0, None, 0)


def test_workspace_bytes():
    for bad in [(1, 1, 4, 3, 64, 100), (1, 1, 4, 4, 80, 100), (1, 1, 4, 4, 64, 0), (-1, 1, 4, 4, 64, 100), (1, -1, 4, 4, 64, 100),
                (65535, 1 << 20, 4096, 4096, 64, 100)]:
        _refused(H.attention_q8_workspace_bytes, *bad)
    assert H.attention_q8_workspace_bytes(0, 1, 4, 4, 64, 100) == 0
    assert H.attention_q8_workspace_bytes(1, 0, 4, 4, 64, 100) == 0
    assert H.attention_q8_workspace_bytes(64, 512, 32, 8, 64, 4096) == 0   # enough rows to fill the GPU
    one = H.attention_q8_workspace_bytes(1, 1, 32, 4, 64, 4096)
    assert 0 < one <= H.attention_q8_workspace_bytes(1, 1, 32, 4, 64, 100000) < (64 << 20)


def test_calls_of_more_threads_than_a_launch_has():
    many = _cache(batch=4096, kv_heads=4096)
    _refused(H.kv_q8_keep, many, P, P, P, 4)
    # 1024 x 65536 tokens of four heads
    _refused(H.kv_q8_append, _cache(batch=1024, kv_heads=1), P, H.DTYPE_F32, 65536, 2, P, P, P, None, None, P)
    assert H.attention_q8_workspace_bytes(1024, 65536, 2, 1, 64, 100) == 0
    _refused(H.attention_q8_workspace_bytes, 4096, 65536, 2, 1, 64, 100)
    _refused(H.attention_q8, _cache(batch=4096, kv_heads=1), P, P, H.DTYPE_F32, 65536, 2, P, None, None, 1.0, None, 0)
