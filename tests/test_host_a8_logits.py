"""What the INT8 x INT8 product and the logits' rules refuse, and their
buffers' sizes, checked without a GPU: every refusal comes before anything is
launched."""
from __future__ import annotations

import pytest

import velomind_hip as H

P = 0x1000   # an aligned address that is never read here


def _refused(call, *args):
    with pytest.raises(H.VmHipError) as e:
        call(*args)
    assert e.value.status == H.EINVAL and str(e.value)


def _each(call, ok, bad):
    for at, value in bad:
        args = list(ok)
        args[at] = value
        _refused(call, *args)


def test_a8_sizes():
    assert H.a8_weights_bytes(64, 32) == 2048 and H.a8_weights_bytes(65, 33) == 4 * 2048
    assert H.a8_stage_bytes(1, 1) >= 32 * 64 + 32 * 4 and H.a8_stage_bytes(0, 5) == 0
    for bad in [(0, 8), (131073, 8), (-1, 8), (8, -1), (8, (1 << 24) + 1)]:
        _refused(H.a8_weights_bytes, *bad)
    for bad in [(-1, 8), (8, 0), (8, 131073), ((1 << 24) + 1, 8)]:
        _refused(H.a8_stage_bytes, *bad)
    for bad in [(-1, 8, 8), (8, 0, 8), (8, 8, -1), (1 << 24, 8, 1 << 24)]:
        _refused(H.qmm_a8_workspace_bytes, *bad)
    assert H.qmm_a8_workspace_bytes(0, 8, 8) == 0 and H.qmm_a8_workspace_bytes(8, 8, 0) == 0
    assert 0 <= H.qmm_a8_workspace_bytes(16, 5632, 2048) < (64 << 20)


def test_a8_pack_and_stage_arguments():
    _each(H.a8_pack, [P, 64, 64, P], [(0, None), (1, 0), (1, 131073), (2, -1), (3, None), (3, P + 8)])
    H.a8_pack(None, 64, 0, None)
    _each(H.a8_stage, [P, H.DTYPE_F32, 4, 64, P],
          [(0, None), (0, P + 2), (1, 1), (2, -1), (3, 0), (3, 131073), (4, None), (4, P + 4)])
    _each(H.a8_stage, [P + 2, H.DTYPE_F16, 4, 64, P], [(0, P + 1)])
    H.a8_stage(None, H.DTYPE_F32, 0, 64, None)


def test_qmm_a8_arguments():
    need = H.qmm_a8_workspace_bytes(16, 8192, 512)
    assert need > 0
    _each(H.qmm_a8, [P, P, P, P, H.DTYPE_F32, 16, 8192, 512, P, need],
          [(0, None), (0, P + 8), (1, None), (1, P + 4), (2, None), (2, P + 2), (3, None), (3, P + 2), (4, 2), (5, -1), (6, 0),
           (6, 131073), (7, -1), (8, None), (8, P + 8), (9, need - 1), (9, -1)])
    H.qmm_a8(None, None, None, None, H.DTYPE_F32, 0, 64, 64, None, 0)
    H.qmm_a8(None, None, None, None, H.DTYPE_F32, 4, 64, 0, None, 0)


def test_logits_arguments():
    need = H.logits_rules_workspace_bytes(2, 3, 1000)
    assert need > 0 and H.logits_rules_workspace_bytes(0, 3, 1000) == 0
    r = H.LogitsRules()
    ok = [r, P, P, H.DTYPE_F32, P, 2, 3, 1000, None, P, need]
    _each(H.logits_rules, ok, [(1, None), (1, P + 2), (2, P + 1), (3, 1), (5, -1), (5, 65537), (6, -1), (6, 40000), (7, 0),
                               (7, 1 << 31), (9, None), (9, P + 8), (10, need - 1)])
    _refused(H.logits_rules, r, P, None, H.DTYPE_F32, None, 2, 3, 1000, None, P, need)
    for bad in [dict(history=P), dict(history=P, history_lengths=P, history_stride=-1), dict(bias_tokens=P, bias_stride=4),
                dict(bias_tokens=P, bias_values=P, bias_stride=4), dict(bias_tokens=P, bias_values=P, bias_lengths=P, bias_stride=-1)]:
        _refused(H.logits_rules, H.LogitsRules(**bad), *ok[1:])
    assert H.open_library().vm_hip_logits_rules_apply(None, P, P, 0, P, 2, 3, 1000, None, P, need, None) == H.EINVAL
    for bad in [(-1, 1, 10), (65537, 1, 10), (1, 1, 0), (1, 1, 1 << 31)]:
        _refused(H.logits_rules_workspace_bytes, *bad)
    H.logits_rules(r, None, None, H.DTYPE_F32, None, 0, 3, 1000, None, None, 0)


def test_a8_calls_of_more_threads_than_a_launch_has():
    assert H.a8_stage_bytes(1 << 23, 1) > 0 and H.a8_weights_bytes(1, 1 << 24) > 0
    assert H.qmm_a8_workspace_bytes(1 << 18, 64, 1 << 19) == 0
    _refused(H.a8_stage_bytes, (1 << 23) + 1, 1)
    _refused(H.a8_stage, P, H.DTYPE_F32, 1 << 24, 1, P)
    _refused(H.qmm_a8_workspace_bytes, 1 << 19, 64, 1 << 19)
    _refused(H.qmm_a8, P, P, P, P, H.DTYPE_F32, 1 << 19, 64, 1 << 19, None, 0)
