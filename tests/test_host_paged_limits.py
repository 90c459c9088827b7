"""Limits of the paged and packed attention's arguments, checked without a GPU:
every refusal comes before anything is launched (no call here has a workspace)."""
from __future__ import annotations

import pytest

import velomind_hip as H

P = 0x1000   # a 16-byte aligned address that is never read here


def _message(call, *args):
    with pytest.raises(H.VmHipError) as e:
        call(*args)
    assert e.value.status == H.EINVAL
    return str(e.value)


def _paged(batch, kv_heads, max_pages, page=128, scale=0.0):
    cache = H.KvPaged(P, P, H.DTYPE_BF16, 10, page, kv_heads, 64)
    return _message(H.attention_paged, cache, P, max_pages, P, P, batch, 5, 1, kv_heads, P, P, scale, None, 0)


@pytest.mark.parametrize("batch,kv_heads,max_pages", [(14, 2637, 58169), (42, 879, 58169), (2048, 1024, 1024)], ids=str)
def test_keys_of_all_requests_and_what_a_workgroup_adds_stay_below_2_to_31(batch, kv_heads, max_pages):
    """Rounds of 128 keys are dealt out to 512 workgroups, rounded up: their count
    plus 511 is 32 bits."""
    assert batch * kv_heads * max_pages + 511 >= 2 ** 31
    assert "2^38" in _paged(batch, kv_heads, max_pages)


def test_the_most_keys_that_are_taken():
    assert 512 * 2049 * 2047 == 2 ** 31 - 512
    assert "workspace" in _paged(512, 2049, 2047)
    assert "2^38" in _paged(512, 2049, 2048)


@pytest.mark.parametrize("scale", [3.4e38, 2.4e38], ids=str)
def test_scales_that_overflow_with_the_factor_of_exp2(scale):
    assert "scale" in _paged(1, 2, 4, scale=scale)
    assert "scale" in _message(H.attention_packed, P, P, P, P, H.DTYPE_F16, 512, 512, 512, 2, 10, 4, 2, 64, P, scale,
                               None, 0)


@pytest.mark.parametrize("scale", [2.3e38, 1e-38, 0.0, -1.0, float("-inf")], ids=str)
def test_scales_that_are_taken(scale):
    assert "workspace" in _paged(1, 2, 4, scale=scale)
    assert "workspace" in _message(H.attention_packed, P, P, P, P, H.DTYPE_F16, 512, 512, 512, 2, 10, 4, 2, 64, P,
                                   scale, None, 0)
