"""What the paged cache's entry points refuse, and their workspaces, checked
without a GPU: every refusal comes before anything is launched."""
from __future__ import annotations

import math

import pytest

import velomind_hip as H

P = 0x1000   # a 16-byte aligned address that is never read here


def _refused(call, *args, **kw):
    with pytest.raises(H.VmHipError) as e:
        call(*args, **kw)
    assert e.value.status == H.EINVAL and str(e.value)


def _each_refused(call, ok, bad):
    for at, value in bad:
        args = list(ok)
        args[at] = value
        _refused(call, *args)


def _cache(**over):
    a = dict(k=P, v=P, dtype=H.DTYPE_F32, pages=10, page_size=16, kv_heads=2, head_dim=64)
    a.update(over)
    return H.KvPaged(*a.values())


BAD_CACHES = [dict(k=None), dict(v=None), dict(k=P + 8), dict(v=P + 4), dict(dtype=1), dict(dtype=3), dict(pages=0),
              dict(pages=-1), dict(pages=1 << 27), dict(page_size=0), dict(page_size=8), dict(page_size=24),
              dict(page_size=512), dict(page_size=-16), dict(kv_heads=0), dict(kv_heads=4097), dict(head_dim=96),
              dict(head_dim=0), dict(head_dim=256)]


@pytest.mark.parametrize("over", BAD_CACHES, ids=str)
def test_bad_caches(over):
    c = _cache(**over)
    _refused(H.kv_paged_append, c, P, 1, 4, None, None, P, P, P)
    _refused(H.attention_paged, c, P, 4, P, P, 1, 1, 1, 4, P, P, 0.0, P, 1 << 40)


PLAN = dict(batch=2, rows=4, max_pages=3, pages=10, page_size=16, lengths=P, counts=P, free_pages=P, free_count=P,
            tables=P, row_start=P, lengths_out=P, free_count_out=P, positions=P, slots=P)


@pytest.mark.parametrize("over", [dict(batch=-1), dict(batch=2049), dict(rows=-1), dict(rows=(1 << 24) + 1),
                                  dict(max_pages=0), dict(max_pages=1 << 27), dict(pages=0), dict(pages=1 << 27),
                                  dict(page_size=12), dict(page_size=0), dict(page_size=1024)]
                         + [{k: None} for k in list(PLAN)[5:]] + [{k: P + 2} for k in list(PLAN)[5:]], ids=str)
def test_bad_plans(over):
    _refused(H.kv_paged_plan, H.PagePlan(**{**PLAN, **over}), P, 64)


def test_plan_workspace():
    for ws in [(None, 64), (P, 63), (P + 8, 64)]:
        _refused(H.kv_paged_plan, H.PagePlan(**PLAN), *ws)
    assert H.kv_paged_plan_workspace_bytes(2048, 1 << 24) == 64
    _refused(H.kv_paged_plan_workspace_bytes, 2049, 1)
    _refused(H.kv_paged_plan_workspace_bytes, 1, -1)
    H.kv_paged_plan(H.PagePlan(batch=0, rows=0, max_pages=1, pages=1, page_size=16), None, 0)   # nothing to do


def test_release_arguments():
    ok = [2, 3, 10, 16, P, P, P, P, P]
    _each_refused(H.kv_paged_release, ok, [(0, -1), (0, 2049), (1, 0), (1, 1 << 27), (2, 0), (2, 1 << 27), (3, 20)]
                  + [(i, None) for i in range(4, 9)] + [(i, P + 1) for i in range(4, 9)])
    H.kv_paged_release(0, 1, 1, 16, None, None, None, None, None)


def test_rope_tables_arguments():
    ok = [P, P, 0, 4, 64, 10000.0, None]
    _each_refused(H.rope_tables, ok, [(0, None), (1, None), (0, P + 2), (2, -1), (2, 1 << 31), (3, -1),
                                      (3, (1 << 31) + 1), (4, 0), (4, 63), (4, 130), (5, 1.0), (5, -2.0),
                                      (5, math.inf), (5, math.nan)])
    good = dict(kind=H.ROPE_RAMP, factor=4.0, low=1.0, high=32.0, original=2048.0, attention=1.0)
    for over in [dict(kind=-1), dict(kind=4), dict(factor=0.0), dict(factor=math.nan), dict(factor=math.inf),
                 dict(low=0.0), dict(low=32.0), dict(high=math.inf), dict(original=0.0), dict(original=math.nan),
                 dict(attention=0.0), dict(attention=math.inf), dict(kind=H.ROPE_LINEAR, factor=-1.0),
                 dict(kind=H.ROPE_BANDS, low=4.0, high=1.0), dict(kind=H.ROPE_PLAIN, attention=math.nan)]:
        _refused(H.rope_tables, P, P, 0, 4, 64, 10000.0, H.RopeScaling(**{**good, **over}))
    H.rope_tables(None, None, 5, 0, 64, 10000.0, H.RopeScaling(**good))


BAD_ROPES = [dict(dim=-2), dict(dim=65), dict(dim=66), dict(layout=2), dict(layout=-1), dict(rows=0),
             dict(cos_table=None), dict(sin_table=None), dict(cos_table=P + 1)]
BAD_NORMS = [dict(q_weight=None), dict(k_weight=None), dict(q_weight=P + 2), dict(eps=-1.0), dict(eps=math.nan),
             dict(eps=math.inf)]


def _rope(**over):
    return H.Rope(**{**dict(cos_table=P, sin_table=P, rows=9, dim=64, layout=0), **over})


def _norm(**over):
    return H.QkNorm(**{**dict(q_weight=P, k_weight=P, eps=1e-6), **over})


def test_append_arguments():
    ok = [_cache(), P, 1, 4, _norm(), _rope(), P, P, P]
    _each_refused(H.kv_paged_append, ok,
                  [(1, None), (1, P + 8), (2, -1), (2, (1 << 24) + 1), (3, 0), (3, 3), (3, 65538), (6, None), (6, P + 2),
                   (7, None), (7, P + 2), (8, None), (8, P + 4)]
                  + [(4, _norm(**o)) for o in BAD_NORMS] + [(5, _rope(**o)) for o in BAD_ROPES])
    H.kv_paged_append(_cache(), None, 0, 4, None, None, None, None, None)


def test_qk_norm_rope_arguments():
    ok = [P, H.DTYPE_F16, 1, 4, 2, 64, _norm(), _rope(), P, P, P]
    _each_refused(H.qk_norm_rope, ok,
                  [(0, None), (0, P + 8), (1, 2), (2, -1), (3, 3), (4, 0), (4, 4097), (5, 80), (8, None), (9, None),
                   (9, P + 8), (10, None), (10, P + 8)]
                  + [(6, _norm(**o)) for o in BAD_NORMS] + [(7, _rope(**o)) for o in BAD_ROPES])
    H.qk_norm_rope(None, H.DTYPE_F16, 0, 4, 2, 64, None, None, None, None, None)


def test_attention_packed_arguments():
    #     q  k  v  out dtype  strides        b  rows heads kv d row_start scale ws bytes
    ok = [P, P, P, P, H.DTYPE_BF16, 512, 512, 512, 2, 1000, 4, 2, 64, P, 0.0, P, 1 << 40]
    _each_refused(H.attention_packed, ok,
                  [(i, None) for i in (0, 1, 2, 3, 13, 15)] + [(i, P + 8) for i in (0, 1, 2, 3, 15)]
                  + [(13, P + 2), (4, 1), (5, 248), (5, 516), (6, 120), (7, 120), (6, (1 << 24) + 8), (8, -1), (8, 2049),
                     (9, -1), (9, (1 << 24) + 1), (10, 3), (10, 0), (11, 0), (11, 4097), (12, 96), (14, math.inf),
                     (14, math.nan), (16, 0)])
    H.attention_packed(None, None, None, None, H.DTYPE_BF16, 512, 512, 512, 0, 5, 4, 2, 64, None, 0.0, None, 0)
    H.attention_packed(None, None, None, None, H.DTYPE_BF16, 512, 512, 512, 2, 0, 4, 2, 64, None, 0.0, None, 0)


def test_attention_paged_arguments():
    #     cache  tables max_pages q out b rows max_rows heads row_start lengths scale ws bytes
    ok = [_cache(), P, 4, P, P, 2, 5, 3, 4, P, P, 0.0, P, 1 << 40]
    _each_refused(H.attention_paged, ok,
                  [(i, None) for i in (1, 3, 4, 9, 10, 12)] + [(i, P + 8) for i in (3, 4, 12)]
                  + [(i, P + 2) for i in (1, 9, 10)]
                  + [(2, 0), (2, (1 << 20) + 1), (5, -1), (5, 2049), (6, -1), (6, (1 << 24) + 1), (7, -1), (8, 3), (8, 0),
                     (8, 1 << 20), (11, math.inf), (11, math.nan), (13, 0)])
    _refused(H.attention_paged, _cache(kv_heads=4096), P, 1 << 20, P, P, 2048, 5, 3, 4096, P, P, 0.0, P, 1 << 40)
    H.attention_paged(_cache(), None, 4, None, None, 0, 5, 3, 4, None, None, 0.0, None, 0)
    H.attention_paged(_cache(), None, 4, None, None, 2, 0, 3, 4, None, None, 0.0, None, 0)


def test_attention_workspaces():
    """A workspace for the largest rows and max_rows does for smaller ones (the
    same batch, heads and table)."""
    for heads, hk, d in [(32, 4, 64), (64, 8, 128), (15, 5, 64), (40, 1, 128)]:
        for batch in (1, 2, 7, 64, 2048):
            sizes = [H.attention_paged_workspace_bytes(batch, r, m, heads, hk, d, 4096)
                     for r, m in [(1, 1), (batch, 1), (batch + 1, 2), (batch + 99, 100), (batch + 5000, 0)]]
            assert sizes == sorted(sizes) and sizes[0] >= 0 and not any(s % 16 for s in sizes)
            for tokens in (16, 64, 100, 128, 129, 300):
                few, many = (H.attention_paged_workspace_bytes(batch, r, 0, heads, hk, d, tokens) for r in (1, 5000))
                assert 0 <= few <= many
            sizes = [H.attention_packed_workspace_bytes(batch, rows, heads, hk, d) for rows in (1, 60, 128, 129, 5000)]
            assert sizes == sorted(sizes)
    _refused(H.attention_paged_workspace_bytes, 1, 1, 1, 4, 3, 64, 16)
    _refused(H.attention_paged_workspace_bytes, 1, 1, 1, 4, 2, 64, 0)
    _refused(H.attention_paged_workspace_bytes, 1, 1, 1, 4, 2, 64, (1 << 24) + 1)
    _refused(H.attention_packed_workspace_bytes, 1, 1, 4, 2, 32)
    assert H.attention_paged_workspace_bytes(0, 5, 1, 4, 2, 64, 16) == 0
