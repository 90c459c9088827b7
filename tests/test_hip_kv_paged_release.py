"""Pages given back where tables hold entries that are no page, where the pool is
full, and of many requests of many pages, on the GPU, against plain Python."""
from __future__ import annotations

import numpy as np
import pytest

from test_hip_kv_paged import Pool, i32

pytestmark = pytest.mark.gpu


def release(p, finished, free):
    """Gives back, and compares everything with the rule: of finished requests every
    entry in use is cleared, and those that are pages go behind `free`, as many as fit."""
    left = p.tables.copy()
    lengths = p.lengths.copy()
    free = list(free)
    for b in np.flatnonzero(finished):
        for j in range(min(max(-(-int(lengths[b]) // p.page), 0), p.max_pages)):
            if 0 <= left[b, j] < p.pages and len(free) < p.pages:
                free.append(int(left[b, j]))
            left[b, j] = -1
        lengths[b] = 0
    f = i32(p.hip, finished)
    p.hip.kv_paged_release(p.batch, p.max_pages, p.pages, p.page, f.addr, p.dl.addr, p.dt.addr, p.df.addr, p.dn.addr)
    p.tables, p.lengths, p.free = left, lengths, free
    p.check_state()


@pytest.mark.parametrize("batch", [1, 3, 256, 257, 2048])
@pytest.mark.parametrize("bad", [-1, -7, 10 ** 9, -2 ** 31, "pages"], ids=str)
def test_entries_that_are_no_page_stay_out_of_the_pool(hip, batch, bad):
    """And a later step gives every token that it admits a slot."""
    r = np.random.default_rng(batch)
    lengths = r.integers(0, 150, batch)
    p = Pool(hip, lengths, 16, int((-(-lengths // 16)).sum()) + 4, 12, 61, 4096)
    gone = (r.random(p.tables.shape) < 0.2) & (p.tables >= 0)
    gone[batch // 2, 0] = True
    p.tables[gone] = p.pages if bad == "pages" else bad
    p.dt.upload(p.tables.astype(np.int32))
    release(p, r.random(batch) < 0.6, p.free)
    release(p, np.ones(batch), p.free)
    assert all(0 <= x < p.pages for x in p.free)
    p.step(np.full(batch, 17))
    rows = p.dstart.download(np.int32, (batch + 1,))[-1]
    assert (p.dslots.download(np.int32, (p.rows,))[:rows] >= 0).all()


@pytest.mark.parametrize("count", [0, 1, 4, 6, 9, -3], ids=str)
def test_a_full_pool(hip, count):
    """What does not fit is dropped, tables and lengths are cleared all the same."""
    p = Pool(hip, [40, 0, 40, 17], 16, 8, 3, 62, 4)
    p.dn.upload(np.asarray([count], np.int32))
    have = p.df.download(np.int32, (8,))[:min(max(count, 0), 8)]
    release(p, [1, 1, 1, 0], have)


@pytest.mark.parametrize("batch,length,page", [(1, 60000, 16), (256, 8000, 16), (300, 2000, 16), (2048, 700, 16),
                                               (5, 2 ** 31 - 1, 16), (40, 0, 16)], ids=str)
def test_many_pages(hip, batch, length, page):
    """More entries than a step of the kernel takes, requests without any between them."""
    r = np.random.default_rng(length)
    lengths = np.where(r.random(batch) < 0.2, 0, length) if batch > 1 else np.asarray([length])
    width = min(-(-length // page), 5000) + 1
    need = int(np.minimum(-(-lengths // page), width).sum())
    p = Pool(hip, lengths, page, need + 3, width, 63, 4)
    release(p, np.ones(batch) if batch < 3 else r.random(batch) < 0.7, p.free)
    release(p, np.ones(batch), p.free)
