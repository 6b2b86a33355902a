"""Page accounting of ``PagedLogoCache`` (CPU: nothing is launched)."""

import pytest
import torch

from logo_amd.ops.paged import PagedLogoCache


def _cache(pages=12, local=8, page=16, window=20):
    return PagedLogoCache(2, 1, 64, pages, local, page_size=page, window=window, device="cpu")


def test_step_layout():
    c = _cache()
    a, b = c.add(), c.add()
    s = c.step([(b, 17), (a, 1)])
    assert s.cu.tolist() == [0, 17, 18] and s.lens.tolist() == [17, 1] and s.last.tolist() == [16, 17]
    assert s.max_q == 17 and s.max_len == 17 and s.table.shape == s.local_table.shape == (2, 2)
    used = [p for p in s.table.flatten().tolist() if p >= 0]
    assert len(set(used)) == 3 and s.table[1, 1] == -1
    assert all(t.dtype == torch.int32 for t in (s.cu, s.lens, s.last, s.table, s.local_table))
    # the next step keeps the pages and adds what grew
    s2 = c.step([(b, 16), (a, 16)])
    assert s2.table[0, :2].tolist() == s.table[0].tolist() and s2.table[0, 2] >= 0 and s2.table[1, 0] == s.table[1, 0]
    assert c.length(b) == 33 and c.length(a) == 17


def test_local_pages_behind_the_window_come_back():
    c = _cache(pages=40, local=4)
    a = c.add()
    held = []
    for n in (16, 16, 16, 16, 1, 15, 16, 16):
        s = c.step([(a, n)])
        before = c.length(a) - n
        row = s.local_table[0].tolist()
        # every key that a new token sees has a page: positions before - 20 .. length - 1
        assert all(row[j // 16] >= 0 for j in range(max(0, before - 20), c.length(a)))
        live = [p for p in row if p >= 0]
        assert len(set(live)) == len(live) <= 4
        held.append(len(live))
    assert c.free_pages()[1] == 4 - held[-1]
    assert all(p >= 0 for p in s.table[0].tolist())
    c.release(a)
    assert c.free_pages() == (40, 4)


def test_a_prompt_longer_than_the_local_pool_is_refused_whole():
    """Its first piece is stored before any of it lies behind the window."""
    c = _cache(pages=12, local=2)
    a = c.add()
    with pytest.raises(RuntimeError, match="out of pages"):
        c.step([(a, 48)])
    assert c.free_pages() == (12, 2) and c.length(a) == 0
    c.step([(a, 32)])
    assert c.free_pages() == (10, 0)


def test_out_of_pages_takes_nothing():
    c = _cache(pages=3, local=8)
    a, b = c.add(), c.add()
    c.step([(a, 30)])
    with pytest.raises(RuntimeError, match="out of pages"):
        c.step([(a, 3), (b, 1)])
    assert c.free_pages() == (1, 6) and c.length(a) == 30 and c.length(b) == 0
    c.step([(b, 16)])
    c.release(a)
    assert c.free_pages() == (2, 7)


def test_refusals():
    c = _cache()
    a = c.add()
    for new, msg in (([], "at least one"), ([(a, 1), (a, 1)], "once"), ([(a, 0)], "at least one token"), ([(9, 1)], "unknown")):
        with pytest.raises(ValueError, match=msg):
            c.step(new)
    c.release(a)
    for call in (lambda: c.release(a), lambda: c.length(a), lambda: c.step([(a, 1)])):
        with pytest.raises(ValueError, match="unknown"):
            call()
    with pytest.raises(ValueError, match="page_size"):
        _cache(page=24)
