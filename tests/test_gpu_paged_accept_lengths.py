"""cache_accept never makes a sequence longer: what a refused cache_reserve did not give, it does not take."""
import pytest
import torch

import paged_ref as R
from test_gpu_paged import _grow, _ints, _pools_of

pytestmark = pytest.mark.gpu
PAGE = 16


def _refused(ext, tables, ref, pools, seqs, base, drafts, path, taken):
    old = [p.clone() for p in pools]
    ext.cache_accept(pools, tables, _ints(seqs), base, _ints(drafts), _ints(path), _ints(taken))
    ref.status |= ext.PAGES_BAD
    assert ref.same(tables) == []
    assert all(torch.equal(a, b) for a, b in zip(pools, old))
    tables["counters"][1] = ref.status = 0


@pytest.mark.parametrize("path", [[0, 1], [1, 0]])
def test_accept_after_a_reserve_refused_for_a_shared_page(ext, path):
    tables = ext.page_tables(4, 6, 20, "cuda")
    ref = R.Pages(tables)
    pools = _pools_of(ext, 1, 20, 2, PAGE, 128, "fp16", "HND", 1, stacked=False)
    _grow(ext, tables, ref, [0], [40], PAGE)
    ext.cache_fork(pools, tables, _ints([0]), _ints([1]))
    ref.fork([0], [1], PAGE)
    ext.cache_accept(pools, tables, _ints([0]), _ints([20]), _ints([20]), _ints([[0]]), _ints([0]))      # back to 20 of 40 tokens
    ref.lens[0] = 20
    slots, _, _, base = ext.cache_reserve(tables, _ints([0]), _ints([2]), PAGE, 2)
    assert slots.tolist() == [-1, -1] and base.tolist() == [20]
    ref.status |= ext.PAGES_BAD
    _refused(ext, tables, ref, pools, [0], base, [2], [path], [2])


def test_accept_after_a_reserve_refused_for_room(ext):
    tables = ext.page_tables(4, 6, 20, "cuda")
    ref = R.Pages(tables)
    pools = _pools_of(ext, 1, 20, 2, PAGE, 128, "fp16", "HND", 2, stacked=False)
    _grow(ext, tables, ref, [0, 1], [20, 5], PAGE)
    _, _, _, base = _grow(ext, tables, ref, [1, 0], [3, 4], PAGE, room=5)       # the second does not fit, its page would
    assert ref.lens[:2] == [20, 8]
    old = [p.clone() for p in pools]
    ext.cache_accept(pools, tables, _ints([1, 0]), base, _ints([3, 4]), _ints([[0, 1], [0, 1]]), _ints([2, 2]))
    ref.lens[1] = 7
    assert ref.status == ext.PAGES_BAD and ref.same(tables) == []               # the first is served
    assert all(torch.equal(a, b) for a, b in zip(pools, old))
    tables["counters"][1] = ref.status = 0
    _refused(ext, tables, ref, pools, [0], _ints([20]), [4], [[3, 1]], [1])     # rows of a page that it holds, behind its end
    _refused(ext, tables, ref, pools, [0], _ints([21]), [0], [[0, 0]], [0])     # a base behind its end
    ext.cache_accept(pools, tables, _ints([0]), _ints([20]), _ints([4]), _ints([[0, 0]]), _ints([0]))    # nothing taken: as it is
    assert ref.same(tables) == []


def test_accept_after_a_reserve_refused_for_pages(ext):
    tables = ext.page_tables(2, 6, 3, "cuda")
    ref = R.Pages(tables)
    pools = _pools_of(ext, 1, 3, 2, PAGE, 128, "fp16", "HND", 3, stacked=False)
    _grow(ext, tables, ref, [0, 1], [30, 4], PAGE)
    _, _, _, base = _grow(ext, tables, ref, [0], [4], PAGE)
    assert ref.status == ext.PAGES_EXHAUSTED and ref.lens[0] == 30
    _refused(ext, tables, ref, pools, [0], base, [2], [[0, 1]], [2])
