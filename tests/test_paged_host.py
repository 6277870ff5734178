"""Argument checks of the entry points around the paged cache that run before any CUDA call, without a GPU; and the
list form of the page bookkeeping that the GPU tests compare with."""
import ctypes

import pytest
import torch

import paged_ref as R
from orcasaq2 import _ext

FAKE = 4096          # never dereferenced: these calls fail validation first


@pytest.fixture(scope="module")
def lib():
    import os
    if not os.path.exists(_ext.library_path()):
        import __graft_entry__
        __graft_entry__.build()
    return _ext.lib()


def _cache(**kw):
    a = dict(k_pages=FAKE, v_pages=FAKE, page_stride=4 * 16 * 256, head_stride=16 * 256, token_stride=256, num_pages=8,
             page_size=16, kv_heads=4, head_dim=256, dtype=0, k_scale=1.0, v_scale=1.0)
    a.update(kw)
    return ctypes.byref(_ext.Exl3PagedCache(**a))


def test_tree_attn_argument_checks(lib):
    def call(cache=None, **kw):
        a = dict(q=FAKE, qs=24 * 256, out=FAKE, os=24 * 256, table=FAKE, ts=4, tw=4, lens=FAKE, starts=FAKE, mask=None, B=2,
                 T=8, most=4, qh=24, scale=0.1, bf=0)
        a.update(kw)
        return lib.exl3_tree_attn(*a.values(), cache or _cache(), None, 0, None)
    for name in ("q", "out", "table", "lens", "starts"):
        assert call(**{name: None}) == -6
    assert call(_cache(k_pages=None)) == -6
    assert call(_cache(head_dim=64)) == -3
    assert call(_cache(dtype=1)) == -3 and call(_cache(dtype=0), bf=1) == -3 and call(_cache(dtype=5)) == -3
    for c in (_cache(page_size=24), _cache(page_size=0), _cache(num_pages=0), _cache(kv_heads=0), _cache(token_stride=128),
              _cache(head_stride=16 * 256 + 4), _cache(page_stride=0), _cache(k_scale=0.0), _cache(v_scale=float("nan")),
              _cache(dtype=2, head_stride=16 * 256 + 8)):
        assert call(c) == -1
    for kw in (dict(qh=25), dict(qh=0), dict(B=-1), dict(B=65536), dict(T=-1), dict(tw=0), dict(ts=3), dict(qs=24 * 256 + 4),
               dict(os=23 * 256), dict(most=0), dict(most=65), dict(tw=2 ** 30, ts=2 ** 30)):
        assert call(**kw) == -1, kw
    assert call(_cache(k_pages=FAKE + 8)) == -2 and call(q=FAKE + 2) == -2 and call(mask=FAKE + 4) == -2
    assert call(B=0) == 0 and call(T=0) == 0                # nothing to do
    assert lib.exl3_tree_attn_workspace_bytes(0, 24, 4, _cache()) == 0


def test_append_argument_checks(lib):
    def call(cache=None, **kw):
        a = dict(qkv=FAKE, ld=32 * 256, q=None, ldq=0, qw=None, kw=None, norm=1, eps=1e-6, cos=FAKE, sin=FAKE, rot=256, inter=0,
                 rows=10, pos=FAKE, slots=FAKE, T=3, qh=24, bf=0)
        a.update(kw)
        return lib.exl3_qk_norm_rope_append(*a.values(), cache or _cache(), None)
    for name in ("qkv", "cos", "sin", "pos", "slots"):
        assert call(**{name: None}) == -6
    assert call(_cache(v_pages=None)) == -6
    assert call(_cache(head_dim=192)) == -3 and call(bf=1) == -3
    for kw in (dict(ld=31 * 256), dict(ld=32 * 256 + 4), dict(rot=40), dict(rot=272), dict(rot=-16), dict(rows=0), dict(T=-1),
               dict(qh=0), dict(eps=-1.0), dict(q=FAKE, ldq=23 * 256), dict(q=FAKE, ldq=24 * 256 + 4)):
        assert call(**kw) == -1, kw
    assert call(qkv=FAKE + 8) == -2 and call(pos=FAKE + 4) == -2 and call(qw=FAKE + 2) == -2
    assert call(T=0) == 0 and call(_cache(page_size=7), T=0) == 0


def test_pages_argument_checks(lib):
    def tables(**kw):
        a = dict(block_table=FAKE, seq_lens=FAKE, held=FAKE, refs=FAKE, free_list=FAKE, counters=FAKE, table_stride=4,
                 table_width=4, max_seqs=4, num_pages=8, page_size=16)
        a.update(kw)
        return ctypes.byref(_ext.Exl3PageTables(**a))

    def pools(ptrs=(FAKE, FAKE + 65536), **kw):
        arr = (ctypes.c_void_p * max(1, len(ptrs)))(*ptrs)
        a = dict(page_stride=4096, head_stride=1024, token_stride=256, num_pools=len(ptrs), heads=4, row_bytes=256)
        a.update(kw)
        return ctypes.byref(_ext.Exl3PagePools(ctypes.cast(arr, ctypes.POINTER(ctypes.c_void_p)), *a.values()))

    fork = lambda p=None, t=None, n=1, a=FAKE, ws=FAKE, size=1 << 20: lib.exl3_cache_fork(p or pools(), t or tables(), a, FAKE, n, ws, size, None)   # noqa: E731
    assert fork(a=None) == -6 and fork(pools((FAKE, None))) == -6 and fork(t=tables(refs=None)) == -6
    for p in (pools(()), pools([FAKE] * 257), pools(row_bytes=24), pools(row_bytes=2048), pools(heads=0), pools(page_stride=0),
              pools(token_stride=128), pools(head_stride=1032)):
        assert fork(p) == -1
    for t in (tables(table_stride=3), tables(max_seqs=0), tables(num_pages=0), tables(page_size=0), tables(num_pages=1 << 21),
              tables(table_width=1 << 20, table_stride=1 << 20, page_size=1 << 12)):
        assert fork(t=t) == -1
    assert fork(n=-1) == -1 and fork(n=1025) == -1 and fork(ws=None) == -5 and fork(size=4) == -5 and fork(ws=FAKE + 4) == -2
    assert fork(pools((FAKE + 8,))) == -2 and fork(n=0) == 0
    assert lib.exl3_cache_fork_workspace_bytes(0) == 0 and lib.exl3_cache_fork_workspace_bytes(1024) >= 1024 * 24
    reserve = lambda t=None, n=1, s=FAKE, T=4, slots=FAKE: lib.exl3_cache_reserve(t or tables(), s, FAKE, n, slots, FAKE, T, FAKE, FAKE, None)       # noqa: E731
    assert reserve(s=None) == -6 and reserve(slots=None) == -6 and reserve(n=0) == -1 and reserve(T=-1) == -1
    assert reserve(T=(1 << 20) + 1) == -1 and reserve(slots=FAKE + 4) == -2
    free = lambda t=None, n=1, s=FAKE: lib.exl3_cache_free(t or tables(), s, n, None)       # noqa: E731
    assert free(s=None) == -6 and free(n=1025) == -1 and free(n=0) == 0 and free(t=tables(held=None)) == -6
    accept = lambda n=1, path=FAKE, ps=4, most=4: lib.exl3_cache_accept(pools(), tables(), FAKE, FAKE, FAKE, path, ps, most, FAKE, n, None)      # noqa: E731
    assert accept(path=None) == -6 and accept(ps=3) == -1 and accept(most=65, ps=65) == -1 and accept(n=0) == 0 and accept(path=FAKE + 2) == -2


def test_bindings_refuse_host_tensors():
    q = torch.zeros(1, 4, 128, dtype=torch.half)
    kp = torch.zeros(2, 2, 16, 128, dtype=torch.half)
    with pytest.raises(RuntimeError):
        _ext.tree_attn_paged(q, kp, kp, torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, dtype=torch.int32),
                             torch.tensor([0, 1], dtype=torch.int32), 1)
    with pytest.raises(RuntimeError):
        _ext.qk_norm_rope_append(torch.zeros(1, 8 * 128, dtype=torch.half), None, None, torch.zeros(1, dtype=torch.int64),
                                 torch.zeros(1, dtype=torch.int64), kp, kp, 4)
    with pytest.raises(RuntimeError):
        _ext.cache_free(_ext.page_tables(2, 2, 2, "cpu"), torch.zeros(1, dtype=torch.int32))


def test_list_form_of_the_bookkeeping():
    """fork, reserve and free undo each other, and shared pages return with their last holder."""
    t = _ext.page_tables(4, 4, 8, "cpu")
    p = R.Pages(t)
    slots, pos, starts, base = p.reserve([0, 1], [20, 3], 8, 25)
    assert p.table[0][:3] == [0, 1, 2] and p.table[1][0] == 3 and starts == [0, 20, 23] and base == [0, 0]
    assert slots[:9] == [0, 1, 2, 3, 4, 5, 6, 7, 8] and slots[20:] == [24, 25, 26, -1, -1] and pos[20:] == [0, 1, 2, 0, 0]
    before = (list(p.stack), p.left)
    p.fork([0, 0], [2, 3], 8)
    assert p.refs[:3] == [3, 3, 1] and p.copies == [(2, 4, 4), (2, 5, 4)] and p.left == 2
    p.free([2, 3])
    assert p.left == before[1] and p.stack[:p.left] == before[0][:p.left] and p.refs[:4] == [1, 1, 1, 1]
    p.free([0, 1])
    assert p.left == 8 and sorted(p.stack) == list(range(8)) and p.status == 0 and not any(p.refs)
