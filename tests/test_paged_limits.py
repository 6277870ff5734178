"""Limits of the entry points around the paged cache that are refused before any CUDA call, without a GPU."""
import ctypes

import pytest

from orcasaq2 import _ext
from test_paged_host import FAKE, _cache, lib  # noqa: F401


@pytest.mark.parametrize("scale", [float("nan"), float("inf"), float("-inf"), 3.3e38])
def test_tree_attn_scale_is_finite(lib, scale):  # noqa: F811
    args = (FAKE, 24 * 256, FAKE, 24 * 256, FAKE, 4, 4, FAKE, FAKE, None, 2, 8, 4, 24, scale, 0, _cache(), None, 0, None)
    assert lib.exl3_tree_attn(*args) == -1


def test_tree_attn_heads_per_kv_head(lib):  # noqa: F811
    def call(qh):
        return lib.exl3_tree_attn(FAKE, qh * 256, FAKE, qh * 256, FAKE, 4, 4, FAKE, FAKE, None, 2, 8, 4, qh, 0.1, 0, _cache(), None, 0, None)
    assert call(4 * 33) == -3 and call(4 * 32) == -5          # unsupported; no workspace


def test_fork_page_size(lib):  # noqa: F811
    def call(page, heads):
        t = _ext.Exl3PageTables(FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, 1, 1, 4, 8, page)
        p = _ext.Exl3PagePools((ctypes.c_void_p * 1)(FAKE), 1 << 40, page * 512, 512, 1, heads, 512, 0)
        return lib.exl3_cache_fork(ctypes.byref(p), ctypes.byref(t), FAKE, FAKE, 1, None, 0, None)
    assert call(1 << 22, 16) == -1                            # 2^31 sixteen-byte pieces in a page
    assert call(1 << 20, 16) == -5                            # allowed; no workspace
