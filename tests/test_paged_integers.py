"""Whole numbers that do not fit the 32 bits of the C entry points are refused, not cut to what fits.  Without a GPU."""
import pytest
import torch

from orcasaq2 import _ext


class _Calls:
    """Stands in for the library: records that a call was made."""

    def __init__(self):
        self.made = []

    def __getattr__(self, name):
        def fn(*args):
            self.made.append(name)
            return 0
        return fn


def _tensor(shape, dtype, stride=None):
    """A tensor without memory that says it lies on CUDA device 0."""
    class OnGpu(torch.Tensor):
        is_cuda = True

        def get_device(self):
            return 0

        def data_ptr(self):
            return 4096

        def new_empty(self, *_, **__):
            raise AssertionError("no allocation")
    t = torch.empty_strided(shape, stride, dtype=dtype, device="meta") if stride else torch.empty(shape, dtype=dtype, device="meta")
    return t.as_subclass(OnGpu)


@pytest.fixture
def calls(monkeypatch):
    c = _Calls()
    monkeypatch.setattr(_ext, "lib", lambda: c)
    monkeypatch.setattr(_ext, "_call", lambda *a: c.made.append("launch"))
    return c


def _tree(most=4, step=None):
    q, kp = _tensor((8, 24, 256), torch.half), _tensor((8, 4, 16, 256), torch.half)
    table = _tensor((2, 4), torch.int32, (step, 1) if step else None)
    lens, starts = _tensor((2,), torch.int32), _tensor((3,), torch.int32)
    out = _tensor((8, 24, 256), torch.half)
    return _ext.tree_attn_paged(q, kp, kp, table, lens, starts, most, out=out)


def test_stand_ins_reach_the_launch(calls):
    with pytest.raises(AssertionError):                            # the workspace: every check before it passed
        calls.exl3_tree_attn_workspace_bytes = lambda *_: 1024
        _tree()


@pytest.mark.parametrize("most", [2 ** 32 + 4, 2 ** 32, -2 ** 32 + 1, 65, 0])
def test_tree_attn_max_drafts(calls, most):
    with pytest.raises(RuntimeError):
        _tree(most)
    assert "launch" not in calls.made


def test_tree_attn_table_step(calls):
    with pytest.raises(RuntimeError):
        _tree(step=2 ** 32 + 4)
    assert "launch" not in calls.made


@pytest.mark.parametrize("tokens", [2 ** 32, 2 ** 32 + 5, 2 ** 20 + 1, -1])
def test_reserve_tokens(calls, tokens):
    S, N = 4, 8
    t = dict(block_table=_tensor((S, 4), torch.int32), seq_lens=_tensor((S,), torch.int32), held=_tensor((S,), torch.int32),
             refs=_tensor((N,), torch.int32), free_list=_tensor((N,), torch.int32), counters=_tensor((2,), torch.int32))
    with pytest.raises(RuntimeError):
        _ext.cache_reserve(t, _tensor((1,), torch.int32), _tensor((1,), torch.int32), 16, tokens)
    assert "launch" not in calls.made


def test_accept_path_step(calls):
    S, N = 4, 8
    t = dict(block_table=_tensor((S, 4), torch.int32), seq_lens=_tensor((S,), torch.int32), held=_tensor((S,), torch.int32),
             refs=_tensor((N,), torch.int32), free_list=_tensor((N,), torch.int32), counters=_tensor((2,), torch.int32))
    pools = _tensor((2, N, 2, 16, 128), torch.half)
    v = _tensor((2,), torch.int32)
    _ext.cache_accept(pools, t, v, v, v, _tensor((2, 3), torch.int32), v)
    assert calls.made == ["launch"]
    calls.made.clear()
    with pytest.raises(RuntimeError):
        _ext.cache_accept(pools, t, v, v, v, _tensor((2, 3), torch.int32, (2 ** 32 + 3, 1)), v)
    assert "launch" not in calls.made
