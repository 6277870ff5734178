"""tree_attn_paged with `out` in the place of q: the result and nothing else, for rows of one CTA, of several, of several tiles."""
import pytest
import torch

from test_gpu_paged import Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("i,shape", enumerate([
    ([300], [5], 24, 4, 256, 16, "HND", "fp16", "fp16"),
    ([9000, 40], [4, 7], 4, 1, 256, 16, "HND", "fp16", "fp16"),
    ([8000, 2049, 255], [61, 64, 20], 24, 4, 256, 16, "NHD", "fp16", "fp8"),
    ([33] * 300, [2] * 300, 32, 8, 128, 16, "HND", "bf16", "bf16"),
    ([900, 64], [64, 64], 32, 1, 128, 16, "HND", "fp16", "fp16"),
]))
def test_tree_attn_in_place(ext, i, shape):
    c = Case(900 + i, *shape, extra_rows=2)
    live, q0 = int(c.starts[-1]), c.q.clone()
    want = c.run(ext)
    for _ in range(3):
        c.q.copy_(q0)
        assert c.run(ext, out=c.q).data_ptr() == c.q.data_ptr()
        assert torch.equal(c.q[:live], want[:live]) and torch.equal(c.q[live:], q0[live:])
