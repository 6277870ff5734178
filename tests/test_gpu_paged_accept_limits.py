"""cache_accept at path lengths where its shared memory passes the 48 KB that a launch has without asking.  In fresh
processes: what an earlier, larger call asked for would hide a size that asks for too little."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

CHILD = """
import sys
import torch
from orcasaq2 import _ext as ext
hd, page, pages, seqs = int(sys.argv[1]), 16, 24, 3
for most in map(int, sys.argv[2].split(",")):
    g = torch.Generator().manual_seed(most)
    base = torch.tensor([0, 5, 30], dtype=torch.int32)
    pools = torch.randn(2, pages, 2, page, hd, generator=g).half().cuda()
    tables = ext.page_tables(seqs, 8, pages, "cuda")
    which = torch.arange(seqs, dtype=torch.int32).cuda()
    drafts = torch.full((seqs,), most, dtype=torch.int32)
    ext.cache_reserve(tables, which, (base + drafts).cuda(), page, 512)
    path = torch.stack([torch.randperm(most, generator=g) for _ in range(seqs)]).int()
    taken = torch.tensor([most, most - 1, 1], dtype=torch.int32)
    want, table = pools.clone(), tables["block_table"].cpu()
    for b in range(seqs):
        for j in range(taken[b]):
            x, y = int(base[b] + path[b, j]), int(base[b]) + j
            want[:, table[b, y // page], :, y % page] = pools[:, table[b, x // page], :, x % page]
    ext.cache_accept(pools, tables, which, base.cuda(), drafts.cuda(), path.cuda(), taken.cuda())
    assert torch.equal(pools, want), most
    assert tables["seq_lens"].cpu().tolist() == (base + taken).tolist() and tables["counters"][1] == 0
print("moved")
"""


@pytest.mark.parametrize("hd,most", [(256, "48,47,49,64,48"), (512, "24"), (512, "64,24,1")])
def test_accept_at_the_limit_of_shared_memory(ext, hd, most):
    root = os.path.dirname(os.path.dirname(os.path.abspath(ext.__file__)))
    env = dict(os.environ, PYTHONPATH=os.pathsep.join([root, os.environ.get("PYTHONPATH", "")]))
    got = subprocess.run([sys.executable, "-c", CHILD, str(hd), most], env=env, capture_output=True, text=True, timeout=300)
    assert got.returncode == 0 and got.stdout.strip() == "moved", got.stderr[-2000:]
