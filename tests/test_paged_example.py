"""The speculative step that the integration notes show, run with stand-ins for the operators: the positions that it
hands to the append are those of the drafts' depths in their trees."""
import os
import random
import re
import types

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _example():
    text = open(os.path.join(ROOT, "INTEGRATION.md")).read()
    blocks = [b for b in re.findall(r"```python\n(.*?)```", text, re.S) if "cache_reserve" in b]
    assert len(blocks) == 1
    lines = blocks[0].splitlines()
    indent = min(len(x) - len(x.lstrip()) for x in lines if x.strip())
    return "\n".join(x[indent:] for x in lines)


def test_example_positions_are_depths():
    r = random.Random(3)
    counts, lens, room = [7, 1, 12], [30, 4, 19], 25
    depth, mask = [], []
    for n in counts:
        rows = []
        for j in range(n):
            up = r.randrange(-1, j) if j else -1
            rows.append((rows[up] if up >= 0 else 0) | 1 << j)
        mask += rows
        depth += [bin(v).count("1") - 1 for v in rows]
    place = [j for n in counts for j in range(n)]
    base = [b for n, b in zip(counts, lens) for _ in range(n)]
    pad = room - len(place)
    assert depth != place
    seen = []

    def reserve(*_):
        pos = torch.tensor([b + j for b, j in zip(base, place)] + [0] * pad)
        return torch.tensor([1] * len(place) + [-1] * pad), pos, torch.tensor([0, 7, 8, 20]), torch.tensor(lens)

    def append(qkv, cos, sin, positions, *_, **__):
        seen.append(positions.clone())

    quiet = lambda *_, **__: None                                   # noqa: E731
    ext = types.SimpleNamespace(page_tables=lambda *_: dict(block_table=None, seq_lens=None), cache_fork=quiet, cache_reserve=reserve,
                                qk_norm_rope_append=append, tree_attn_paged=quiet, cache_accept=quiet, cache_free=quiet)
    names = dict.fromkeys(("max_seqs pages_per_seq num_pages device pools parents children seqs drafts page_size tokens qkv cos sin "
                           "k v q_heads wq wk qbuf max_drafts path taken done").split())
    names.update(_ext=ext, layers=range(3), mask=torch.tensor(mask + [0] * pad),
                 shift=torch.tensor([d - j for d, j in zip(depth, place)] + [0] * pad))
    exec(_example(), names)
    assert len(seen) == 3
    for positions in seen:
        assert positions[:len(place)].tolist() == [b + d for b, d in zip(base, depth)]
