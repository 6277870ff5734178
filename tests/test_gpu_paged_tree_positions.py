"""A speculative step with trees in which siblings share a position: what the accepted path leaves in the cache is what
appending the accepted tokens one after the other, at the positions that cache_reserve gives a chain, would have put there."""
import random

import pytest
import torch

import paged_ref as R
from test_gpu_paged import _gen, _ints, _random_tree, _signed

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kv,layout,hd", [("fp16", "HND", 256), ("fp8", "NHD", 128)])
def test_step_with_positions_by_depth(ext, kv, layout, hd):
    g, r = _gen(5), random.Random(5)
    qh, kvh, page, N = 4, 2, 16, 40
    kw = dict(layout=layout, k_scale=0.5, v_scale=0.25) if kv == "fp8" else dict(layout=layout)
    ang = torch.arange(200, device="cuda")[:, None] / 10000.0 ** (torch.arange(hd // 2, device="cuda") / (hd // 2))
    cos, sin = torch.cos(ang).float(), torch.sin(ang).float()

    def empty():
        return [torch.zeros(R.pool_shape(layout, N, kvh, page, hd), device="cuda", dtype=torch.half).to(R.DT[kv]) for _ in range(2)]

    def append(pools, qkv, positions, slots):
        q = torch.empty(qkv.shape[0], qh, hd, dtype=torch.half, device="cuda")
        return ext.qk_norm_rope_append(qkv, cos, sin, positions, slots, *pools, qh, q_out=q, **kw)
    lens, m = [37, 16], [9, 14]                                     # prompts, drafts
    prompt = [torch.randn(n, (qh + 2 * kvh) * hd, device="cuda", generator=g).half() for n in lens]
    drafts = torch.randn(sum(m), (qh + 2 * kvh) * hd, device="cuda", generator=g).half()
    masks = [_random_tree(n, r) for n in m]
    paths = [[j for j in range(n) if t[-1] >> j & 1] for n, t in zip(m, masks)]                # the last draft and its ancestors
    assert all(p != list(range(len(p))) for p in paths)                                        # with others between them
    mask = _ints([_signed(v) for t in masks for v in t], torch.int64)
    shift = _ints([bin(v).count("1") - 1 - j for t in masks for j, v in enumerate(t)], torch.int64)      # depth - place
    both, counts = _ints([0, 1]), _ints(m)
    pools, tables = empty(), ext.page_tables(2, 8, N, "cuda")
    slots, pos, _, _ = ext.cache_reserve(tables, both, _ints(lens), page, sum(lens))
    append(pools, torch.cat(prompt), pos, slots)
    slots, pos, starts, base = ext.cache_reserve(tables, both, counts, page, sum(m))
    q = append(pools, drafts, pos + shift, slots)
    out = ext.tree_attn_paged(q, *pools, tables["block_table"], tables["seq_lens"], starts, max(m), tree_mask=mask, **kw)
    most = max(map(len, paths))
    ext.cache_accept(pools, tables, both, base, counts, _ints([p + [0] * (most - len(p)) for p in paths]),
                     _ints([len(p) for p in paths]), layout=layout)
    for b, path in enumerate(paths):
        alone, fresh, total = ext.page_tables(1, 8, N, "cuda"), empty(), lens[b] + len(path)
        first = sum(m[:b])
        chain = torch.cat([prompt[b], drafts[first:][path]])
        slots, pos, starts, _ = ext.cache_reserve(alone, _ints([0]), _ints([total]), page, total)
        q1 = append(fresh, chain, pos, slots)
        assert int(tables["seq_lens"][b]) == total
        ids, ids1 = tables["block_table"][b, :-(-total // page)].tolist(), alone["block_table"][0, :-(-total // page)].tolist()
        for x, y in zip(pools, fresh):
            assert torch.equal(R.tokens_of(x, ids, layout)[:total], R.tokens_of(y, ids1, layout)[:total])
        # and each row of the path was attended as the chain's token at that length; one kernel, two orders of the tokens:
        # each within its tolerance of the definition
        rows = [first + j for j in path]
        n = len(path)
        want = ext.tree_attn_paged(q1[lens[b]:], *fresh, alone["block_table"], alone["seq_lens"], _ints([0, n]), n, **kw)
        ks, vs = kw.get("k_scale", 1.0), kw.get("v_scale", 1.0)
        ref, spread, size = R.tree_attn(q1[lens[b]:], *fresh, alone["block_table"], alone["seq_lens"], _ints([0, n]), None,
                                        layout, hd ** -0.5, ks, vs)
        tol = R.tree_tolerance(ref, spread, size, q.dtype, total, 8.0)
        assert ((want.double() - ref).abs() <= tol).all()
        assert ((out[rows].double() - ref).abs() <= tol).all()
    assert tables["counters"][1] == 0
