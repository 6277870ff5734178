"""Long contexts, at tolerances that a single token left out or counted twice would pass by far, and page tables of
thousands of entries."""
import random

import pytest
import torch

import paged_ref as R
from test_gpu_paged import Case, _grow, _ints, _pools_of

pytestmark = pytest.mark.gpu

LONG = [
    # lens, drafts, qh, kvh, hd, page, layout, dtype, kv
    ([32768], [61], 24, 4, 256, 16, "HND", "fp16", "fp16"),                    # three tiles of rows, each split over CTAs
    ([20001, 130, 32768], [64, 3, 17], 24, 4, 256, 16, "NHD", "fp16", "fp8"),
    ([20001, 4097, 15000], [33, 64, 1], 32, 8, 128, 32, "HND", "bf16", "bf16"),
    ([30000, 129, 9999], [5, 64, 30], 32, 1, 128, 16, "HND", "bf16", "fp8"),
    ([32767], [1], 24, 4, 256, 64, "HND", "fp16", "fp16"),                     # one token
]


@pytest.mark.parametrize("i", range(len(LONG)))
def test_tree_attn_counts_every_token_once(ext, i):
    """Queries of zero: every visible token has the same weight, and V holds whole numbers, so that the sums over V and
    over the weights are exact in fp32 and the result is their quotient: two fp32 roundings and the output's."""
    c = Case(800 + i, *LONG[i])
    g = torch.Generator(device="cuda").manual_seed(i)
    c.q.zero_()
    c.v.copy_(torch.randint(-8, 9, c.v.shape, generator=g, device="cuda").to(c.v.dtype))       # whole numbers to 8: exact in e4m3
    fp8 = c.v.dtype == R.DT["fp8"]
    kw = dict(k_scale=0.5, v_scale=0.25) if fp8 else {}
    out = ext.tree_attn_paged(c.q, c.k, c.v, c.table, c.lens, c.starts, c.most, tree_mask=c.mask, layout=c.layout, **kw)
    kvh = LONG[i][3]
    G = c.q.shape[1] // kvh
    for b, n in enumerate(c.lens.tolist()):
        lo, hi = c.starts[b].item(), c.starts[b + 1].item()
        v = R.tokens_of(c.v, c.table[b, :-(-n // LONG[i][5])].tolist(), c.layout)[:n] * kw.get("v_scale", 1.0)     # [n, kvh, hd]
        ctx = n - (hi - lo)
        whole = v[:ctx].sum(0)
        bits = (c.mask[lo:hi, None] >> torch.arange(hi - lo, device="cuda")) & 1
        total = whole[None] + torch.einsum("ij,jhd->ihd", bits.double(), v[ctx:])
        want = (total / (ctx + bits.sum(1))[:, None, None]).repeat_interleave(G, 1)
        tol = want.abs() * (R.HALF_STEP[c.q.dtype] * (1 + 2.0 ** -20) + 2 * 2.0 ** -24) + R.TINY[c.q.dtype]
        assert ((out[lo:hi].double() - want).abs() <= tol).all()


@pytest.mark.parametrize("i", range(len(LONG)))
def test_tree_attn_finds_one_token(ext, i):
    """Every (draft, head of its group) looks for a token of its own, whose score lies 110 above the others': their weights,
    2^-158, are zero in fp32.  The found one's weight is off by at most 159 * 2^-24 (the fp32 rounding of its exponent), less
    than half a step of the output's type, so that the result is that token's V, bit for bit."""
    lens, drafts, qh, kvh, hd, page, layout, _, kv = LONG[i]
    c = Case(820 + i, *LONG[i])
    r = random.Random(i)
    G = qh // kvh
    fp8 = kv == "fp8"
    ks, vs = (0.5, 0.25) if fp8 else (1.0, 1.0)
    c.k.copy_(torch.zeros_like(c.k, dtype=torch.float).to(c.k.dtype))
    c.q.zero_()
    big = 32.0                                                       # exact in every type; 32 * 32 = 1024
    scale = 110.0 / (big * big)
    where = {}
    for b, n in enumerate(lens):
        m = drafts[b]
        lo, ctx = c.starts[b].item(), n - m
        # what is looked for: dimension d of K of one token of the context, the first and last of blocks among them
        edges = [t for t in range(0, ctx, 128)] + [t - 1 for t in range(128, ctx + 1, 128)] + [max(ctx - 1, 0)]
        count = min(hd, m * G, ctx)
        tokens = r.sample(sorted(set(edges)), min(len(set(edges)), count // 2))
        tokens += r.sample([t for t in range(ctx) if t not in set(tokens)], count - len(tokens))
        tok = torch.tensor(tokens, device="cuda")
        pg, off = c.table[b, tok // page].long(), tok % page
        dims = torch.arange(count, device="cuda")
        value = torch.full((count,), big / ks, device="cuda").to(c.k.dtype)
        raw, val = R.raw(c.k), R.raw(value)
        for h in range(kvh):
            if layout == "HND":
                raw[pg, h, off, dims] = val
            else:
                raw[pg, off, h, dims] = val
        for row in range(m):
            for x in range(G):
                d = (row * G + x) % count
                for h in range(kvh):
                    c.q[lo + row, h * G + x, d] = big
        where[b] = (tokens, count)
    out = ext.tree_attn_paged(c.q, c.k, c.v, c.table, c.lens, c.starts, c.most, tree_mask=c.mask, layout=layout, scale=scale,
                              k_scale=ks, v_scale=vs)
    for b, n in enumerate(lens):
        tokens, count = where[b]
        lo, m = c.starts[b].item(), drafts[b]
        v = R.tokens_of(c.v, c.table[b, :-(-n // page)].tolist(), layout)[:n] * vs
        at = torch.tensor(tokens, device="cuda")[torch.arange(m * G, device="cuda") % count]
        want = v[at].view(m, G, kvh, hd).transpose(1, 2).reshape(m, qh, hd).to(c.q.dtype)
        assert torch.equal(out[lo:lo + m], want)


def test_pages_of_long_sequences(ext):
    """Reserve, fork and free of more pages than one round of threads, some shared by several, one sequence in the middle freed first."""
    page, N, S, kvh, hd = 16, 5000, 12, 1, 128
    tables = ext.page_tables(S, 1500, N, "cuda")
    pools = _pools_of(ext, 1, N, kvh, page, hd, "fp16", "HND", 3)
    ref = R.Pages(tables)
    lens = [16000, 5, 7001, 24000 - 3, 16 * 700]
    _grow(ext, tables, ref, [0, 1, 2, 3, 4], lens, page)
    _grow(ext, tables, ref, [4, 1, 0], [900, 1600, 33], page)
    before = pools.clone()
    pars, kids = [0, 2, 3, 0, 4], [5, 6, 7, 8, 9]
    ref.copies = []
    ext.cache_fork(pools, tables, _ints(pars), _ints(kids))
    ref.fork(pars, kids, page)
    assert ref.same(tables) == [] and ref.status == 0
    for src, dst, rows in ref.copies:
        before[:, dst, :, :rows] = before[:, src, :, :rows]
    assert torch.equal(pools, before)
    _grow(ext, tables, ref, [5, 9, 7], [300, 1, 2], page)
    for some in ([0], [3, 6, 9, 0], [7, 1, 8]):
        ext.cache_free(tables, _ints(some))
        ref.free(some)
        assert ref.same(tables) == []
        if some == [0]:
            _grow(ext, tables, ref, [0, 10], [2000, 4000], page)
    rest = list(range(S))
    ext.cache_free(tables, _ints(rest))
    ref.free(rest)
    assert ref.same(tables) == [] and ref.left == N and set(ref.stack) == set(range(N)) and not any(ref.refs)
