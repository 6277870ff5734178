"""More of the operators around the paged cache: the sizes at which the kernels change their way (many tokens, many
sequences, many pools, sixteen tiles of query rows), scales of both signs, NaN queries, pools that are views, pages cut
back into shared ones, a broken state, waits that run out.  Oracles and tolerances as in test_gpu_paged.py."""
import random

import pytest
import torch

import paged_ref as R
from test_gpu_paged import Case, _append_case, _close, _gen, _grow, _ints, _pools_of, _rows

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------------------ tree attention
SHAPES = [
    # lens, drafts, qh, kvh, hd, page, layout, dtype, kv, masks
    ([900, 64], [64, 64], 32, 1, 128, 16, "HND", "fp16", "fp16", "tree"),            # sixteen tiles of query rows
    ([400, 66, 130], [64, 2, 63], 64, 2, 256, 32, "NHD", "bf16", "fp8", "tree"),
    ([5000, 130, 4097, 1], [64, 3, 17, 1], 16, 2, 256, 48, "NHD", "bf16", "fp8", "tree"),
    ([3000, 2999, 385, 128], [30, 64, 1, 5], 16, 4, 128, 16, "HND", "bf16", "bf16", "tree"),
    ([3000, 2999, 385, 128], [30, 64, 1, 5], 16, 4, 128, 16, "HND", "fp16", "fp8", "tree"),
    ([70, 0, 0, 5, 300], [0, 4, 0, 5, 0], 6, 2, 256, 16, "HND", "fp16", "fp16", "tree"),    # no drafts; drafts of length zero
]


@pytest.mark.parametrize("i", range(len(SHAPES)))
def test_tree_attn_shapes(ext, i):
    c = Case(500 + i, *SHAPES[i])
    got = c.run(ext)
    c.check(got)
    assert torch.equal(got, c.run(ext))


@pytest.mark.parametrize("seed", range(12))
def test_tree_attn_random_batches(ext, seed):
    r = random.Random(seed)
    hd, kvh, G = r.choice([128, 256]), r.choice([1, 2, 3, 8]), r.choice([1, 2, 3, 5, 6, 8])
    kv = r.choice(["fp16", "bf16", "fp8"])
    dtype = r.choice(["fp16", "bf16"]) if kv == "fp8" else kv
    B = r.choice([1, 2, 5, 11])
    drafts = [r.choice([0, 1, 2, 7, 16, 33, 64]) for _ in range(B)]
    lens = [max(n, r.choice([n, n + 1, 127, 128, 129, 511, 1300])) for n in drafts]
    c = Case(600 + seed, lens, drafts, kvh * G, kvh, hd, r.choice([16, 32, 80]), r.choice(["HND", "NHD"]), dtype, kv,
             r.choice(["tree", "bits", None]), extra_rows=r.choice([0, 3]))
    out = torch.full_like(c.q, 7.0)
    got = c.run(ext, out=out)
    c.check(got)
    assert (out[int(c.starts[-1]):] == 7).all()


def test_tree_attn_more_sequences_than_threads(ext):
    r = random.Random(1)
    drafts = [r.randint(0, 3) for _ in range(700)]
    lens = [n + r.randint(0, 40) for n in drafts]
    c = Case(520, lens, drafts, 4, 2, 128, 16, "HND", "fp16", "fp16", "tree")
    c.check(c.run(ext))


@pytest.mark.parametrize("kv", ["fp16", "fp8"])
@pytest.mark.parametrize("scale", [-0.07, 0.0, 1e-30, 1.5])
def test_tree_attn_scales(ext, kv, scale):
    c = Case(530, [300, 20, 2000], [7, 20, 3], 6, 2, 256, 16, "NHD", "fp16", kv, "bits")
    c.check(c.run(ext, scale=scale), scale=scale)


@pytest.mark.parametrize("n", [200, 30000])
def test_tree_attn_nan_query_row(ext, n):
    """A NaN in one head of one query row makes that row NaN and no other, split over CTAs or not."""
    c = Case(540, [n], [5], 8, 2, 128, 16, "HND", "fp16", "fp16", "tree")
    clean = c.run(ext)
    c.q[3, 5, 17] = float("nan")
    got = c.run(ext)
    assert torch.isnan(got[3, 5]).all()
    hit = torch.zeros(5, 8, dtype=torch.bool, device="cuda")
    hit[3, 5] = True
    assert torch.equal(got[~hit], clean[~hit])


def test_tree_attn_pools_that_are_views(ext):
    """K and V halves of one tensor; a contiguous cache as a pool of one page per sequence; pages of different order."""
    c = Case(550, [500, 77], [6, 9], 12, 2, 128, 16, "HND", "fp16", "fp16", "tree")
    want = c.run(ext)
    both = torch.stack([c.k, c.v], 1)
    c.k, c.v = both[:, 0], both[:, 1]
    assert torch.equal(c.run(ext), want)
    cap = 512
    k, v = (torch.full((2, 2, cap, 128), float("nan"), dtype=torch.half, device="cuda") for _ in range(2))
    for b, n in enumerate([500, 77]):
        ids = c.table[b, :-(-n // 16)].long()
        for flat, pool in ((k, c.k), (v, c.v)):
            flat[b, :, :n] = pool[ids].transpose(0, 1).reshape(2, -1, 128)[:, :n]
    got = ext.tree_attn_paged(c.q, k, v, _ints([[0], [1]]), c.lens, c.starts, c.most, tree_mask=c.mask)
    assert torch.equal(got, want)
    c.q = torch.as_strided(torch.cat([c.q.flatten(1), c.q.flatten(1)], 1), c.q.shape, (2 * 12 * 128, 128, 1))
    assert torch.equal(c.run(ext), want)


def test_tree_attn_calls_back_to_back(ext):
    """Calls that follow each other on a stream, of different shapes, and so in each other's workspace."""
    cases = [Case(560 + i, *a) for i, a in enumerate([
        ([9000], [4], 4, 1, 256, 16, "HND", "fp16", "fp16", "tree"), ([40, 3000], [7, 30], 12, 2, 128, 16, "NHD", "bf16", "fp8", "tree"),
        ([1], [1], 24, 4, 256, 16, "HND", "fp16", "fp16", "tree"), ([700] * 9, [16] * 9, 16, 2, 128, 16, "HND", "fp16", "fp16", None)])]
    want = [c.run(ext) for c in cases]
    torch.cuda.synchronize()
    order = [random.Random(2).randrange(4) for _ in range(60)]
    got = [cases[i].run(ext) for i in order]
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i]) for g, i in zip(got, order))


def test_tree_attn_refuses_scales_that_are_not_finite(ext):
    c = Case(570, [64], [4], 4, 2, 128, 16, "HND", "fp16", "fp16")
    for s in (float("nan"), float("inf"), float("-inf"), 1e39):
        with pytest.raises(RuntimeError):
            c.run(ext, scale=s)


def test_tree_attn_wait_runs_out_and_reports(ext):
    L = ext.lib()
    dev = torch.device("cuda", torch.cuda.current_device())
    torch.cuda.synchronize()
    assert ext.tree_attn_status(dev) == 0
    try:
        assert L.exl3_tree_attn_selftest_wait(3000, None) == 0
        torch.cuda.synchronize()
        assert ext.tree_attn_status(dev) != 0
    finally:
        assert L.exl3_tree_attn_status_reset() == 0
    assert ext.tree_attn_status(dev) == 0
    c = Case(580, [300, 40], [5, 7], 24, 4, 256, 16, "HND", "fp16", "fp8", "tree")
    c.check(c.run(ext))
    assert ext.tree_attn_status(dev) == 0
    assert L.exl3_tree_attn_selftest_wait(0, None) == -1


# ------------------------------------------------------------------------------------------------ append, many tokens
MANY = [
    # tokens, qh, kvh, hd, rot, pairs, norm, weights, page, layout, dtype, kv
    (1025, 6, 2, 256, 256, False, True, True, 16, "HND", "fp16", "fp16"),
    (1100, 5, 3, 128, 128, False, True, True, 16, "NHD", "bf16", "fp8"),       # odd numbers of heads, two to a warp
    (1030, 9, 1, 128, 48, True, True, True, 7, "HND", "fp16", "fp8"),
    (1200, 24, 4, 256, 64, True, True, False, 32, "NHD", "bf16", "bf16"),
    (1029, 3, 1, 256, 96, False, False, False, 16, "HND", "fp16", "fp16"),
    (1027, 4, 2, 128, 0, False, True, True, 16, "HND", "bf16", "bf16"),
]


@pytest.mark.parametrize("i", range(len(MANY)))
def test_append_of_many_tokens(ext, i):
    """A warp per token instead of a CTA: against the definition, and token by token as the other kernel does it."""
    T, qh, kvh, hd, rot, pairs, norm, weights, page, layout, dtype, kv = MANY[i]
    qkv, cos, sin, pos, slots, w, pools, scales = _append_case(700 + i, *MANY[i], extra=8)
    eps = 1e-5 if norm else None
    slots[1], pos[2], pos[T - 1] = -1, -1, 50 if rot else -1        # not appended, left as it is, left as it is
    src, old = qkv.clone(), [p.clone() for p in pools]
    ok = torch.ones(T, dtype=torch.bool, device="cuda")
    ok[2] = ok[T - 1] = False
    wrote = ok.clone()
    wrote[1] = False
    q, k, v, size = R.append(src[ok], cos, sin, pos[ok], qh, kvh, hd, w[0], w[1], eps, pairs)
    kw = dict(q_weight=w[0], k_weight=w[1], eps=eps, interleaved=pairs, layout=layout, k_scale=scales[0], v_scale=scales[1])
    out = torch.full((T, qh, hd), 9.0, dtype=qkv.dtype, device="cuda")
    ext.qk_norm_rope_append(qkv, cos, sin, pos, slots, *pools, qh, q_out=out, **kw)
    assert torch.equal(qkv, src) and (out[~ok] == 9).all()
    _close(out[ok], q, size[:, :qh], qkv.dtype)
    keep, dt = wrote[ok], pools[0].dtype
    _close(_rows(pools[0], slots[wrote], layout, page), k[keep] / scales[0], size[keep][:, qh:] / scales[0], dt)
    _close(_rows(pools[1], slots[wrote], layout, page), v[keep] / scales[1], v[keep].abs() / scales[1], dt)
    rest = torch.ones(pools[0].shape[0] * page, dtype=torch.bool, device="cuda")
    rest[slots[wrote]] = False
    rest = rest.nonzero()[:, 0]
    for a, b in zip(pools, old):
        assert torch.equal(_rows(a, rest, layout, page), _rows(b, rest, layout, page))
    got = ext.qk_norm_rope_append(qkv, cos, sin, pos, slots, *old, qh, **kw)               # in place
    assert torch.equal(got[ok], out[ok]) and torch.equal(qkv[~ok], src[~ok]) and torch.equal(qkv[:, qh * hd:], src[:, qh * hd:])
    assert all(torch.equal(R.raw(a), R.raw(b)) for a, b in zip(pools, old))


# ------------------------------------------------------------------------------------------------ pages
def test_accept_in_many_pools(ext):
    """So many pools and sequences that a CTA takes several pools, the last one fewer."""
    n, pools_n, pages, kvh, page, hd, most = 48, 127, 110, 4, 16, 128, 16
    g, r = _gen(11), random.Random(11)
    pools = torch.randn((pools_n,) + R.pool_shape("HND", pages, kvh, page, hd), device="cuda", generator=g, dtype=torch.half)
    tables = ext.page_tables(n, 4, pages, "cuda")
    ref = R.Pages(tables)
    seqs = list(range(n))
    r.shuffle(seqs)
    _grow(ext, tables, ref, seqs, [r.randint(1, 14) for _ in seqs], page)
    _, _, _, base = _grow(ext, tables, ref, seqs, [16] * n, page)
    path = [r.sample(range(16), 16) for _ in seqs]
    taken = [r.randint(0, 16) for _ in seqs]
    want = pools.clone()
    for i, s in enumerate(seqs):
        at = [int(base[i]) + p for p in path[i][:taken[i]]]
        to = [int(base[i]) + j for j in range(taken[i])]
        page_of = lambda t: ref.table[s][t // page]
        if at:
            rows = pools[:, [page_of(t) for t in at], :, [t % page for t in at]]             # [rows, pools, kvh, hd]
            want[:, [page_of(t) for t in to], :, [t % page for t in to]] = rows
    ext.cache_accept(pools, tables, _ints(seqs), base, _ints([16] * n), _ints(path), _ints(taken))
    assert torch.equal(pools, want)
    for i, s in enumerate(seqs):
        ref.lens[s] = int(base[i]) + taken[i]
    assert ref.same(tables) == []


def test_accept_nothing_from_an_empty_path(ext):
    tables = ext.page_tables(2, 4, 8, "cuda")
    ref = R.Pages(tables)
    pools = _pools_of(ext, 1, 8, 2, 16, 128, "fp16", "HND", 1)
    _grow(ext, tables, ref, [0, 1], [20, 3], 16)
    _, _, _, base = _grow(ext, tables, ref, [0, 1], [4, 4], 16)
    old = pools.clone()
    ext.cache_accept(pools, tables, _ints([0, 1]), base, _ints([4, 4]), torch.empty((2, 0), dtype=torch.int32, device="cuda"), _ints([0, 0]))
    ref.lens = [20, 3]
    assert ref.same(tables) == [] and torch.equal(pools, old)
    ext.cache_accept(pools[:1], tables, _ints([0]), base[:1], _ints([4]), _ints([[0]]), _ints([0]))          # one pool alone


def test_reserve_does_not_hand_out_shared_pages(ext):
    """A sequence cut back into a page that it shares gets no room there; after the others gave it up it does."""
    page = 16
    tables = ext.page_tables(4, 6, 20, "cuda")
    ref = R.Pages(tables)
    pools = _pools_of(ext, 1, 20, 2, page, 128, "fp16", "HND", 1)
    _grow(ext, tables, ref, [0], [40], page)
    ext.cache_fork(pools, tables, _ints([0]), _ints([1]))
    ref.fork([0], [1], page)
    ext.cache_accept(pools, tables, _ints([0]), _ints([20]), _ints([20]), _ints([[0]]), _ints([0]))     # to 20 of 40 tokens
    ref.lens[0] = 20
    assert ref.same(tables) == []
    slots, pos, starts, base = ext.cache_reserve(tables, _ints([0, 1]), _ints([2, 3]), page, 5)
    assert slots[:2].tolist() == [-1, -1] and base.tolist() == [20, 40] and starts.tolist() == [0, 2, 5]
    ref.status |= ext.PAGES_BAD
    ref.lens[1] = 43
    assert ref.same(tables) == [] and (slots[2:] >= 0).all()
    assert ext.cache_reserve(tables, _ints([0]), _ints([0]), page, 0)[3].tolist() == [20]              # no tokens: nothing to refuse
    ext.cache_free(tables, _ints([1]))
    ref.free([1])
    _grow(ext, tables, ref, [0], [30], page)


def test_pages_broken_stack(ext):
    """Page numbers that are none, in the stack: status bit, table entry -1, nothing else written."""
    page = 16
    tables = ext.page_tables(3, 4, 6, "cuda")
    pools = _pools_of(ext, 1, 6, 2, page, 128, "fp16", "HND", 1)
    tables["free_list"][4] = 99                                      # the second page to be taken
    old = pools.clone()
    slots = ext.cache_reserve(tables, _ints([0]), _ints([30]), page, 30)[0]
    assert (slots[:16] == torch.arange(16, device="cuda")).all() and (slots[16:] == -1).all()
    assert tables["counters"].tolist() == [4, ext.PAGES_BAD] and tables["block_table"][0, :2].tolist() == [0, -1]
    ext.cache_fork(pools, tables, _ints([0]), _ints([2]))            # its partial page is that one
    assert torch.equal(pools, old) and tables["block_table"][2, :2].tolist() == [0, -1]
    assert tables["refs"].tolist() == [2, 0, 0, 0, 0, 0]
    ext.cache_free(tables, _ints([0, 2]))
    assert tables["refs"].tolist() == [0] * 6 and tables["held"].tolist() == [0] * 3
