"""The operators around the paged cache (tree attention, qk-norm + rotary + append, pages) through their public entry
points, against plain 64-bit restatements (tests/paged_ref.py).  Tolerances are sums of the roundings the kernels are
allowed to make, element by element (paged_ref.tree_tolerance; for the append half a step of the target type of the
result plus 2^-20 of the terms for fp32 arithmetic)."""
import random

import pytest
import torch

import paged_ref as R

pytestmark = pytest.mark.gpu


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _ints(v, dtype=torch.int32):
    return torch.tensor(v, dtype=dtype, device="cuda")


def _random_tree(n, r):
    rows = []
    for j in range(n):
        up = r.randrange(-1, j) if j else -1
        rows.append((rows[up] if up >= 0 else 0) | 1 << j)
    return rows


def _signed(v):
    return v - (1 << 64) if v >> 63 else v


class Case:
    """A batch of draft trees over a paged cache, with shuffled pages and three pages nobody uses."""

    def __init__(self, seed, lens, drafts, qh, kvh, hd, page, layout, dtype, kv, masks="tree", extra_rows=0, table_extra=1):
        r, g = random.Random(seed), _gen(seed)
        need = [-(-n // page) for n in lens]
        self.pages, width = sum(need) + 3, max(max(need), 1) + table_extra
        perm = list(range(self.pages))
        r.shuffle(perm)
        table = torch.full((len(lens), width), self.pages + 7, dtype=torch.int32)        # not read, or not visible
        at = 0
        for b, c in enumerate(need):
            table[b, :c] = torch.tensor(perm[at:at + c], dtype=torch.int32)
            at += c
        self.unused = perm[at:]
        starts, rows = [0], []
        for n in drafts:
            rows += _random_tree(n, r) if masks == "tree" else [r.getrandbits(64) for _ in range(n)]
            starts.append(starts[-1] + n)
        rows += [r.getrandbits(64) for _ in range(extra_rows)]
        self.q = torch.randn(starts[-1] + extra_rows, qh, hd, device="cuda", generator=g).to(R.DT[dtype])
        self.k = R.make_pool(layout, self.pages, kvh, page, hd, kv, g, "cuda")
        self.v = R.make_pool(layout, self.pages, kvh, page, hd, kv, g, "cuda")
        self.table, self.lens, self.starts = table.cuda(), _ints(lens), _ints(starts)
        self.mask = None if masks is None else _ints([_signed(v) for v in rows], torch.int64)
        self.most, self.layout, self.page, self.hd = max(1, max(drafts)), layout, page, hd
        self.ks, self.vs = (0.5, 2.0) if kv == "fp8" else (1.0, 1.0)
        self.scale = hd ** -0.5

    def run(self, ext, **kw):
        return ext.tree_attn_paged(kw.pop("q", self.q), self.k, self.v, self.table, self.lens, self.starts, self.most,
                                   tree_mask=self.mask, layout=self.layout, k_scale=self.ks, v_scale=self.vs, **kw)

    def check(self, got, q=None, scale=None, vmax=8.0):
        q, scale = self.q if q is None else q, self.scale if scale is None else scale
        ref, spread, size = R.tree_attn(q, self.k, self.v, self.table, self.lens, self.starts, self.mask, self.layout,
                                        scale, self.ks, self.vs)
        live = int(self.starts[-1])
        tol = R.tree_tolerance(ref, spread, size, q.dtype, int(self.lens.max()) + 64, vmax * self.vs)
        err = (got.double() - ref).abs()[:live]
        assert torch.isfinite(got[:live].float()).all()
        worst = (err / tol[:live]).max().item() if err.numel() else 0.0
        assert worst <= 1.0, worst
        return ref


TREES = [
    # lens, drafts, qh, kvh, hd, page, layout, dtype, kv, masks
    ([300], [5], 24, 4, 256, 16, "HND", "fp16", "fp16", "tree"),
    ([1], [1], 24, 4, 256, 16, "HND", "fp16", "fp16", "tree"),                   # a single token in all
    ([7, 64, 1], [7, 64, 1], 6, 1, 256, 16, "NHD", "fp16", "fp16", "tree"),      # no context: drafts alone
    ([129, 0, 128, 127], [3, 0, 1, 64], 12, 2, 256, 48, "HND", "bf16", "bf16", "tree"),    # an absent sequence
    ([1000, 17, 513], [64, 2, 33], 8, 8, 128, 32, "NHD", "fp16", "fp16", "tree"),           # no grouping, head 128
    ([2049, 255], [61, 20], 24, 4, 256, 16, "NHD", "fp16", "fp16", "tree"),      # several blocks of query rows
    ([777, 65], [9, 10], 40, 8, 128, 128, "HND", "bf16", "bf16", "tree"),
    ([640, 31, 90], [8, 8, 1], 24, 4, 256, 64, "NHD", "fp16", "fp8", "tree"),    # e4m3 cache
    ([640, 31, 90], [64, 8, 30], 16, 2, 128, 64, "HND", "bf16", "fp8", "tree"),
    ([500, 90], [16, 9], 32, 1, 128, 16, "HND", "fp16", "fp16", "tree"),         # all heads share one KV head
    ([450, 70, 16], [16, 5, 16], 3, 1, 256, 16, "HND", "fp16", "fp16", None),    # a chain of drafts
    ([450, 200], [64, 64], 4, 4, 128, 16, "NHD", "bf16", "bf16", None),
    ([130, 40, 64], [40, 40, 64], 6, 2, 256, 16, "HND", "fp16", "fp16", "bits"),  # any bits: rows that see nothing
    ([33] * 40, [1] * 40, 24, 4, 256, 16, "HND", "fp16", "fp16", None),          # plain decode of a batch
    ([9000], [4], 4, 1, 256, 16, "HND", "fp16", "fp16", "tree"),                 # few rows, a long cache
    ([20000, 3], [2, 3], 2, 1, 128, 16, "NHD", "fp16", "fp8", "tree"),
]


@pytest.mark.parametrize("i", range(len(TREES)))
def test_tree_attn_matches_the_definition(ext, i):
    c = Case(100 + i, *TREES[i])
    got = c.run(ext)
    c.check(got)
    assert torch.equal(got, c.run(ext))                              # fixed order of summation


def test_tree_attn_rows_that_see_nothing_give_zeros(ext):
    c = Case(7, [5, 40], [5, 40], 6, 2, 256, 16, "HND", "fp16", "fp16", "tree")
    c.mask[0] = 0
    c.mask[2] = 0
    c.mask[44] = 0
    got = c.run(ext)
    assert torch.count_nonzero(got[[0, 2, 44]]) == 0
    c.check(got)
    c.table[1, 0] = -1                                               # the first sixteen tokens are on no page
    c.check(c.run(ext))
    c.table[0, 0] = c.pages                                          # and the first sequence on none at all
    got = c.run(ext)
    assert torch.count_nonzero(got[:5]) == 0
    c.check(got)


@pytest.mark.parametrize("layout,kv,hd", [("HND", "fp16", 256), ("NHD", "fp8", 256), ("HND", "bf16", 128)])
def test_tree_attn_unseen_values_do_not_matter(ext, layout, kv, hd):
    """NaN and infinities behind the sequences' ends, on pages that are not used, and in drafts that some rows do not see."""
    dtype = "bf16" if kv == "bf16" else "fp16"
    c = Case(21, [200, 77, 130, 8], [20, 7, 64, 5], 12, 2, hd, 16, layout, dtype, kv)
    clean = c.run(ext)
    for bad in (float("nan"), float("inf")):
        for pool in (c.k, c.v):
            byte = 0x7F if kv == "fp8" else None
            for p in c.unused:
                R.raw(pool)[p] = bad if byte is None else byte
            for b, n in enumerate(c.lens.tolist()):
                if n % 16:
                    page = int(c.table[b, n // 16])
                    tail = R.raw(pool)[page][:, n % 16:] if layout == "HND" else R.raw(pool)[page][n % 16:]
                    tail.fill_(bad if byte is None else byte)
        assert torch.equal(c.run(ext), clean)
    # draft 3 of the third sequence holds NaN: the rows that see it change, no other bit does
    first, n, m = int(c.starts[2]), int(c.lens[2]), 64
    at = n - m + 3
    page = int(c.table[2, at // 16])
    for pool in (c.k, c.v):
        row = R.raw(pool)[page][:, at % 16] if layout == "HND" else R.raw(pool)[page][at % 16]
        row.fill_(float("nan") if kv != "fp8" else 0x7F)
    got = c.run(ext)
    sees = torch.zeros(c.q.shape[0], dtype=torch.bool, device="cuda")
    sees[first:first + m] = (c.mask[first:first + m] >> 3 & 1).bool()
    assert sees.any() and not sees[first:first + m].all()
    assert torch.equal(got[~sees], clean[~sees])
    assert torch.isnan(got[sees].float()).all()


def test_tree_attn_infinite_value_in_one_draft(ext):
    """An infinity in one dimension of V of one draft reaches that dimension of the rows that see it, nothing else."""
    c = Case(22, [150], [30], 8, 1, 256, 16, "HND", "fp16", "fp16")
    clean = c.run(ext)
    at = 150 - 30 + 2
    c.v[int(c.table[0, at // 16]), 0, at % 16, 77] = float("-inf")
    got = c.run(ext)
    sees = (c.mask >> 2 & 1).bool()
    assert torch.equal(got[~sees], clean[~sees])
    assert (got[sees][:, :, 77] == float("-inf")).all()
    other = torch.arange(256, device="cuda") != 77
    assert torch.equal(got[sees][:, :, other], clean[sees][:, :, other])


def test_tree_attn_peaked_scores_views_and_rows_behind(ext):
    """A large spread of scores (the running maximum moves often), q and out as views of wider rows, rows behind the
    last sequence left as they were, a scale of its own."""
    qh, kvh, hd = 24, 4, 256
    c = Case(31, [700, 90], [12, 3], qh, kvh, hd, 16, "HND", "fp16", "fp16", extra_rows=5)
    wide = torch.randn(20, (qh + 2 * kvh) * hd, device="cuda", generator=_gen(5)).half() * 3
    wide[15:] = float("nan")
    q = torch.as_strided(wide, (20, qh, hd), (wide.stride(0), hd, 1))
    buf = torch.full((20, qh * hd + 64), 7.0, device="cuda", dtype=torch.half)
    out = torch.as_strided(buf, (20, qh, hd), (buf.stride(0), hd, 1))
    got = c.run(ext, q=q, out=out, scale=0.3)
    assert got.data_ptr() == out.data_ptr()
    c.check(out, q=q, scale=0.3)
    assert (buf[15:] == 7).all() and (buf[:, qh * hd:] == 7).all()


def test_tree_attn_equals_decode_attn_for_single_tokens(ext):
    """One draft per sequence is decode attention: both kernels within the tolerance of the definition."""
    c = Case(41, [100, 1, 513, 64], [1, 1, 1, 1], 24, 4, 256, 16, "HND", "fp16", "fp16", None)
    got = c.run(ext)
    c.check(got)
    old = ext.decode_attn_paged(c.q, c.k, c.v, c.table, c.lens, 513)
    assert (got.float() - old.float()).abs().max().item() <= 4e-3


def test_tree_attn_long_offsets(ext):
    """Pages whose offsets pass 2^31 elements and 2^32 bytes."""
    g = _gen(3)
    pages, kvh, page, hd = 1100, 8, 1024, 256                            # 2.3e9 elements a pool
    k = torch.empty((pages, kvh, page, hd), dtype=torch.float16, device="cuda")
    v = torch.empty_like(k)
    ids = [1099, 3, 1050]
    for p in ids:
        k[p] = torch.randn(kvh, page, hd, device="cuda", generator=g)
        v[p] = torch.randn(kvh, page, hd, device="cuda", generator=g)
    q = torch.randn(6, 16, hd, device="cuda", generator=g).half()
    table, lens, starts = _ints([ids]), _ints([2100]), _ints([0, 6])
    got = ext.tree_attn_paged(q, k, v, table, lens, starts, 6)
    ref, spread, size = R.tree_attn(q, k, v, table, lens, starts, None, "HND", hd ** -0.5)
    tol = R.tree_tolerance(ref, spread, size, q.dtype, 2200, 8.0)
    assert ((got.double() - ref).abs() <= tol).all()


def test_tree_attn_lengths_beyond_the_table(ext):
    """A length beyond the table's pages is cut there; starts beyond the rows are cut too; max_drafts below a
    sequence's drafts leaves its later rows alone."""
    c = Case(51, [64], [4], 4, 1, 128, 16, "HND", "fp16", "fp16", None, table_extra=0)
    ref = c.run(ext)
    assert c.table.shape[1] == 4
    out = torch.zeros_like(c.q)
    ext.tree_attn_paged(c.q, c.k, c.v, c.table, c.lens, c.starts, 2, out=out)
    assert torch.equal(out[:2], ref[:2]) and torch.count_nonzero(out[2:]) == 0
    c.lens[0] = 1000
    got = c.run(ext)
    c.lens[0] = 64
    assert torch.equal(got, ref)
    c.starts[1] = 9
    out = torch.zeros((4, 4, 128), dtype=torch.half, device="cuda")
    c.run(ext, out=out)
    c.starts[1] = 4
    assert torch.equal(out, ref)


def test_tree_attn_streams_and_graphs(ext):
    """Captured and replayed with other lengths and trees in the same buffers; two graphs, and two streams at once."""
    c = Case(61, [900, 333, 16], [10, 30, 3], 24, 4, 256, 16, "HND", "fp16", "fp16")
    want = c.run(ext)
    out = torch.zeros_like(c.q)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        c.run(ext, out=out)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            c.run(ext, out=out)
            again = c.run(ext)
    torch.cuda.current_stream().wait_stream(st)
    out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want) and torch.equal(again, want)
    c.lens.copy_(_ints([60, 333, 3]))
    c.mask[10] = 1
    want2 = c.run(ext)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want2) and not torch.equal(out, want)
    outs = []
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    for s in streams * 3:
        with torch.cuda.stream(s):
            outs.append(c.run(ext))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want2) for o in outs)


def test_tree_attn_refusals(ext):
    c = Case(71, [64], [4], 4, 2, 128, 16, "HND", "fp16", "fp16")

    def bad(**kw):
        a = dict(q=c.q, k=c.k, v=c.v, table=c.table, lens=c.lens, starts=c.starts, most=4, tree_mask=c.mask)
        a.update(kw)
        args = [a.pop(n) for n in ("q", "k", "v", "table", "lens", "starts", "most")]
        with pytest.raises(RuntimeError):
            ext.tree_attn_paged(*args, **a)
    bad(q=c.q.cpu())
    bad(q=c.q.bfloat16())                                   # another type than the pools
    bad(q=c.q[:, :3])                                       # three heads over two
    bad(q=c.q[:, :, :64])
    bad(most=0)
    bad(most=65)
    bad(table=c.table.long())
    bad(table=c.table[:0])
    bad(lens=c.lens.long())
    bad(starts=c.starts[:1])
    bad(tree_mask=c.mask[:3])
    bad(tree_mask=c.mask.int())
    bad(layout="DNH")
    bad(k_scale=2.0)                                        # scales belong to e4m3 pools
    bad(out=torch.empty(4, 4, 128, device="cuda"))
    bad(k=c.k[:, :, :8], v=c.v[:, :, :8])                   # eight tokens per page
    bad(k=c.k[..., :64], v=c.v[..., :64], q=c.q[..., :64].contiguous())
    bad(v=c.v[:-1])
    out = ext.tree_attn_paged(c.q[:0], c.k, c.v, c.table, c.lens, c.starts * 0, 4)
    assert out.shape == (0, 4, 128)


# ------------------------------------------------------------------------------------------------ append
APPENDS = [
    # tokens, qh, kvh, hd, rot, pairs, norm, weights, page, layout, dtype, kv
    (1, 24, 4, 256, 256, False, True, True, 16, "HND", "fp16", "fp16"),
    (5, 24, 4, 256, 64, True, True, True, 16, "NHD", "bf16", "fp8"),
    (37, 3, 1, 256, 128, False, True, False, 7, "HND", "fp16", "fp8"),       # any page size
    (64, 7, 7, 128, 128, False, True, True, 32, "NHD", "bf16", "bf16"),      # an odd number of heads
    (100, 40, 8, 128, 32, False, True, True, 16, "HND", "fp16", "fp16"),
    (33, 1, 1, 128, 48, False, True, True, 16, "HND", "fp16", "fp16"),       # a rotation that is no power of two
    (33, 5, 1, 256, 96, True, True, True, 16, "HND", "bf16", "bf16"),
    (260, 24, 4, 256, 0, False, True, True, 64, "NHD", "fp16", "fp8"),       # not rotated
    (19, 12, 2, 256, 256, False, False, False, 16, "HND", "fp16", "fp16"),   # not normed
]


def _append_case(seed, T, qh, kvh, hd, rot, pairs, norm, weights, page, layout, dtype, kv, extra=0):
    g = _gen(seed)
    dt = R.DT[dtype]
    pages = -(-T // page) + 2
    qkv = (torch.randn(T, (qh + 2 * kvh) * hd + extra, device="cuda", generator=g) * 3).to(dt)
    ang = torch.rand(50, rot // 2, device="cuda", generator=g, dtype=torch.float64) * 6.28
    cos, sin = (torch.cos(ang).float(), torch.sin(ang).float()) if rot else (None, None)
    pos = torch.randint(0, 50, (T,), device="cuda", generator=g)
    perm = torch.randperm(pages * page, device="cuda", generator=g)[:T]
    w = [(1 + 0.3 * torch.randn(hd, device="cuda", generator=g)).to(dt) if weights else None for _ in range(2)]
    pools = [R.make_pool(layout, pages, kvh, page, hd, kv, g, "cuda") for _ in range(2)]
    scales = (0.25, 0.5) if kv == "fp8" else (1.0, 1.0)
    return qkv, cos, sin, pos, perm, w, pools, scales


def _rows(pool, slots, layout, page):
    p = R.raw(pool)
    return (p[slots // page, :, slots % page] if layout == "HND" else p[slots // page, slots % page]).view(pool.dtype).double()


def _close(got, ref, size, dtype):
    err = (got.double() - ref).abs()
    tol = ref.abs() * R.HALF_STEP[dtype] + R.TINY[dtype] + size * 2.0 ** -20 * (1 + R.HALF_STEP[dtype])
    assert (err <= tol).all(), (err / tol).max().item()


@pytest.mark.parametrize("i", range(len(APPENDS)))
def test_append_matches_the_definition(ext, i):
    T, qh, kvh, hd, rot, pairs, norm, weights, page, layout, dtype, kv = APPENDS[i]
    qkv, cos, sin, pos, slots, w, pools, scales = _append_case(200 + i, *APPENDS[i], extra=64)
    eps = 1e-5 if norm else None
    old = [p.clone() for p in pools]
    src = qkv.clone()
    q, k, v, size = R.append(src, cos, sin, pos, qh, kvh, hd, w[0], w[1], eps, pairs)
    kw = dict(q_weight=w[0], k_weight=w[1], eps=eps, interleaved=pairs, layout=layout, k_scale=scales[0], v_scale=scales[1])
    out = torch.full((T, qh, hd), 9.0, dtype=qkv.dtype, device="cuda")
    got = ext.qk_norm_rope_append(qkv, cos, sin, pos, slots, *pools, qh, q_out=out, **kw)
    assert got.data_ptr() == out.data_ptr() and torch.equal(qkv, src)
    _close(out, q, size[:, :qh], qkv.dtype)
    dt = pools[0].dtype
    _close(_rows(pools[0], slots, layout, page), k / scales[0], size[:, qh:] / scales[0], dt)
    _close(_rows(pools[1], slots, layout, page), v / scales[1], v.abs() / scales[1], dt)
    rest = torch.ones(pools[0].shape[0] * page, dtype=torch.bool, device="cuda")
    rest[slots] = False
    rest = rest.nonzero()[:, 0]
    for a, b in zip(pools, old):
        assert torch.equal(_rows(a, rest, layout, page), _rows(b, rest, layout, page))
    # in place: the same queries, the same cache, keys and values of qkv as they were
    new = [p.clone() for p in old]
    got = ext.qk_norm_rope_append(qkv, cos, sin, pos, slots, *new, qh, **kw)
    assert got.data_ptr() == qkv.data_ptr() and torch.equal(got, out)
    assert torch.equal(qkv[:, qh * hd:], src[:, qh * hd:])
    assert all(torch.equal(R.raw(a), R.raw(b)) for a, b in zip(pools, new))


def test_append_padding_positions_and_saturation(ext):
    qkv, cos, sin, pos, slots, w, pools, _ = _append_case(300, 12, 4, 2, 128, 128, False, True, True, 16, "HND", "fp16", "fp8")
    total = pools[0].shape[0] * 16
    slots[3], slots[5], pos[7], pos[8] = -1, total, -1, 50          # not appended, not appended, left, left
    slots[9], pos[9] = 2 ** 40, 2 ** 33
    old, src = [p.clone() for p in pools], qkv.clone()
    q = torch.full((12, 4, 128), 9.0, dtype=torch.half, device="cuda")
    ext.qk_norm_rope_append(qkv, cos, sin, pos, slots, *pools, 4, q_weight=w[0], k_weight=w[1], eps=1e-6, q_out=q)
    ok = torch.tensor([i not in (7, 8, 9) for i in range(12)], device="cuda")
    ref = R.append(src[ok], cos, sin, pos[ok], 4, 2, 128, w[0], w[1], 1e-6, False)
    _close(q[ok], ref[0], ref[3][:, :4], q.dtype)
    assert (q[~ok] == 9).all() and torch.equal(qkv, src)
    wrote = torch.tensor([i not in (3, 5, 7, 8, 9) for i in range(12)], device="cuda")
    rest = torch.ones(total, dtype=torch.bool, device="cuda")
    rest[slots[wrote]] = False
    rest = rest.nonzero()[:, 0]
    for a, b in zip(pools, old):
        assert torch.equal(_rows(a, rest, "HND", 16), _rows(b, rest, "HND", 16))
    qkv.fill_(60000.0)
    qkv[:, ::2] = -60000.0
    pos.zero_()
    slots.copy_(torch.arange(12, device="cuda"))
    ext.qk_norm_rope_append(qkv, None, None, pos, slots, *pools, 4, eps=None, k_scale=0.01, v_scale=0.01)
    for p in pools:
        assert (_rows(p, slots, "HND", 16).abs() == 448).all()
    qkv.zero_()                                                     # a zero head stays zero
    got = ext.qk_norm_rope_append(qkv, cos, sin, pos, slots, *pools, 4, eps=1e-6)
    assert torch.count_nonzero(got) == 0 and torch.count_nonzero(_rows(pools[0], slots, "HND", 16)) == 0


def test_append_contiguous_cache_equals_rope_append(ext):
    """A contiguous cache is a pool of one page per sequence: the step that rope_append does, at a position of each
    sequence's own."""
    g = _gen(9)
    B, qh, kvh, cap = 5, 6, 2, 40
    qkv = torch.randn(B, (qh + 2 * kvh) * 256, device="cuda", generator=g).half()
    ang = torch.rand(cap, 128, device="cuda", generator=g) * 6.28
    cos, sin = torch.cos(ang).half(), torch.sin(ang).half()
    a = [torch.zeros(B, kvh, cap, 256, device="cuda", dtype=torch.half) for _ in range(2)]
    b = [torch.zeros_like(t) for t in a]
    x, y = qkv.clone(), qkv.clone()
    ext.rope_append(x, cos[17].contiguous(), sin[17].contiguous(), *a, 17, qh)
    pos = torch.full((B,), 17, dtype=torch.int64, device="cuda")
    ext.qk_norm_rope_append(y, cos.float(), sin.float(), pos, torch.arange(B, device="cuda") * cap + 17, *b, qh, eps=None)
    assert (x.float() - y.float()).abs().max().item() <= 2 * 2.0 ** -11 * 8
    assert torch.equal(a[1], b[1]) and (a[0].float() - b[0].float()).abs().max().item() <= 2 * 2.0 ** -11 * 8


def test_append_refusals(ext):
    qkv, cos, sin, pos, slots, w, pools, _ = _append_case(301, 6, 4, 2, 128, 128, False, True, True, 16, "HND", "fp16", "fp16")

    def bad(**kw):
        a = dict(qkv=qkv, cos=cos, sin=sin, pos=pos, slots=slots, k=pools[0], v=pools[1], qh=4, q_weight=w[0])
        a.update(kw)
        args = [a.pop(n) for n in ("qkv", "cos", "sin", "pos", "slots", "k", "v", "qh")]
        with pytest.raises(RuntimeError):
            ext.qk_norm_rope_append(*args, **a)
    bad(qkv=qkv.cpu())
    bad(qkv=qkv.float())
    bad(qkv=qkv[:, :-8])
    bad(qkv=qkv[:, 1:])
    bad(cos=cos.half(), sin=sin.half())
    bad(cos=None)
    bad(cos=cos[:, :20].contiguous(), sin=sin[:, :20].contiguous())     # 40 is no multiple of 16
    bad(cos=torch.ones(4, 72, device="cuda"), sin=torch.ones(4, 72, device="cuda"))       # more than the head
    bad(pos=pos.int())
    bad(slots=slots[:5])
    bad(q_weight=w[0][:64])
    bad(q_weight=w[0].float())
    bad(qh=0)
    bad(qh=5)
    bad(eps=-1.0)
    bad(eps=float("nan"))
    bad(k_scale=0.5)
    bad(q_out=torch.empty(6, 4, 128, device="cuda"))
    bad(v=pools[1][:1])
    got = ext.qk_norm_rope_append(qkv[:0], cos, sin, pos[:0], slots[:0], *pools, 4)
    assert got.shape == (0, 4, 128)


# ------------------------------------------------------------------------------------------------ pages
def _pools_of(ext, layers, pages, kvh, page, hd, kv, layout, seed, stacked=True):
    g = _gen(seed)
    t = torch.randn((2 * layers,) + R.pool_shape(layout, pages, kvh, page, hd), device="cuda", generator=g).to(R.DT[kv])
    return t if stacked else [t[i].clone() for i in range(2 * layers)]


def _grow(ext, tables, ref, seqs, counts, page, room=None):
    room = sum(max(c, 0) for c in counts) if room is None else room
    got = ext.cache_reserve(tables, _ints(seqs), _ints(counts), page, room)
    want = ref.reserve(seqs, counts, page, room)
    assert [t.tolist() for t in got] == [list(w) for w in want]
    assert ref.same(tables) == []
    return got


@pytest.mark.parametrize("page,layout,kv,stacked", [(16, "HND", "fp16", True), (16, "NHD", "fp8", False), (5, "HND", "fp8", True)])
def test_pages_random_life(ext, page, layout, kv, stacked):
    """Forks, growth and frees in random order against lists, with the data of forked pages."""
    r = random.Random(page)
    S, N, kvh, hd = 24, 60, 2, 128
    tables = ext.page_tables(S, 12, N, "cuda")
    pools = _pools_of(ext, 2, N, kvh, page, hd, kv, layout, 5, stacked)
    ref = R.Pages(tables)
    for step in range(60):
        live = [s for s in range(S) if ref.lens[s]]
        empty = [s for s in range(S) if not ref.held[s]]
        what = r.choice(["grow", "fork", "free", "grow"])
        if what == "grow":
            seqs = r.sample(range(S), r.randint(1, 6))
            _grow(ext, tables, ref, seqs, [r.randint(0, 2 * page) for _ in seqs], page)
        elif what == "fork" and live and empty:
            kids = r.sample(empty, min(len(empty), r.randint(1, 6)))
            pars = [r.choice(live) for _ in kids]
            before = [p.clone() for p in pools]
            ref.copies = []
            ext.cache_fork(pools, tables, _ints(pars), _ints(kids), layout=layout)
            ref.fork(pars, kids, page)
            assert ref.same(tables) == []
            for now, was in zip(pools, before):
                for src, dst, rows in ref.copies:
                    if layout == "HND":
                        R.raw(was)[dst, :, :rows] = R.raw(was)[src, :, :rows]
                    else:
                        R.raw(was)[dst, :rows] = R.raw(was)[src, :rows]
                assert torch.equal(R.raw(now), R.raw(was))
        elif what == "free" and live:
            seqs = r.sample(live, r.randint(1, len(live)))
            if r.random() < 0.2:
                seqs.append(r.choice(empty or live))
            ext.cache_free(tables, _ints(seqs))
            ref.free(seqs)
            assert ref.same(tables) == []
        if ref.status:
            ref.status = 0
            tables["counters"][1] = 0
    rest = list(range(S))
    ext.cache_free(tables, _ints(rest))
    ref.free(rest)
    assert ref.same(tables) == [] and ref.left == N and set(ref.stack) == set(range(N)) and not any(ref.refs)


def test_pages_that_cannot_be_served(ext):
    page = 16
    tables = ext.page_tables(6, 4, 7, "cuda")
    pools = _pools_of(ext, 1, 7, 1, page, 128, "fp16", "HND", 6)
    ref = R.Pages(tables)
    _grow(ext, tables, ref, [0, 1], [40, 20], page)                 # three and two pages
    assert ref.left == 2 and ref.status == 0
    _grow(ext, tables, ref, [2, 3, 4, 1], [33, 16, 0, 1], page)     # three are not there; behind that nobody gets any
    assert ref.status == 1 and ref.lens[2:4] == [0, 0] and ref.lens[1] == 21
    _grow(ext, tables, ref, [3, 3, -1, 6, 0], [1, 1, 1, 1, -4], page)
    assert ref.status == 3 and ref.lens[3] == 1
    _grow(ext, tables, ref, [1], [100], page)                       # more than a row of the table holds
    assert ref.lens[1] == 21
    _grow(ext, tables, ref, [0, 1], [2, 5], page, room=4)           # more tokens than the outputs hold
    assert ref.lens[0] == 42 and ref.lens[1] == 21
    for pars, kids in (([0, 1], [4, 4]), ([0, 4], [4, 5]), ([0], [0]), ([0], [1]), ([9, 0], [5, -1])):
        ext.cache_fork(pools, tables, _ints(pars), _ints(kids))
        ref.fork(pars, kids, page)
        assert ref.same(tables) == [], (pars, kids)
        tables["counters"][1] = ref.status = 0
    ext.cache_free(tables, _ints([5, 5, 77, 4, -3, 4]))
    ref.free([5, 5, 77, 4, -3, 4])
    assert ref.same(tables) == [] and ref.status == 2


@pytest.mark.parametrize("n,most,layout,kv,page,kvh,hd,stacked", [
    (1, 5, "HND", "fp16", 16, 4, 256, True), (9, 64, "NHD", "fp8", 16, 2, 256, True), (20, 16, "HND", "bf16", 48, 8, 128, False),
    (3, 1, "NHD", "fp16", 7, 1, 128, True), (2, 64, "HND", "fp16", 16, 4, 256, True)])
def test_accept_moves_the_path(ext, n, most, layout, kv, page, kvh, hd, stacked):
    r = random.Random(n)
    draft = most
    base = [r.randint(0, 40) for _ in range(n)]
    width = -(-(40 + draft) // page)
    N = n * width + 1
    tables = ext.page_tables(n + 2, width, N, "cuda")
    pools = _pools_of(ext, 2, N, kvh, page, hd, kv, layout, 8, stacked)
    ref = R.Pages(tables)
    seqs = r.sample(range(n + 2), n)
    _grow(ext, tables, ref, seqs, base, page)
    _grow(ext, tables, ref, seqs, [draft] * n, page)
    taken = [r.randint(0, most) for _ in range(n)]
    taken[0] = most
    # ascending paths as a tree gives them, and one in any order with a draft twice
    path = [sorted(r.sample(range(draft), most)) for _ in range(n)]
    path[-1] = [r.randrange(draft) for _ in range(most)]
    before = [p.clone() for p in pools]
    ext.cache_accept(pools, tables, _ints(seqs), _ints(base), _ints([draft] * n), _ints(path), _ints(taken), layout=layout)
    at = lambda s, t: (ref.table[s][t // page], t % page)                                   # noqa: E731
    for now, was in zip(pools, before):
        new = was.clone()
        for i, s in enumerate(seqs):
            for j in range(taken[i]):
                (a, x), (b, y) = at(s, base[i] + path[i][j]), at(s, base[i] + j)
                if layout == "HND":
                    R.raw(new)[b, :, y] = R.raw(was)[a, :, x]
                else:
                    R.raw(new)[b, y] = R.raw(was)[a, x]
        assert torch.equal(R.raw(now), R.raw(new))
    for i, s in enumerate(seqs):
        ref.lens[s] = base[i] + taken[i]
    assert ref.same(tables) == []


def test_accept_that_cannot_be_served(ext):
    """A path outside the drafts, more taken than drafted, a shared page, a sequence twice: left as they were."""
    page = 16
    tables = ext.page_tables(6, 4, 20, "cuda")
    pools = _pools_of(ext, 1, 20, 2, page, 128, "fp16", "NHD", 9)
    ref = R.Pages(tables)
    _grow(ext, tables, ref, [0, 1, 2, 3], [20, 20, 28, 5], page)
    ext.cache_fork(pools, tables, _ints([2]), _ints([4]), layout="NHD")    # shares the first page of 2
    ref.fork([2], [4], page)
    before, lens = pools.clone(), list(ref.lens)

    def call(seqs, base, drafts, path, taken):
        ext.cache_accept(pools, tables, _ints(seqs), _ints(base), _ints(drafts), _ints(path), _ints(taken), layout="NHD")
        status = int(tables["counters"][1])
        tables["counters"][1] = 0
        return status
    assert call([0], [10], [4], [[1, 4]], [2]) == 2
    assert call([0], [10], [4], [[1, -1]], [2]) == 2
    assert call([0], [10], [4], [[1, 2]], [3]) == 2
    assert call([0], [30], [4], [[1, 2]], [2]) == 2                 # behind the pages of the sequence
    assert call([9], [0], [4], [[1, 2]], [2]) == 2
    assert call([2], [12], [4], [[1, 2]], [2]) == 2                 # would write the shared page
    assert torch.equal(pools, before) and tables["seq_lens"].tolist() == lens
    assert call([2], [12], [4], [[0, 1]], [2]) == 0                 # nothing to move: the shared page is not written
    assert tables["seq_lens"].tolist()[2] == 14 and torch.equal(pools, before)
    assert call([1, 1], [10, 10], [4, 4], [[2, 3], [1, 3]], [2, 1]) == 2       # the first entry counts
    assert tables["seq_lens"].tolist()[1] == 12


def test_pages_refusals(ext):
    tables = ext.page_tables(4, 4, 8, "cuda")
    pools = torch.zeros(2, 8, 2, 16, 128, device="cuda", dtype=torch.half)
    one = _ints([0])
    for f in (lambda: ext.cache_fork(pools, tables, one, _ints([1, 2])),
              lambda: ext.cache_fork(pools[:, :7], tables, one, one),
              lambda: ext.cache_fork([pools[0], pools[0]], tables, one, one),
              lambda: ext.cache_fork([], tables, one, one),
              lambda: ext.cache_fork(pools[0], tables, one, one),
              lambda: ext.cache_fork(pools.cpu(), tables, one, one),
              lambda: ext.cache_fork(pools, tables, one.long(), one),
              lambda: ext.cache_fork(pools, tables, torch.zeros(1025, dtype=torch.int32, device="cuda"),
                                     torch.zeros(1025, dtype=torch.int32, device="cuda")),
              lambda: ext.cache_fork(torch.zeros(257, 8, 1, 1, 128, device="cuda", dtype=torch.half), tables, one, one),
              lambda: ext.cache_reserve(tables, one[:0], one[:0], 16, 0),
              lambda: ext.cache_reserve(tables, one, one, 0, 1),
              lambda: ext.cache_reserve(tables, one, one, 16, -1),
              lambda: ext.cache_reserve(dict(tables, held=tables["held"][:3]), one, one, 16, 1),
              lambda: ext.cache_reserve(dict(tables, refs=tables["refs"].long()), one, one, 16, 1),
              lambda: ext.cache_accept(pools, tables, one, one, one, torch.zeros(1, 65, dtype=torch.int32, device="cuda"), one),
              lambda: ext.cache_accept(pools, tables, one, one, one, one, one),
              lambda: ext.cache_free(dict(tables, counters=tables["counters"][:1]), one)):
        with pytest.raises(RuntimeError):
            f()
    ext.cache_fork(pools, tables, one[:0], one[:0])
    ext.cache_free(tables, one[:0])
    assert R.Pages(tables).left == 8 and int(tables["counters"][1]) == 0


# ------------------------------------------------------------------------------------------------ together
@pytest.mark.parametrize("kv", ["fp16", "fp8"])
def test_a_speculative_step(ext, kv):
    """Prompt, fork, a tree of drafts, verification, the accepted path, and the next token: after the step the cache
    holds what appending prompt and accepted tokens one after the other would have put there, and decode attention over
    it agrees; captured as one CUDA graph it gives the same."""
    g, r = _gen(77), random.Random(77)
    layers, qh, kvh, hd, page, N, S = 2, 6, 2, 256, 16, 40, 6
    scales = (0.5, 0.25) if kv == "fp8" else (1.0, 1.0)
    ang = torch.arange(200, device="cuda")[:, None] / 10000.0 ** (torch.arange(128, device="cuda") / 128)
    cos, sin = torch.cos(ang).float(), torch.sin(ang).float()
    weights = [(1 + 0.1 * torch.randn(hd, device="cuda", generator=g)).half() for _ in range(2)]
    ones = [torch.zeros(R.pool_shape("HND", N, kvh, page, hd), device="cuda", dtype=torch.half).to(R.DT[kv]) for _ in range(2 * layers)]
    width = (qh + 2 * kvh) * hd

    def append(pools, qkv, positions, slots):
        return [ext.qk_norm_rope_append(qkv[i], cos, sin, positions, slots, pools[2 * i], pools[2 * i + 1], qh,
                                        q_weight=weights[0], k_weight=weights[1], k_scale=scales[0], v_scale=scales[1],
                                        q_out=torch.empty(qkv[i].shape[0], qh, hd, dtype=torch.half, device="cuda"))
                for i in range(layers)]
    n, m = 37, 9                                                     # prompt, drafts
    prompt = [torch.randn(n, width, device="cuda", generator=g).half() for _ in range(layers)]
    drafts = [torch.randn(2 * m, width, device="cuda", generator=g).half() for _ in range(layers)]
    masks = [_random_tree(m, r), _random_tree(m, r)]
    paths = [[j for j in range(m) if masks[b][m - 1] >> j & 1] for b in range(2)]
    path = _ints([p + [0] * (m - len(p)) for p in paths])
    taken = _ints([len(p) for p in paths])
    mask = _ints([v for b in masks for v in b], torch.int64)
    tables = ext.page_tables(S, 8, N, "cuda")
    slots, positions, _, _ = ext.cache_reserve(tables, _ints([2]), _ints([n]), page, n)
    append(ones, prompt, positions, slots)
    state = {k: v.clone() for k, v in tables.items()}
    pools0 = [p.clone() for p in ones]
    parent, child, both, counts = _ints([2]), _ints([5]), _ints([2, 5]), _ints([m, m])

    def step(pools, tables):
        ext.cache_fork(pools, tables, parent, child)
        slots, positions, starts, base = ext.cache_reserve(tables, both, counts, page, 2 * m + 3)
        pad = [torch.cat([d, d[:3]]) for d in drafts]
        q = append(pools, pad, positions, slots)
        table, lens = tables["block_table"][both.long()], tables["seq_lens"][both.long()]
        outs = [ext.tree_attn_paged(q[i], pools[2 * i], pools[2 * i + 1], table, lens, starts, m, tree_mask=mask_pad,
                                    k_scale=scales[0], v_scale=scales[1]) for i in range(layers)]
        ext.cache_accept(pools, tables, both, base, counts, path, taken)
        return q, outs
    mask_pad = torch.cat([mask, mask[:3]])
    q, outs = step(ones, tables)
    assert int(tables["counters"][1]) == 0
    # every verified row equals the row of a chain of its ancestors appended one after the other
    for b in range(2):
        last = 2 * m if b else m
        i = last - 1                                                 # the deepest row of the accepted path
        alone = ext.page_tables(S, 8, N, "cuda")
        fresh = [torch.zeros_like(p) for p in pools0]
        sl, po, _, _ = ext.cache_reserve(alone, _ints([0]), _ints([n]), page, n)
        append(fresh, prompt, po, sl)
        count = len(paths[b])
        sl, po, _, _ = ext.cache_reserve(alone, _ints([0]), _ints([count]), page, count)
        # in the tree a draft's position is its place among the drafts: give the chain the same rotations
        po = n + _ints(paths[b], torch.int64)
        append(fresh, [d[b * m:][paths[b]] for d in drafts], po, sl)
        s = [2, 5][b]
        total = n + count
        assert int(tables["seq_lens"][s]) == total == int(alone["seq_lens"][0])
        for a, c in zip(ones, fresh):
            ids = tables["block_table"][s, :-(-total // page)].tolist()
            ids2 = alone["block_table"][0, :-(-total // page)].tolist()
            assert torch.equal(R.tokens_of(a, ids, "HND")[:total], R.tokens_of(c, ids2, "HND")[:total])
        for layer in range(layers):
            want = ext.decode_attn_paged(q[layer][i:i + 1], fresh[2 * layer], fresh[2 * layer + 1], alone["block_table"][:1],
                                         alone["seq_lens"][:1], total, k_scale=scales[0], v_scale=scales[1])
            # two kernels, each within half a step of probabilities and output (values up to 4.5): twice that
            assert (outs[layer][i].float() - want[0].float()).abs().max().item() <= 4 * 2.0 ** -11 * 4.5
    # the same step as one graph on a copy of the state
    pools2, tables2 = [p.clone() for p in pools0], {k: v.clone() for k, v in state.items()}
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            _, outs2 = step(pools2, tables2)
    torch.cuda.current_stream().wait_stream(st)
    graph.replay()
    torch.cuda.synchronize()
    for x, y in zip(outs, outs2):
        assert torch.equal(x[:2 * m], y[:2 * m])
    assert all(torch.equal(R.raw(a), R.raw(b)) for a, b in zip(ones, pools2))
    assert all(torch.equal(tables[k], tables2[k]) for k in tables)
    # and back: every page is free again
    ext.cache_free(tables, both)
    assert tables["counters"].tolist() == [N, 0] and not tables["refs"].any()
