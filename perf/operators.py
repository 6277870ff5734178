"""The speculative-decoding operators around the KV cache, as a decoder step meets them: their cases, their plain
forms in elementary torch, and their definitions in 64 bits.

  tree     attention of a tree of drafted tokens over a paged cache (a multi-token query with an ancestor mask)
  append   norms of the query and key heads, rotary embedding and the append to the paged cache, one pass
  accept   the accepted path of a draft tree moved to the front of its place in the cache, in every layer
  branch   sequences forked (full pages shared, the partial page copied in every layer), grown, and freed again

The head counts (24 query / 4 KV heads of 256) are the 27B decoder's of `bench_model.py`; 32 / 8 heads of 128 stand
for the other common layout."""
import random

import torch

own = False

MASK64 = (1 << 64) - 1


# ------------------------------------------------------------------------------------------------ cases
def listed():
    big = dict(qh=24, kvh=4, hd=256)
    return [
        # latency of one user's verify step early in a chat
        dict(name="tree 1x5 ctx 300", op="tree", batch=1, lo=300, hi=300, dlo=5, dhi=5, page=16, layout="HND",
             dtype="fp16", kv="fp16", **big),
        # one user, a long document, a wide draft tree
        dict(name="tree 1x61 ctx 32768", op="tree", batch=1, lo=32768, hi=32768, dlo=61, dhi=61, page=16, layout="HND",
             dtype="fp16", kv="fp16", **big),
        # a serving batch with an fp8 cache, token-major pages
        dict(name="tree 32x8 to 4096 fp8", op="tree", batch=32, lo=200, hi=4096, dlo=8, dhi=8, page=64, layout="NHD",
             dtype="fp16", kv="fp8", **big),
        # ragged trees, bf16, heads of 128
        dict(name="tree 16x1..64 bf16 hd128", op="tree", batch=16, lo=700, hi=8192, dlo=1, dhi=64, page=32,
             layout="HND", dtype="bf16", kv="bf16", qh=32, kvh=8, hd=128),
        # a full serving batch, the largest cache
        dict(name="tree 64x16 to 8192", op="tree", batch=64, lo=1000, hi=8192, dlo=16, dhi=16, page=16, layout="NHD",
             dtype="fp16", kv="fp16", **big),
        # the drafts of one sequence
        dict(name="append 5", op="append", tokens=5, rot=256, pairs="half", page=16, layout="HND", dtype="fp16",
             kv="fp16", pad=0, **big),
        # a serving batch's drafts into an fp8 cache, partial rotary, adjacent pairs, padded to a captured size
        dict(name="append 1024 bf16 fp8", op="append", tokens=1024, rot=64, pairs="adjacent", page=64, layout="NHD",
             dtype="bf16", kv="fp8", pad=24, **big),
        # a prompt
        dict(name="append 16384", op="append", tokens=16384, rot=256, pairs="half", page=16, layout="HND",
             dtype="fp16", kv="fp16", pad=0, **big),
        # one user's accepted path in all 64 layers
        dict(name="accept 1 of 16", op="accept", batch=1, draft=16, most=5, ctx=150, page=16, layout="HND", kv="fp16",
             layers=64, kvh=4, hd=256),
        # a serving batch's
        dict(name="accept 64 of 16", op="accept", batch=64, draft=16, most=8, ctx=90, page=16, layout="NHD",
             kv="fp16", layers=64, kvh=4, hd=256),
        # four samples of one prompt
        dict(name="branch 1 to 4", op="branch", parents=1, children=4, grow=7, ctx=333, page=16, layout="HND",
             kv="fp16", layers=64, kvh=4, hd=256),
        # parallel sampling in a serving batch, fp8 cache, larger pages
        dict(name="branch 16 to 96 fp8", op="branch", parents=16, children=96, grow=16, ctx=250, page=64,
             layout="NHD", kv="fp8", layers=64, kvh=4, hd=256),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["tree", "tree", "append", "accept", "branch"])
    qh, kvh, hd = rng.choice([(24, 4, 256), (12, 2, 256), (3, 1, 256), (8, 1, 256), (32, 8, 128), (40, 8, 128), (7, 7, 128)])
    page, layout = rng.choice([16, 32, 48, 64, 128]), rng.choice(["HND", "NHD"])
    dtype = rng.choice(["fp16", "bf16"])
    kv = rng.choice([dtype, dtype, "fp8"])
    if op == "tree":
        batch = _log(rng, 1, 64)
        hi = _log(rng, 20, 8192 if batch > 8 else 32768)
        while batch * hi * kvh * hd > 64 * 8192 * 1024:
            hi = hi * 2 // 3
        dhi = _log(rng, 1, 64 if batch <= 16 else 20)
        return dict(op=op, batch=batch, lo=max(dhi, int(hi * rng.uniform(0.05, 1))), hi=max(hi, dhi),
                    dlo=rng.choice([1, dhi]), dhi=dhi, page=page, layout=layout, dtype=dtype, kv=kv, qh=qh, kvh=kvh, hd=hd)
    if op == "append":
        return dict(op=op, tokens=_log(rng, 1, 16384), rot=rng.choice([hd, hd // 2, hd // 4]),
                    pairs=rng.choice(["half", "adjacent"]), page=page, layout=layout, dtype=dtype, kv=kv,
                    pad=rng.choice([0, rng.randint(1, 40)]), qh=qh, kvh=kvh, hd=hd)
    layers = _log(rng, 2, 64)
    if op == "accept":
        draft = _log(rng, 2, 64)
        return dict(op=op, batch=_log(rng, 1, 64 if draft <= 16 else 12), draft=draft, most=rng.randint(1, min(draft, 12)),
                    ctx=rng.randint(1, 90), page=rng.choice([16, 32]), layout=layout, kv=kv, layers=layers, kvh=4, hd=hd)
    parents = _log(rng, 1, 16)
    return dict(op=op, parents=parents, children=parents * rng.randint(1, 6), grow=rng.randint(1, 20),
                ctx=rng.randint(1, 250), page=rng.choice([16, 32, 64]), layout=layout, kv=kv, layers=layers, kvh=4, hd=hd)


def _lens(case):
    """(context length, draft count) of every sequence; the first has the longest context, the last the shortest."""
    r = random.Random("%s %s %s %s" % (case["batch"], case["lo"], case["hi"], case["dhi"]))
    B = case["batch"]
    lens = sorted((r.randint(case["lo"], case["hi"]) for _ in range(B)), reverse=True)
    lens[0] = case["hi"]
    drafts = [r.randint(case["dlo"], case["dhi"]) for _ in range(B)]
    drafts[-1] = case["dhi"]
    order = list(range(1, B))
    r.shuffle(order)
    order = [0] + order
    return [max(lens[i], drafts[i]) for i in order], [drafts[i] for i in order]


def _paths(case):
    """(base length, accepted path) of every sequence: the path ascends, as a walk from the root of a tree does."""
    r = random.Random("%s %s %s" % (case["batch"], case["draft"], case["ctx"]))
    out = []
    for _ in range(case["batch"]):
        n = r.randint(1, case["most"])
        out.append((r.randint((case["ctx"] + 1) // 2, case["ctx"]), sorted(r.sample(range(case["draft"]), n))))
    return out


def _parents(case):
    """(length of every parent, parent of every child)."""
    r = random.Random("%s %s %s" % (case["parents"], case["children"], case["ctx"]))
    lens = [r.randint((case["ctx"] + 1) // 2, case["ctx"]) for _ in range(case["parents"])]
    return lens, [i % case["parents"] for i in range(case["children"])]


def _size(kv):
    return 1 if kv == "fp8" else 2


def work(case):
    op, e = case["op"], _size(case["kv"])
    if op == "tree":
        lens, drafts = _lens(case)
        qh, kvh, hd = case["qh"], case["kvh"], case["hd"]
        return dict(bytes=sum(2 * n * kvh * hd * e for n in lens) + sum(drafts) * (2 * qh * hd * 2 + 8),
                    flops=sum(4 * n * d * qh * hd for n, d in zip(lens, drafts)))
    if op == "append":
        T, P, qh, kvh, hd = case["tokens"], case["pad"], case["qh"], case["kvh"], case["hd"]
        return dict(bytes=T * ((2 * qh + 2 * kvh) * hd * 2 + 2 * kvh * hd * e + case["rot"] * 4 + 16) + P * 2 * qh * hd * 2,
                    flops=(T + P) * (qh + kvh) * hd * 7)
    row = 2 * case["layers"] * case["kvh"] * case["hd"] * e                  # bytes of a token in all layers
    if op == "accept":
        return dict(bytes=sum(2 * row * sum(1 for j, p in enumerate(path) if p != j) + 4 * len(path) for _, path in _paths(case)) + 1, flops=0)
    lens, parent = _parents(case)
    pg = case["page"]
    return dict(bytes=sum(2 * row * (lens[p] % pg) + 24 * (-(-lens[p] // pg)) for p in parent) + 1, flops=0)


# ------------------------------------------------------------------------------------------------ inputs
def _dtype(name):
    return {"fp16": torch.float16, "bf16": torch.bfloat16, "fp8": torch.float8_e4m3fn}[name]


def _values(shape, kv, g, scale=1.0):
    """Normal values in the cache's type, filled in pieces."""
    t = torch.empty(shape, dtype=_dtype(kv), device="cuda")
    flat = t.view(-1)
    for at in range(0, flat.numel(), 1 << 27):
        piece = flat[at:at + (1 << 27)]
        piece.copy_(torch.randn(piece.numel(), device="cuda", generator=g) * scale)
    return t


def _pool_shape(case, pages):
    page, kvh, hd = case["page"], case["kvh"], case["hd"]
    return (pages, kvh, page, hd) if case["layout"] == "HND" else (pages, page, kvh, hd)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, page = case["op"], case["page"]

    def ints(v, dtype=torch.int32):
        return torch.tensor(v, dtype=dtype, device="cuda")

    def pages_of(n):
        return torch.randperm(n, device="cuda", generator=g).to(torch.int32)

    if op == "tree":
        lens, drafts = _lens(case)
        B, width = len(lens), -(-max(lens) // page)
        need = [-(-n // page) for n in lens]
        total = sum(need) + 3
        perm, table, at = pages_of(total).cpu(), torch.zeros((B, width), dtype=torch.int32), 0
        for b in range(B):
            table[b, :need[b]] = perm[at:at + need[b]]
            at += need[b]
        r, rows, starts = random.Random(seed), [], [0]
        for n in drafts:                                   # a random tree: every draft hangs below an earlier one
            seen = []
            for j in range(n):
                up = r.randrange(max(0, j - 6), j) if j else -1
                seen.append((seen[up] if up >= 0 else 0) | 1 << j)
            rows += [v - (1 << 64) if v >> 63 else v for v in seen]
            starts.append(starts[-1] + n)
        T, qh, hd = starts[-1], case["qh"], case["hd"]
        fp8 = case["kv"] == "fp8"
        return dict(case=case, q=torch.randn((T, qh, hd), device="cuda", generator=g).to(_dtype(case["dtype"])),
                    k=_values(_pool_shape(case, total), case["kv"], g, 1.5 if not fp8 else 3.0),
                    v=_values(_pool_shape(case, total), case["kv"], g), table=table.cuda(), lens=ints(lens),
                    starts=ints(starts), mask=ints(rows, torch.int64), most=case["dhi"],
                    k_scale=0.5 if fp8 else 1.0, v_scale=0.25 if fp8 else 1.0)
    if op == "append":
        T, P, qh, kvh, hd, rot = (case[k] for k in ("tokens", "pad", "qh", "kvh", "hd", "rot"))
        pages = -(-T // page) + 5
        longest = max(4096, T)
        ang = torch.arange(longest, device="cuda", dtype=torch.float64)[:, None] \
            / 10000.0 ** (torch.arange(rot // 2, device="cuda", dtype=torch.float64) / (rot // 2))
        slots = torch.full((T + P,), -1, dtype=torch.int64, device="cuda")
        where = torch.arange(T, device="cuda")
        slots[:T] = pages_of(pages).long()[where // page] * page + where % page
        pos = torch.zeros((T + P,), dtype=torch.int64, device="cuda")
        pos[:T] = where + torch.randint(0, longest - T + 1, (1,), device="cuda", generator=g)
        dt = _dtype(case["dtype"])
        qkv = (torch.randn((T + P, (qh + 2 * kvh) * hd), device="cuda", generator=g) * 2).to(dt)
        fp8 = case["kv"] == "fp8"
        return dict(case=case, qkv=qkv, q_out=torch.zeros((T + P, qh, hd), dtype=dt, device="cuda"),
                    cos=torch.cos(ang).float(), sin=torch.sin(ang).float(), pos=pos, slots=slots,
                    qw=(1 + 0.2 * torch.randn(hd, device="cuda", generator=g)).to(dt),
                    kw=(1 + 0.2 * torch.randn(hd, device="cuda", generator=g)).to(dt),
                    k=_values(_pool_shape(case, pages), case["kv"], g), v=_values(_pool_shape(case, pages), case["kv"], g),
                    k_scale=0.25 if fp8 else 1.0, v_scale=0.5 if fp8 else 1.0)
    if op == "accept":
        paths = _paths(case)
        B, width = len(paths), -(-(case["ctx"] + case["draft"]) // page)
        total = B * width
        most = case["most"]
        tables = dict(block_table=pages_of(total).view(B, width).contiguous(),
                      seq_lens=ints([n + case["draft"] for n, _ in paths]),
                      held=ints([-(-(n + case["draft"]) // page) for n, _ in paths]),
                      refs=torch.ones(total, dtype=torch.int32, device="cuda"),
                      free_list=torch.zeros(total, dtype=torch.int32, device="cuda"), counters=ints([0, 0]))
        return dict(case=case, pools=_values((2 * case["layers"],) + _pool_shape(case, total), case["kv"], g), tables=tables,
                    seqs=torch.arange(B, dtype=torch.int32, device="cuda"), base=ints([n for n, _ in paths]),
                    drafts=ints([case["draft"]] * B), path=ints([p + [0] * (most - len(p)) for _, p in paths]),
                    taken=ints([len(p) for _, p in paths]))
    lens, parent = _parents(case)
    n, grow = len(parent), case["grow"]
    width = -(-(case["ctx"] + grow) // page)
    need = [-(-x // page) for x in lens]
    total = sum(need) + n * (1 + -(-grow // page)) + 2
    perm = pages_of(total)
    table, at = torch.zeros((len(lens) + n, width), dtype=torch.int32, device="cuda"), 0
    for i, c in enumerate(need):
        table[i, :c] = perm[at:at + c]
        at += c
    free = torch.zeros(total, dtype=torch.int32, device="cuda")
    free[:total - at] = perm[at:]
    refs = torch.ones(total, dtype=torch.int32, device="cuda")
    refs[perm[at:].long()] = 0
    tables = dict(block_table=table, seq_lens=ints(lens + [0] * n), held=ints(need + [0] * n), refs=refs, free_list=free,
                  counters=ints([total - at, 0]))
    return dict(case=case, pools=_values((2 * case["layers"],) + _pool_shape(case, total), case["kv"], g), tables=tables,
                parents=ints(parent), children=torch.arange(len(lens), len(lens) + n, dtype=torch.int32, device="cuda"),
                counts=ints([grow] * n), tokens=n * grow)


# ------------------------------------------------------------------------------------------------ plain forms
def _bytes(t):
    return t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t


def _cached(pool, table, case):
    """The tokens of every sequence, [batch, kv_heads, width * page, hd] in 32 bits."""
    got = _bytes(pool)[table.long()].view(pool.dtype).float()
    if case["layout"] == "NHD":
        got = got.transpose(2, 3)
    return got.transpose(1, 2).flatten(2, 3)


def _plain_tree(s):
    case = s["case"]
    q, kvh, hd, n = s["q"], case["kvh"], case["hd"], s["most"]
    starts, lens = s["starts"].long(), s["lens"].long()
    B, G = lens.numel(), case["qh"] // kvh
    first, count = starts[:-1], starts[1:] - starts[:-1]
    i = torch.arange(n, device=q.device)
    row = (first[:, None] + i).clamp(max=q.shape[0] - 1)                                      # [B, n]
    q4 = q[row].float().view(B, n, kvh, G, hd).permute(0, 2, 1, 3, 4).reshape(B, kvh, n * G, hd)
    k, v = _cached(s["k"], s["table"], case), _cached(s["v"], s["table"], case)
    t = torch.arange(k.shape[2], device=q.device)
    j = t[None, :] - (lens - count)[:, None]                                                  # draft number of a position
    bit = (s["mask"][row][:, :, None] >> j.clamp(0, 63)[:, None, :]) & 1
    see = (t[None, :] < lens[:, None])[:, None, :] & ((j < 0)[:, None, :] | (bit != 0))        # [B, n, L]
    see = see[:, None, :, None, :].expand(B, 1, n, G, t.numel()).reshape(B, 1, n * G, t.numel())
    v = torch.where((t[None, :] < lens[:, None])[:, None, :, None], v, 0.0)
    sc = torch.where(see, (q4 @ k.transpose(2, 3)) * (hd ** -0.5 * s["k_scale"]), float("-inf"))
    top = sc.amax(-1, keepdim=True)
    p = torch.exp(sc - torch.where(top == float("-inf"), 0.0, top))
    total = p.sum(-1, keepdim=True)
    o = (p @ v) * (s["v_scale"] / torch.where(total == 0, 1.0, total))
    o = o.view(B, kvh, n, G, hd).permute(0, 2, 1, 3, 4).reshape(B, n, kvh * G, hd)
    b = torch.bucketize(torch.arange(q.shape[0], device=q.device), starts[1:], right=True)    # sequence of a draft
    return o[b, torch.arange(q.shape[0], device=q.device) - first[b]].to(q.dtype)


def _plain_append(s):
    case, qkv = s["case"], s["qkv"]
    qh, kvh, hd, rot, page, T = (case[k] for k in ("qh", "kvh", "hd", "rot", "page", "tokens"))
    x = qkv[:, :(qh + kvh) * hd].float().view(-1, qh + kvh, hd)
    w = torch.cat([s["qw"].float().expand(qh, hd), s["kw"].float().expand(kvh, hd)])
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w
    c, n = s["cos"][s["pos"]][:, None], s["sin"][s["pos"]][:, None]
    if case["pairs"] == "half":
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        turned = torch.cat([a * c - b * n, b * c + a * n], -1)
    else:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack([a * c - b * n, b * c + a * n], -1).flatten(-2)
    x = torch.cat([turned, x[..., rot:]], -1)
    s["q_out"].copy_(x[:, :qh])
    at, off = s["slots"][:T] // page, s["slots"][:T] % page
    for pool, new, scale in ((s["k"], x[:T, qh:], s["k_scale"]),
                             (s["v"], qkv[:T, (qh + kvh) * hd:].float().view(T, kvh, hd), s["v_scale"])):
        new = new / scale
        new = _bytes((new.clamp(-448, 448) if pool.dtype == torch.float8_e4m3fn else new).to(pool.dtype))
        raw = _bytes(pool)
        if case["layout"] == "HND":
            raw[at, :, off] = new
        else:
            raw[at, off] = new
    return dict(q=s["q_out"], k=s["k"], v=s["v"])


def _plain_accept(s):
    case, t = s["case"], s["tables"]
    page, raw = case["page"], _bytes(s["pools"])
    j = torch.arange(s["path"].shape[1], device=raw.device)
    seqs, base = s["seqs"].long(), s["base"].long()[:, None]
    src = base + torch.where(j < s["taken"][:, None], s["path"].long(), j)       # behind the path: onto itself
    dst = base + j
    table = t["block_table"][seqs].long()
    a, b = table.gather(1, src // page), table.gather(1, dst // page)
    if case["layout"] == "HND":
        raw[:, b, :, dst % page] = raw[:, a, :, src % page]
    else:
        raw[:, b, dst % page] = raw[:, a, src % page]
    t["seq_lens"][seqs] = (s["base"] + s["taken"])
    return dict(pools=s["pools"], seq_lens=t["seq_lens"], status=t["counters"][1])


def _plain_branch(s):
    case, t = s["case"], s["tables"]
    page, raw = case["page"], _bytes(s["pools"])
    table, lens, held, refs, free, counters = (t[k] for k in ("block_table", "seq_lens", "held", "refs", "free_list", "counters"))
    par, kid = s["parents"].long(), s["children"].long()
    n, idx = kid.numel(), torch.arange(table.shape[1], device=raw.device)
    # fork: full pages are shared, a partial one is copied to a page from the top of the free list
    size = lens[par].long()
    full, rest = size // page, size % page
    part = (rest > 0).long()
    left = counters[0].long()
    new = free[(left - 1 - (part.cumsum(0) - part)).clamp(min=0)]
    rows = table[par]
    old = rows.gather(1, full[:, None].clamp(max=table.shape[1] - 1))[:, 0]
    shared = idx < full[:, None]
    fresh = (idx == full[:, None]) & (part[:, None] > 0)
    table[kid] = torch.where(shared, rows, torch.where(fresh, new[:, None], table[kid]))
    refs.index_add_(0, torch.where(shared, rows, 0).long().flatten(), shared.flatten().int())
    refs.index_add_(0, new.long(), part.int())
    to = torch.where(part > 0, new, old).long()
    keep = torch.arange(page, device=raw.device) < rest[:, None]
    keep = keep[:, None, :, None] if case["layout"] == "HND" else keep[:, :, None, None]
    raw[:, to] = torch.where(keep & (part > 0)[:, None, None, None], raw[:, old.long()], raw[:, to])
    lens[kid], held[kid] = size.int(), (full + part).int()
    left = left - part.sum()
    # reserve: pages for the new tokens, and where each goes
    after = size + s["counts"].long()
    have = held[kid].long()
    want = ((after + page - 1) // page - have).clamp(min=0)
    rank = (want.cumsum(0) - want)[:, None] + idx - have[:, None]
    mine = (idx >= have[:, None]) & (idx < (have + want)[:, None])
    got = free[(left - 1 - rank).clamp(0, free.numel() - 1)]
    table[kid] = torch.where(mine, got, table[kid])
    refs.index_add_(0, torch.where(mine, got, 0).long().flatten(), mine.flatten().int())
    left = left - want.sum()
    held[kid] = (have + want).int()
    ends = s["counts"].long().cumsum(0)
    tok = torch.arange(s["tokens"], device=raw.device)
    b = torch.bucketize(tok, ends, right=True)
    pos = size[b] + tok - (ends - s["counts"].long())[b]
    slots = table[kid][b, pos // page].long() * page + pos % page
    starts = torch.cat([ends.new_zeros(1), ends]).int()
    lens[kid] = after.int()
    # free: pages that nobody holds any more go back, the first one to the top of the list
    mine = idx < held[kid].long()[:, None]
    where = torch.where(mine, table[kid], 0).long()
    refs.index_add_(0, where.flatten(), -mine.flatten().int())
    last = torch.full_like(refs, -1, dtype=torch.int64).scatter_reduce_(
        0, where.flatten(), torch.where(mine.flatten(), torch.arange(mine.numel(), device=raw.device), -1), "amax")
    out = (mine & (refs[where] == 0)).flatten() & (last[where.flatten()] == torch.arange(mine.numel(), device=raw.device))
    place = left + out.sum() - out.long().cumsum(0)
    hole = torch.full_like(place, free.numel())
    padded = torch.cat([free, free.new_zeros(1)])
    padded[torch.where(out, place, hole)] = where.flatten().int()
    free.copy_(padded[:-1])
    counters[0] = left + out.sum()
    lens[kid] = 0
    held[kid] = 0
    return dict(pools=s["pools"], slots=slots, positions=pos, starts=starts, base=size.int(), **t)


# ------------------------------------------------------------------------------------------------ the framework's calls
def _ext():
    import os
    import sys
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "orcasaq2-kernel_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    from orcasaq2 import _ext as ext
    return ext


def _own_tree(s):
    return _ext().tree_attn_paged(s["q"], s["k"], s["v"], s["table"], s["lens"], s["starts"], s["most"],
                                  tree_mask=s["mask"], layout=s["case"]["layout"], k_scale=s["k_scale"], v_scale=s["v_scale"])


def _own_append(s):
    case = s["case"]
    _ext().qk_norm_rope_append(s["qkv"], s["cos"], s["sin"], s["pos"], s["slots"], s["k"], s["v"], case["qh"],
                               q_weight=s["qw"], k_weight=s["kw"], eps=1e-6, interleaved=case["pairs"] == "adjacent",
                               layout=case["layout"], q_out=s["q_out"], k_scale=s["k_scale"], v_scale=s["v_scale"])
    return dict(q=s["q_out"], k=s["k"], v=s["v"])


def _own_accept(s):
    t = s["tables"]
    _ext().cache_accept(s["pools"], t, s["seqs"], s["base"], s["drafts"], s["path"], s["taken"], layout=s["case"]["layout"])
    return dict(pools=s["pools"], seq_lens=t["seq_lens"], status=t["counters"][1])


def _own_branch(s):
    ext, t = _ext(), s["tables"]
    ext.cache_fork(s["pools"], t, s["parents"], s["children"], layout=s["case"]["layout"])
    slots, positions, starts, base = ext.cache_reserve(t, s["children"], s["counts"], s["case"]["page"], s["tokens"])
    ext.cache_free(t, s["children"])
    return dict(pools=s["pools"], slots=slots, positions=positions, starts=starts, base=base, **t)


def run(state):
    op = state["case"]["op"]
    if own:
        return dict(tree=_own_tree, append=_own_append, accept=_own_accept, branch=_own_branch)[op](state)
    return dict(tree=_plain_tree, append=_plain_append, accept=_plain_accept, branch=_plain_branch)[op](state)


# ------------------------------------------------------------------------------------------------ definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "tree":
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        starts, page, group = s["starts"].tolist(), case["page"], case["qh"] // case["kvh"]
        for b, n in enumerate(s["lens"].tolist()):
            lo, hi = starts[b], starts[b + 1]
            pages = s["table"][b, :-(-n // page)].long()
            see = torch.ones((hi - lo, n), dtype=torch.bool, device="cuda")
            for d in range(hi - lo):
                see[:, n - (hi - lo) + d] = torch.tensor([bool((int(m) & MASK64) >> d & 1) for m in s["mask"][lo:hi].tolist()], device="cuda")
            for h in range(case["kvh"]):
                side = (lambda p: _bytes(p)[pages, h] if case["layout"] == "HND" else _bytes(p)[pages, :, h])
                k = side(s["k"]).view(s["k"].dtype).double().reshape(-1, case["hd"])[:n] * s["k_scale"]
                v = side(s["v"]).view(s["v"].dtype).double().reshape(-1, case["hd"])[:n] * s["v_scale"]
                heads = slice(h * group, (h + 1) * group)
                sc = torch.einsum("igd,td->igt", s["q"][lo:hi, heads].double(), k) / case["hd"] ** 0.5
                sc = sc.masked_fill(~see[:, None], float("-inf"))
                out[lo:hi, heads] = torch.einsum("igt,td->igd", torch.softmax(sc, -1), v)
        return out
    if case["op"] != "append":
        return None                    # values are moved, not computed
    qh, kvh, hd, rot, page = (case[k] for k in ("qh", "kvh", "hd", "rot", "page"))
    x = s["qkv"].double().view(-1, qh + 2 * kvh, hd)
    theta = torch.atan2(s["sin"].double(), s["cos"].double())[s["pos"]][:, None]
    size = torch.hypot(s["sin"].double(), s["cos"].double())[s["pos"]][:, None]

    def turn(heads, weight):
        y = heads / torch.sqrt(heads.square().mean(-1, keepdim=True) + 1e-6) * weight.double()
        z = y[..., :rot].unflatten(-1, (2, rot // 2)).transpose(-1, -2) if case["pairs"] == "half" else y[..., :rot].unflatten(-1, (rot // 2, 2))
        z = torch.view_as_complex(z.contiguous()) * torch.polar(size, theta)
        z = torch.view_as_real(z)
        z = z.transpose(-1, -2).flatten(-2) if case["pairs"] == "half" else z.flatten(-2)
        return torch.cat([z, y[..., rot:]], -1)

    q, k, v = turn(x[:, :qh], s["qw"]), turn(x[:, qh:qh + kvh], s["kw"]), x[:, qh + kvh:]
    got = []
    for pool, new, scale in ((s["k"], k, s["k_scale"]), (s["v"], v, s["v_scale"])):
        whole = pool.double()
        rows = (whole.transpose(1, 2) if case["layout"] == "HND" else whole)       # [pages, page, heads, hd]
        live = s["slots"] >= 0
        rows[s["slots"][live] // page, s["slots"][live] % page] = new[live] / scale
        got.append(whole)
    return dict(q=q, k=got[0], v=got[1])
