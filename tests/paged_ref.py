"""Plain restatements in 64 bits of the operators around the paged cache, for the tests."""
import torch

DT = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp8": torch.float8_e4m3fn}
HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float8_e4m3fn: 2.0 ** -4}   # eps / 2
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float8_e4m3fn: 2.0 ** -10}   # half a subnormal


def raw(t):
    return t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t


def pool_shape(layout, pages, kvh, page, hd):
    return (pages, kvh, page, hd) if layout == "HND" else (pages, page, kvh, hd)


def make_pool(layout, pages, kvh, page, hd, kv, g, device="cpu", fill=None):
    t = torch.randn(pool_shape(layout, pages, kvh, page, hd), generator=g, device=device)
    return (t if fill is None else torch.full_like(t, fill)).to(DT[kv])


def tokens_of(pool, pages, layout):
    """[len(pages) * page_size, kv_heads, hd] in 64 bits; the pages by number."""
    p = raw(pool)[torch.as_tensor(pages, dtype=torch.long, device=pool.device)].view(pool.dtype).double()
    if layout == "HND":
        p = p.transpose(1, 2)
    return p.flatten(0, 1)


def tree_attn(q, kp, vp, table, lens, starts, mask, layout, scale, ks=1.0, vs=1.0):
    """(out, spread, size): the result in 64 bits, sum_t p |v| and the largest sum_d |q_d k_d| scale over the visible
    tokens, which the error bound needs.  Rows that no sequence covers: NaN."""
    page = kp.shape[2 if layout == "HND" else 1]
    qh, hd = q.shape[1:]
    kvh = kp.shape[1 if layout == "HND" else 2]
    out = torch.full(q.shape, float("nan"), dtype=torch.float64, device=q.device)
    spread, size = torch.zeros_like(out), torch.zeros(q.shape[:2], dtype=torch.float64, device=q.device)
    pages = kp.shape[0]
    for b, n in enumerate(lens.tolist()):
        lo, hi = starts[b].item(), starts[b + 1].item()
        if hi == lo:
            continue
        if n == 0:
            out[lo:hi] = 0
            continue
        ids = table[b, :-(-n // page)].tolist()
        good = torch.tensor([0 <= p < pages for p in ids], device=q.device).repeat_interleave(page)[:n]
        ids = [p if 0 <= p < pages else 0 for p in ids]
        k, v = tokens_of(kp, ids, layout)[:n] * ks, tokens_of(vp, ids, layout)[:n] * vs
        t = torch.arange(n, device=q.device)
        for i in range(lo, hi):
            j = t - (n - (hi - lo))                       # draft number of a token
            if mask is None:
                see = j <= i - lo
            else:
                m = int(mask[i])
                bits = torch.tensor([m >> x & 1 for x in range(64)], dtype=torch.bool, device=q.device)
                see = (j < 0) | bits[j.clamp(0, 63)]
            idx = (see & good).nonzero()[:, 0]
            if idx.numel() == 0:
                out[i] = 0
                continue
            G = qh // kvh
            kk, vv = k[idx].repeat_interleave(G, 1), v[idx].repeat_interleave(G, 1)       # [t, qh, hd]
            x = q[i].double()
            s = torch.einsum("hd,thd->ht", x, kk) * scale
            p = torch.softmax(s, -1)
            out[i] = torch.einsum("ht,thd->hd", p, vv)
            spread[i] = torch.einsum("ht,thd->hd", p, vv.abs())
            size[i] = (torch.einsum("hd,thd->ht", x.abs(), kk.abs()) * abs(scale)).amax(-1)
    return out, spread, size


def tree_tolerance(ref, spread, size, dtype, longest, vmax):
    """Bound of the kernel's error, term by term: the probabilities' rounding to 16 bits (half a step each, or half a
    subnormal where they are that small, against a sum of at least one), the scores' fp32 sums (hd products of at most
    `size`, each addition off by at most 2^-23 of it; the exponential doubles what a score is off), the fp32 sums over the
    tokens, and the output's rounding."""
    h, hd = HALF_STEP[dtype], ref.shape[-1]
    scores = 2 * hd * 2.0 ** -23 * size[..., None]
    return spread * (h + scores + longest * 2.0 ** -23 + 2.0 ** -20) + longest * TINY[dtype] * vmax + ref.abs() * h + TINY[dtype]


def append(qkv, cos, sin, pos, q_heads, kv_heads, hd, qw, kw, eps, interleaved):
    """(q [T, qh, hd], k [T, kvh, hd], v, size of the largest term of a rotated value) in 64 bits."""
    T = qkv.shape[0]
    x = qkv[:, :(q_heads + 2 * kv_heads) * hd].double().reshape(T, q_heads + 2 * kv_heads, hd)
    y, v = x[:, :q_heads + kv_heads], x[:, q_heads + kv_heads:]
    if eps is not None:
        y = y / torch.sqrt(y.square().mean(-1, keepdim=True) + eps)
        w = torch.ones(q_heads + kv_heads, hd, dtype=torch.float64, device=qkv.device)
        if qw is not None:
            w[:q_heads] = qw.double()
        if kw is not None:
            w[q_heads:] = kw.double()
        y = y * w
    size = y.abs()
    if cos is not None:
        c, s = cos.double()[pos][:, None], sin.double()[pos][:, None]
        rot = 2 * cos.shape[1]
        if interleaved:
            a, b = y[..., 0:rot:2].clone(), y[..., 1:rot:2].clone()
        else:
            a, b = y[..., :rot // 2].clone(), y[..., rot // 2:rot].clone()
        y, size = y.clone(), size.clone()
        lo, hi, m = a * c - b * s, b * c + a * s, a.abs() + b.abs()
        if interleaved:
            y[..., 0:rot:2], y[..., 1:rot:2] = lo, hi
            size[..., 0:rot:2], size[..., 1:rot:2] = m, m
        else:
            y[..., :rot // 2], y[..., rot // 2:rot] = lo, hi
            size[..., :rot // 2], size[..., rot // 2:rot] = m, m
    return y[:, :q_heads], y[:, q_heads:], v, size


class Pages:
    """The page bookkeeping, one entry after the other on lists."""

    def __init__(self, tables):
        self.table = tables["block_table"].cpu().tolist()
        self.lens, self.held, self.refs = (tables[n].cpu().tolist() for n in ("seq_lens", "held", "refs"))
        self.stack = tables["free_list"].cpu().tolist()
        self.left, self.status = tables["counters"].cpu().tolist()
        self.copies = []                                  # (from page, to page, rows) of forks

    def fork(self, parents, children, page):
        n = len(parents)
        ok = [0 <= p < len(self.lens) and 0 <= c < len(self.lens) and c not in children[:i] and c not in parents
              and p not in children for i, (p, c) in enumerate(zip(parents, children))]
        stop = False
        for i in range(n):
            p, c = parents[i], children[i]
            if not ok[i] or -(-self.lens[p] // page) > min(self.held[p], len(self.table[0])) or self.held[c]:
                self.status |= 2
                continue
            full, rest = divmod(self.lens[p], page)
            if rest and (stop or self.left == 0):
                self.status |= 1
                stop = True
                continue
            self.table[c][:full] = self.table[p][:full]
            for x in self.table[p][:full]:
                self.refs[x] += 1
            if rest:
                self.left -= 1
                new = self.stack[self.left]
                self.copies.append((self.table[p][full], new, rest))
                self.table[c][full] = new
                self.refs[new] = 1
            self.lens[c], self.held[c] = self.lens[p], full + (rest > 0)

    def reserve(self, seqs, counts, page, tokens):
        base, starts, slots, pos, stop = [], [0], [], [], False
        for i, (s, n) in enumerate(zip(seqs, counts)):
            at = starts[-1]
            starts.append(min(tokens, at + max(n, 0)))
            ok = 0 <= s < len(self.lens) and n >= 0 and s not in seqs[:i]
            start = self.lens[s] if ok else 0
            base.append(start)
            ok = ok and -(-(start + n) // page) <= len(self.table[0]) and at + n <= tokens
            if not ok:
                self.status |= 2
            want = max(0, -(-(start + n) // page) - self.held[s]) if ok else 0
            if ok and (want > self.left or (stop and want)):
                self.status |= 1
                stop, ok = True, False
            if ok:
                for _ in range(want):
                    self.left -= 1
                    x = self.stack[self.left]
                    self.table[s][self.held[s]] = x
                    self.refs[x] = 1
                    self.held[s] += 1
                self.lens[s] = start + n
            for t in range(starts[-1] - at):
                pos.append(start + t)
                slots.append(self.table[s][(start + t) // page] * page + (start + t) % page if ok else -1)
        slots += [-1] * (tokens - len(slots))
        pos += [0] * (tokens - len(pos))
        return slots, pos, starts, base

    def free(self, seqs):
        entries = []
        for i, s in enumerate(seqs):
            if not 0 <= s < len(self.lens) or s in seqs[:i]:
                self.status |= 2
                continue
            for x in self.table[s][:self.held[s]]:
                self.refs[x] -= 1
                entries.append(x)
            self.held[s] = self.lens[s] = 0
        back = [x for i, x in enumerate(entries) if self.refs[x] == 0 and x not in entries[i + 1:]]
        for x in reversed(back):                          # the first entry ends on top
            self.stack[self.left] = x
            self.left += 1

    def same(self, tables):
        """What differs from the state on the device (the stack above its top is of no account)."""
        got = {n: tables[n].cpu().tolist() for n in tables}
        bad = []
        for s, h in enumerate(self.held):
            if got["block_table"][s][:h] != self.table[s][:h]:
                bad.append(("block_table", s, got["block_table"][s][:h], self.table[s][:h]))
        for n, want in (("seq_lens", self.lens), ("held", self.held), ("refs", self.refs), ("counters", [self.left, self.status])):
            if got[n] != want:
                bad.append((n, got[n], want))
        if got["free_list"][:self.left] != self.stack[:self.left]:
            bad.append(("free_list", got["free_list"], self.stack))
        return bad
