"""Plain implementations of the paged cache's operators, for their tests: attention in 64
bits with the error bound that its arithmetic allows, and the page pool as Python lists."""
import math

import torch


class Batch:
    """A cache whose unused slots are NaN and a batch over it.  lens / news: per entry the
    length and the new tokens; perm: table rows in another order than the entries."""

    def __init__(self, lens, news, heads, kv_heads, dim, page, dtype, seed=0, extra_rows=0,
                 spare=3, window=0, n_pages=None, interleaved=False):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.lens, self.news = list(lens), list(news)
        self.heads, self.kv_heads, self.dim, self.page, self.dtype = heads, kv_heads, dim, page, dtype
        n = len(lens)
        counts = [-(-x // page) for x in lens]
        total = sum(counts) + spare
        self.n_pages = n_pages or total
        # interleaved: keys and values of a page side by side in one tensor
        if interleaved:
            pool = torch.full((self.n_pages, 2, kv_heads, page, dim), float("nan"), dtype=dtype,
                              device="cuda")
            self.k, self.v = pool[:, 0], pool[:, 1]
        else:
            pool = torch.empty((2, self.n_pages, kv_heads, page, dim), dtype=dtype, device="cuda")
            if n_pages is None:
                pool.fill_(float("nan"))
            self.k, self.v = pool[0], pool[1]
        pages = (torch.randperm(total, device="cuda", generator=g) + self.n_pages - total).tolist()
        width = max(counts + [1]) + 1
        self.rows = torch.randperm(n, device="cpu",
                                   generator=torch.Generator().manual_seed(seed)).tolist()
        table = torch.full((n, width), -1, dtype=torch.int32)
        row_lens = torch.zeros(n, dtype=torch.int32)
        self.dense = []
        for b in range(n):
            own, pages = pages[:counts[b]], pages[counts[b]:]
            first = max(0, lens[b] - news[b] - window + 1) // page if window else 0
            kk = torch.randn((lens[b], kv_heads, dim), device="cuda", generator=g).to(dtype)
            vv = torch.randn((lens[b], kv_heads, dim), device="cuda", generator=g).to(dtype)
            self.dense.append((kk, vv))
            for i, p in enumerate(own):
                lo, hi = i * page, min((i + 1) * page, lens[b])
                if n_pages is not None:
                    self.k[p] = float("nan")
                    self.v[p] = float("nan")
                if i >= first:  # pages that no window reaches are given up
                    table[self.rows[b], i] = p
                    self.k[p, :, :hi - lo] = kk[lo:hi].transpose(0, 1)
                    self.v[p, :, :hi - lo] = vv[lo:hi].transpose(0, 1)
            row_lens[self.rows[b]] = lens[b]
        self.table, self.row_lens = table.cuda(), row_lens.cuda()
        self.seqs = torch.tensor(self.rows, dtype=torch.int32, device="cuda")
        starts = [0]
        for x in news:
            starts.append(starts[-1] + x)
        self.starts = torch.tensor(starts, dtype=torch.int32, device="cuda")
        self.tokens = starts[-1]
        qkv = torch.randn((self.tokens + extra_rows, (heads + 2 * kv_heads) * dim), device="cuda",
                          generator=g).to(dtype)
        self.q = qkv[:, :heads * dim].unflatten(1, (heads, dim))

    def call(self, nb, **kw):
        return nb.paged_attention(self.q, self.k, self.v, self.table, self.row_lens,
                                  q_starts=self.starts, seqs=self.seqs, **kw)


def attention64(b, window=0, scale=None):
    """(result, bound) [tokens, heads, dim] in 64 bits.  bound: how far a result in the
    cache's type may be off, element by element:
      u |o|                      the result's rounding, u = eps / 2 of the type
      (u + r) sum p |v| / sum p  u: the weights' rounding; r: the scores' error (dim + 2
                                 roundings of 2^-24 on scale |q|.|k|, in numerator and
                                 denominator), the sums over n keys and over parts
                                 (n + 64 roundings in each) and exp's 2^-20
    and, for fp16 weights below the normal range, n 2^-25 max |v|."""
    scale = 1 / math.sqrt(b.dim) if scale is None else scale
    u = torch.finfo(b.dtype).eps / 2
    out = torch.zeros((b.tokens, b.heads, b.dim), dtype=torch.float64, device="cuda")
    bound = torch.zeros_like(out)
    at, group = 0, b.heads // b.kv_heads
    for (k, v), n, m in zip(b.dense, b.lens, b.news):
        pos = torch.arange(n - m, n, device="cuda")
        key = torch.arange(n, device="cuda")
        see = key[None] <= pos[:, None]
        if window:
            see &= key[None] > pos[:, None] - window
        for h in range(b.heads if n and m else 0):
            q = b.q[at:at + m, h].double()
            kk, vv = k[:, h // group].double(), v[:, h // group].double()
            s = torch.where(see, q @ kk.t() * scale, -math.inf)
            top = s.amax(1, keepdim=True)
            p = torch.where(see, torch.exp(s - top.clamp(min=-1e300)), 0.0)
            total = p.sum(1, keepdim=True).clamp(min=1e-300)
            o = p @ vv / total
            mag = (torch.where(see, q.abs() @ kk.abs().t(), 0.0).amax(1, keepdim=True) * scale)
            r = 2 * (b.dim + 2) * 2.0 ** -24 * mag + 2 * (n + 64) * 2.0 ** -24 + 2.0 ** -20
            out[at:at + m, h] = o
            bound[at:at + m, h] = u * o.abs() + (u + r) * (p @ vv.abs() / total)
            if b.dtype == torch.float16:
                bound[at:at + m, h] += n * 2.0 ** -25 * vv.abs().amax()
        at += m
    return out, bound


def check_attention(got, b, window=0, scale=None):
    want, bound = attention64(b, window, scale)
    got = got[:b.tokens].double()
    assert torch.isfinite(got).all()
    over = (got - want).abs() - bound
    assert (over <= 1e-12).all(), f"{over.max().item():.3e} over the bound"


class Pool:
    """refs, table and lens as lists, with the operators' rules."""

    def __init__(self, n_pages, rows, width, page):
        self.refs = [0] * n_pages
        self.table = [[-1] * width for _ in range(rows)]
        self.lens = [0] * rows
        self.page, self.width = page, width
        self.errors = 0

    def free(self, seqs):
        for s in seqs:
            if s < 0:
                continue
            if s >= len(self.lens):
                self.errors |= 4
                continue
            for p in self.table[s]:
                if p >= 0:
                    self.refs[p] -= 1
            self.table[s], self.lens[s] = [-1] * self.width, 0

    def fork(self, parents, children):
        rows = range(len(self.lens))
        made = []
        for i, (p, c) in enumerate(zip(parents, children)):
            if p < 0 and c < 0:
                continue
            if p not in rows or c not in rows or c in children[:i] or c in parents or \
                    p in children or self.lens[c] or self.table[c][0] != -1:
                self.errors |= 4
            else:
                made.append((p, c))
        for p, c in made:
            self.table[c], self.lens[c] = list(self.table[p]), self.lens[p]
            for x in self.table[c]:
                if x >= 0:
                    self.refs[x] += 1

    def reserve(self, seqs, new_lens):
        """The copies (from, to) it makes."""
        live = [(s, n) for s, n in zip(seqs, new_lens) if s >= 0]
        ids = [s for s, _ in live]
        bad = len(set(ids)) < len(ids) or any(
            s >= len(self.lens) or n < self.lens[s] or n > self.width * self.page for s, n in live)
        if not bad:
            keep = ([*self.refs], [[*r] for r in self.table], [*self.lens])
            free = [p for p, r in enumerate(self.refs) if r == 0]
            moves = []
            try:
                for s, n in live:
                    old = self.lens[s]
                    if old % self.page and n > old and self.refs[self.table[s][old // self.page]] > 1:
                        was, now = self.table[s][old // self.page], free.pop(0)
                        moves.append((was, now))
                        self.refs[was] -= 1
                        self.refs[now] = 1
                        self.table[s][old // self.page] = now
                    for i in range(-(-old // self.page), -(-n // self.page)):
                        self.table[s][i] = free.pop(0)
                        self.refs[self.table[s][i]] = 1
                    self.lens[s] = n
                return moves
            except IndexError:
                self.refs, self.table, self.lens = keep
        self.errors |= 4
        return []

    def compact(self):
        used = sum(r > 0 for r in self.refs)
        holes = [p for p in range(used) if not self.refs[p]]
        moves = list(zip([p for p in range(used, len(self.refs)) if self.refs[p]], holes))
        to = dict(moves)
        for a, b in moves:
            self.refs[b], self.refs[a] = self.refs[a], 0
        self.table = [[to.get(p, p) for p in r] for r in self.table]
        return moves
