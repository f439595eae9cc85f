"""The paged KV cache operators as they are measured: attention of new tokens
over the pages, the append that rotates and stores them, and the page pool's
fork and compaction.

A cache is a pool [layers, 2, pages, kv heads, page size, head dim]; a layer
reads pool[l, 0] (keys) and pool[l, 1] (values).  Row s of `table` lists the
pages of sequence s, `lens[s]` is its length and `refs[p]` how many sequences
hold page p.  The new tokens of a step lie one sequence after another, those of
sequence b in rows q_starts[b] .. q_starts[b + 1]; they are its last tokens, so
that row t of n stands at position lens[b] - n + t.

With `own` false each operator is a few elementary torch operations in 32 bits
(angles in 64), with `own` true it is the framework's call.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # the first tokens of one conversation: nothing but latency
        dict(name="attend_step_one", op="attend", seqs=1, kv=200, q=1, chunks=0, heads=32,
             kv_heads=8, dim=128, page=16, window=0, dtype="bf16"),
        # a serving step of 64 conversations of all lengths, 8 query heads to a key head
        dict(name="attend_step_batch", op="attend", seqs=64, kv=8192, q=1, chunks=0, heads=32,
             kv_heads=4, dim=128, page=16, window=0, dtype="bf16"),
        # two long documents: few rows, a long axis
        dict(name="attend_step_long", op="attend", seqs=2, kv=100003, q=1, chunks=0, heads=32,
             kv_heads=8, dim=64, page=64, window=0, dtype="fp16"),
        # chunked prefill beside running conversations in one step
        dict(name="attend_mixed", op="attend", seqs=8, kv=8000, q=512, chunks=3, heads=32,
             kv_heads=8, dim=128, page=32, window=0, dtype="bf16"),
        # a whole prompt at once
        dict(name="attend_prompt", op="attend", seqs=1, kv=8192, q=8192, chunks=1, heads=32,
             kv_heads=8, dim=128, page=128, window=0, dtype="bf16"),
        # a sliding-window layer with wide heads
        dict(name="attend_window", op="attend", seqs=2, kv=4100, q=1024, chunks=2, heads=8,
             kv_heads=4, dim=256, page=16, window=1024, dtype="bf16"),
        # one token of each of 64 conversations into the cache
        dict(name="append_step", op="append", seqs=64, kv=8192, q=1, chunks=0, heads=32,
             kv_heads=8, dim=128, page=16, dtype="bf16"),
        # prompts into the cache, at far positions
        dict(name="append_prompt", op="append", seqs=4, kv=120000, q=4096, chunks=4, heads=32,
             kv_heads=8, dim=128, page=64, dtype="fp16"),
        # one prompt continued in three ways
        dict(name="fork_few", op="fork", seqs=1, kv=500, ways=3, grow=1, layers=16, kv_heads=8,
             dim=64, page=16, dtype="bf16"),
        # parallel sampling from eight prompts, with room for the next 64 tokens of each way
        dict(name="fork_many", op="fork", seqs=8, kv=2000, ways=7, grow=64, layers=28, kv_heads=8,
             dim=128, page=16, dtype="bf16"),
        # a small pool after a few conversations have ended
        dict(name="compact_few", op="compact", seqs=6, kv=300, ways=1, layers=16, kv_heads=8,
             dim=64, page=16, dtype="fp16"),
        # a serving pool, half of whose pages lie scattered
        dict(name="compact_many", op="compact", seqs=48, kv=1000, ways=1, layers=28, kv_heads=8,
             dim=128, page=32, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "append", "fork", "compact"])
    dtype = rng.choice(["bf16", "fp16"])
    page = rng.choice([16, 32, 48, 64, 128, 256])
    kv_heads = rng.choice([1, 2, 4, 8])
    dim = rng.choice([64, 128, 128, 256])
    if op in ("fork", "compact"):
        seqs, kv = _log(rng, 1 if op == "fork" else 4, 40), _log(rng, 20, 1500)
        ways = rng.randint(1, 6) if op == "fork" else 1
        layer = 4 * kv_heads * page * dim * seqs * (kv // page + 1 + ways)  # bytes, about
        case = dict(op=op, seqs=seqs, kv=kv, ways=ways,
                    layers=max(1, min(rng.randint(1, 28), 1500000000 // layer)),
                    kv_heads=kv_heads, dim=dim, page=page, dtype=dtype)
        if op == "fork":
            case["grow"] = _log(rng, 1, 100)
        return case
    kind = rng.choice(["step", "step", "mixed", "prompt"])
    group = rng.choice([1, 2, 3, 4, 7, 8])
    if kind == "step":
        seqs = _log(rng, 1, 96)
        kv, q, chunks = _log(rng, 2, min(60000, 500000 // seqs)), 1, 0
    elif kind == "mixed":
        seqs = _log(rng, 2, 10)
        q = _log(rng, 2, 700)
        kv, chunks = q + _log(rng, 1, 7000), rng.randint(1, seqs)
    else:
        seqs = _log(rng, 1, 4)
        kv = q = _log(rng, 16, 6000 // seqs)
        chunks = seqs
    case = dict(op=op, seqs=seqs, kv=kv, q=q, chunks=chunks, heads=kv_heads * group,
                kv_heads=kv_heads, dim=dim, page=page, dtype=dtype)
    if op == "attend":
        case["window"] = rng.choice([0, 0, 0, _log(rng, 8, 4096)])
    return case


def _lengths(case):
    """The sequences' lengths and their numbers of new tokens: the longest first, the
    others spread over the range below it."""
    part = [1.0] + [(0.6180339887 * i) % 1.0 for i in range(1, case["seqs"])]
    kv = [max(1, int(case["kv"] * f)) for f in part]
    q = [min(n, max(1, int(case["q"] * f))) if i < case["chunks"] else 1
         for i, (n, f) in enumerate(zip(kv, part))]
    return kv, q


def _pages_of(lengths, page):
    return [-(-n // page) for n in lengths]


def _table(counts, width, gen, spare):
    """Every sequence's pages at random places of a pool of sum(counts) + spare pages."""
    total = sum(counts)
    order = torch.randperm(total + spare, device="cuda", generator=gen)[:total].int()
    table = torch.full((len(counts), width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for s, n in enumerate(counts):
        table[s, :n] = order[at:at + n]
        at += n
    return table


def _normal(shape, dtype, gen):
    """Normal values, made in pieces, so that no copy in 32 bits of a whole pool is needed."""
    out = torch.empty(shape, dtype=dtype, device="cuda")
    flat = out.view(-1)
    for at in range(0, flat.numel(), 1 << 28):
        flat[at:at + (1 << 28)].normal_(generator=gen)
    return out


def _frequencies(dim):
    return torch.tensor([500000.0 ** (-2.0 * i / dim) for i in range(dim // 2)],
                        dtype=torch.float64).float().cuda()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    page, hk, d = case["page"], case["kv_heads"], case["dim"]
    if case["op"] in ("attend", "append"):
        kv, q = _lengths(case)
        counts = _pages_of(kv, page)
        table = _table(counts, max(counts), gen, 8)
        pool = _normal((2, sum(counts) + 8, hk, page, d), dtype, gen)
        starts = [0]
        for n in q:
            starts.append(starts[-1] + n)
        rows, h = starts[-1], case["heads"]
        # q, k and v are slices of the fused projection's rows
        qkv = _normal((rows, (h + 2 * hk) * d), dtype, gen)
        state = dict(case=case, table=table, k=pool[0], v=pool[1], rows=rows,
                     lens=torch.tensor(kv, dtype=torch.int32, device="cuda"),
                     starts=torch.tensor(starts, dtype=torch.int32, device="cuda"),
                     max_kv=max(kv), max_q=max(q),
                     q_new=qkv[:, :h * d].unflatten(1, (h, d)),
                     k_new=qkv[:, h * d:(h + hk) * d].unflatten(1, (hk, d)),
                     v_new=qkv[:, (h + hk) * d:].unflatten(1, (hk, d)))
        if case["op"] == "append":
            state["freqs"] = _frequencies(d)
            state["q_out"] = torch.empty((rows, h, d), dtype=dtype, device="cuda")
        return state
    kv = _lengths(dict(case, q=1, chunks=0))[0]
    held = _pages_of(kv, page)
    ways = case["ways"] if case["op"] == "fork" else 0
    grown = _pages_of([n + case.get("grow", 0) for n in kv], page)
    extra = sum((g - n + 1) * ways for g, n in zip(grown, held))
    spare = extra + 4 if ways else sum(held)
    n_pages = sum(held) + spare
    pool = _normal((case["layers"], 2, n_pages, hk, page, d), dtype, gen)
    table = torch.full((len(kv) * (1 + ways), max(grown)), -1, dtype=torch.int32, device="cuda")
    table[:len(kv), :max(held)] = _table(held, max(held), gen, spare)
    refs = torch.zeros(n_pages, dtype=torch.int32, device="cuda")
    refs[table[table >= 0].long()] = 1
    lens = torch.zeros(len(kv) * (1 + ways), dtype=torch.int32, device="cuda")
    lens[:len(kv)] = torch.tensor(kv, dtype=torch.int32, device="cuda")
    state = dict(case=case, pool=pool, table=table, refs=refs, lens=lens)
    if ways:
        parents = torch.arange(len(kv), dtype=torch.int32, device="cuda").repeat_interleave(ways)
        state["parents"] = parents
        state["children"] = torch.arange(len(kv), len(kv) * (1 + ways), dtype=torch.int32,
                                         device="cuda")
        state["new_lens"] = lens[parents.long()] + case["grow"]
    else:
        state["table_then"], state["refs_then"] = table.clone(), refs.clone()
    return state


def run(state):
    return {"attend": _attend, "append": _append, "fork": _fork,
            "compact": _compact}[state["case"]["op"]](state)


# ------------------------------------------------------------------ attention


def _gathered(pages, table, n):
    """The first n keys or values of every sequence, [seqs, kv heads, n, dim], 32 bits."""
    at = torch.arange(n, device="cuda")
    page = table.long().clamp(min=0)[:, at // pages.shape[2]]
    return pages[page, :, at % pages.shape[2]].float().permute(0, 2, 1, 3)


def _attend(s):
    case = s["case"]
    q, starts = s["q_new"], s["starts"]
    if own:
        import neurons_b200 as nb
        return nb.paged_attention(q, s["k"], s["v"], s["table"], s["lens"],
                                  q_starts=starts if s["max_q"] > 1 else None,
                                  max_q=s["max_q"], window=case["window"])
    seqs, h, hk, d = case["seqs"], case["heads"], case["kv_heads"], case["dim"]
    n, m = s["max_kv"], s["max_q"]
    key = torch.arange(n, device="cuda")
    t = torch.arange(m, device="cuda")
    count = (starts[1:] - starts[:-1])[:, None]
    row = torch.where(t < count, starts[:-1, None] + t, s["rows"])  # [seqs, m]
    x = q[row.clamp(max=s["rows"] - 1)].float().view(seqs, m, hk, h // hk, d)
    x = x.permute(0, 2, 3, 1, 4).reshape(seqs, hk, (h // hk) * m, d)
    score = x @ _gathered(s["k"], s["table"], n).transpose(2, 3)
    score = score.mul_(1 / math.sqrt(d)).view(seqs, hk, h // hk, m, n)
    pos = (s["lens"][:, None] - count + t)[:, :, None]
    hidden = key > pos
    if case["window"]:
        hidden |= key <= pos - case["window"]
    score.masked_fill_(hidden[:, None, None], -math.inf)
    score = score.sub_(score.amax(-1, keepdim=True).clamp(min=-1e30)).exp_()
    total = score.sum(-1, keepdim=True).clamp(min=1e-30)
    out = score.view(seqs, hk, -1, n) @ _gathered(s["v"], s["table"], n)
    out = out.view(seqs, hk, h // hk, m, d) / total
    result = torch.zeros((s["rows"] + 1, h, d), dtype=q.dtype, device="cuda")
    result[row] = out.permute(0, 3, 1, 2, 4).reshape(seqs, m, h, d).to(q.dtype)
    return result[:-1]


def _exact_attend(s):
    case = s["case"]
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    out = torch.zeros((s["rows"], h, d), dtype=torch.float64, device="cuda")
    starts, lens = s["starts"].tolist(), s["lens"].tolist()
    for b, n in enumerate(lens):
        lo, hi = starts[b], starts[b + 1]
        held = s["table"][b, :-(-n // case["page"])].long()
        pos = torch.arange(n - (hi - lo), n, device="cuda")
        key = torch.arange(n, device="cuda")
        see = key[None, :] <= pos[:, None]
        if case["window"]:
            see &= key[None, :] > pos[:, None] - case["window"]
        for j in range(hk):
            k = s["k"][held, j].reshape(-1, d)[:n].double()
            v = s["v"][held, j].reshape(-1, d)[:n].double()
            for i in range(j * (h // hk), (j + 1) * (h // hk)):
                w = s["q_new"][lo:hi, i].double() @ k.t() / math.sqrt(d)
                w = torch.softmax(torch.where(see, w, -math.inf), dim=-1)
                out[lo:hi, i] = w @ v
    return out


# --------------------------------------------------------------------- append


def _places(s):
    """Each new token's sequence, position, page and slot."""
    i = torch.arange(s["rows"], device="cuda")
    seq = torch.searchsorted(s["starts"].long(), i, right=True) - 1
    pos = s["lens"].long()[seq] - s["starts"].long()[seq + 1] + i
    page = s["table"].long()[seq, pos // s["case"]["page"]]
    return pos, page, pos % s["case"]["page"]


def _rotated(x, pos, freqs):
    angle = pos.double()[:, None] * freqs.double()
    c, n = angle.cos().float()[:, None], angle.sin().float()[:, None]
    a, b = x.float().chunk(2, dim=-1)
    return torch.cat([a * c - b * n, a * n + b * c], dim=-1).to(x.dtype)


def _append(s):
    if own:
        import neurons_b200 as nb
        nb.paged_append(s["q_new"], s["k_new"], s["v_new"], s["k"], s["v"], s["table"], s["lens"],
                        q_starts=s["starts"] if s["max_q"] > 1 else None, freqs=s["freqs"],
                        q_out=s["q_out"])
        return s["q_out"], s["k"], s["v"]
    pos, page, slot = _places(s)
    s["q_out"].copy_(_rotated(s["q_new"], pos, s["freqs"]))
    s["k"][page, :, slot] = _rotated(s["k_new"], pos, s["freqs"])
    s["v"][page, :, slot] = s["v_new"]
    return s["q_out"], s["k"], s["v"]


def _exact_append(s):
    half = s["case"]["dim"] // 2
    page = s["case"]["page"]
    starts, lens = s["starts"].tolist(), s["lens"].tolist()
    qs, k, v = [], s["k"].double(), s["v"].double()
    for b, n in enumerate(lens):
        lo, hi = starts[b], starts[b + 1]
        pos = torch.arange(n - (hi - lo), n, dtype=torch.float64, device="cuda")
        turn = torch.polar(torch.ones((hi - lo, half), dtype=torch.float64, device="cuda"),
                           pos[:, None] * s["freqs"].double()[None, :])[:, None]

        def rotate(x):
            z = torch.complex(x[..., :half].double(), x[..., half:].double()) * turn
            return torch.cat([z.real, z.imag], dim=-1)

        qs.append(rotate(s["q_new"][lo:hi]))
        at = pos.long()
        where = s["table"][b].long()[at // page]
        k[where, :, at % page] = rotate(s["k_new"][lo:hi])
        v[where, :, at % page] = s["v_new"][lo:hi].double()
    return torch.cat(qs), k, v


# ----------------------------------------------------------------------- fork


def _fork(s):
    """Frees the ways of the last pass, forks them again and gives each its room: a page
    that is not full and has other holders is copied first."""
    refs, table, lens, pool = s["refs"], s["table"], s["lens"], s["pool"]
    if own:
        import neurons_b200 as nb
        nb.pages_free(refs, table, lens, s["children"])
        nb.pages_fork(refs, table, lens, s["parents"], s["children"])
        nb.pages_reserve(pool, refs, table, lens, s["children"], s["new_lens"])
        return refs, table, lens, pool
    ps = s["case"]["page"]
    kids, slot = s["children"].long(), torch.arange(table.shape[1], device="cuda")
    # free
    mine = table[kids]
    refs.index_add_(0, mine.clamp(min=0).view(-1).long(), -(mine >= 0).int().view(-1))
    table[kids] = -1
    # fork
    mine = table[s["parents"].long()]
    old = lens[s["parents"].long()].long()
    refs.index_add_(0, mine.clamp(min=0).view(-1).long(), (mine >= 0).int().view(-1))
    # reserve
    new = s["new_lens"].long()
    last = mine.long().gather(1, ((old - 1) // ps).clamp(min=0)[:, None])[:, 0]
    part = (old % ps != 0) & (new > old)
    same = (last[:, None] == last[None, :]) & part[:, None] & part[None, :]
    rank = same.tril(-1).sum(1)
    split = part & (rank < refs[last.clamp(min=0)] - 1)
    first = torch.where(split, old // ps, (old + ps - 1) // ps)
    need = (slot >= first[:, None]) & (slot < ((new + ps - 1) // ps)[:, None])
    order = need.view(-1).cumsum(0).view(need.shape) - 1
    free = torch.sort((refs > 0).int(), stable=True)[1].int()
    mine = torch.where(need, free[order.clamp(min=0)], mine)
    taken = mine.gather(1, ((old - 1) // ps).clamp(min=0)[:, None])[:, 0].long()
    pool[:, :, torch.where(split, taken, last)] = pool[:, :, last]
    refs.index_add_(0, last, -split.int())
    refs.index_add_(0, mine.clamp(min=0).view(-1).long(), need.int().view(-1))
    table[kids] = mine
    lens[kids] = s["new_lens"]
    return refs, table, lens, pool


def _exact_fork(s):
    ps = s["case"]["page"]
    refs, table, lens = s["refs"].tolist(), s["table"].tolist(), s["lens"].tolist()
    pool = s["pool"].double()
    for p, c in zip(s["parents"].tolist(), s["children"].tolist()):
        table[c], lens[c] = list(table[p]), lens[p]
        for x in table[c]:
            if x >= 0:
                refs[x] += 1
    for c, n in zip(s["children"].tolist(), s["new_lens"].tolist()):
        at = lens[c] // ps
        if lens[c] % ps and n > lens[c] and refs[table[c][at]] > 1:
            was, now = table[c][at], refs.index(0)
            refs[was] -= 1
            refs[now], table[c][at] = 1, now
            pool[:, :, now] = pool[:, :, was]
        for at in range(-(-lens[c] // ps), -(-n // ps)):
            now = refs.index(0)
            refs[now], table[c][at] = 1, now
        lens[c] = n
    return (torch.tensor(refs, dtype=torch.int32), torch.tensor(table, dtype=torch.int32),
            torch.tensor(lens, dtype=torch.int32), pool)


# -------------------------------------------------------------------- compact


def _compact(s):
    """The used pages move to the pool's low end.  Each pass begins with the scattered table."""
    refs, table, pool = s["refs"], s["table"], s["pool"]
    refs.copy_(s["refs_then"])
    table.copy_(s["table_then"])
    if own:
        import neurons_b200 as nb
        nb.pages_compact(pool, refs, table)
        return refs, table, pool
    index = torch.arange(refs.numel(), device="cuda")
    used = refs > 0
    low = index < used.sum()
    moves, holes = used & ~low, ~used & low
    src, dst = moves.nonzero()[:, 0], holes.nonzero()[:, 0]
    place = index.int()
    place[src] = dst.int()
    pool[:, :, dst] = pool[:, :, src]
    refs[dst] = refs[src]
    refs[src] = 0
    table.copy_(torch.where(table >= 0, place[table.clamp(min=0).long()], table))
    return refs, table, pool


def _exact_compact(s):
    refs, table, pool = s["refs_then"].tolist(), s["table_then"].tolist(), s["pool"].double()
    used = sum(r > 0 for r in refs)
    low = [p for p in range(used) if refs[p] == 0]
    high = [p for p in range(used, len(refs)) if refs[p] > 0]
    to = dict(zip(high, low))
    for a, b in to.items():
        pool[:, :, b] = pool[:, :, a]
        refs[a], refs[b] = 0, refs[a]
    table = [[to.get(x, x) for x in row] for row in table]
    return torch.tensor(refs, dtype=torch.int32), torch.tensor(table, dtype=torch.int32), pool


# ----------------------------------------------------------------------- work


def exact(case, seed):
    s = prepare(case, seed)
    return {"attend": _exact_attend, "append": _exact_append, "fork": _exact_fork,
            "compact": _exact_compact}[case["op"]](s)


def _seen(n, q, window):
    """The (query, key) pairs of q new tokens at the end of n, and the keys that any of them sees."""
    pairs = q * (n - q) + q * (q + 1) // 2
    if not window:
        return pairs, n
    over = [max(0, n - q + t + 1 - window) for t in range(q)]
    return pairs - sum(over), n - over[0]


def work(case):
    page, hk, d = case["page"], case["kv_heads"], case["dim"]
    if case["op"] in ("attend", "append"):
        kv, q = _lengths(case)
        h, rows = case["heads"], sum(q)
        index = 4 * (sum(_pages_of(kv, page)) + 2 * len(kv) + 1)
        if case["op"] == "append":
            # q, k and v in and out
            return {"bytes": index + 2 * 2 * rows * (h + 2 * hk) * d, "flops": 6 * rows * (h + hk) * d}
        seen = [_seen(n, m, case["window"]) for n, m in zip(kv, q)]
        # q in, the result out, every visible key and value once; two products
        return {"bytes": index + 2 * 2 * rows * h * d + 2 * 2 * hk * d * sum(s[1] for s in seen),
                "flops": 4 * h * d * sum(s[0] for s in seen)}
    kv = _lengths(dict(case, q=1, chunks=0))[0]
    held = _pages_of(kv, page)
    size = case["layers"] * 2 * hk * page * d * 2
    if case["op"] == "fork":
        copies = case["ways"] * sum(n % page != 0 for n in kv)
        return {"bytes": 2 * size * copies + 4 * (2 * sum(held) * (1 + 2 * case["ways"])), "flops": 0}
    # half of the pool is in use, at random places: about half of the used pages have to move
    return {"bytes": 2 * size * sum(held) // 2 + 4 * 6 * sum(held), "flops": 0}
