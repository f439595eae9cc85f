"""GPU tests of the paged cache: attention against 64 bits within the bound that its
arithmetic allows (tests/_paged.py), the append against 64 bits, the page pool against
lists, and all of them together as a server uses them."""
import math
import random

import pytest
import torch

import neurons_b200 as nb
from _paged import Batch, Pool, attention64, check_attention

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def clean_error_word(nqlib):
    nb.take_device_error()
    yield
    torch.cuda.synchronize()


BF, HF = torch.bfloat16, torch.float16

# (lens, new tokens, heads, key heads, dim, page, type, window)
ATTENTION = {
    "one key": ([1], [1], 4, 4, 64, 16, BF, 0),
    "one token": ([200], [1], 32, 8, 128, 16, BF, 0),
    "tile borders": ([15, 16, 17, 63, 64, 65, 127, 128, 129], [1] * 9, 8, 2, 128, 16, BF, 0),
    "ragged steps": ([1, 2, 1000, 37, 513, 256, 0, 3000], [1] * 8, 8, 1, 128, 32, HF, 0),
    "long step": ([20011], [1], 16, 2, 64, 64, HF, 0),
    "wide heads": ([700, 33], [1, 1], 8, 4, 256, 16, BF, 0),
    "wide heads fp16": ([130, 900], [1, 5], 4, 1, 256, 48, HF, 0),
    "odd group": ([300, 41], [1, 3], 21, 3, 128, 48, BF, 0),
    "one head": ([90, 5], [7, 5], 1, 1, 64, 16, BF, 0),
    "group of 16": ([301], [2], 16, 1, 128, 16, BF, 0),
    "chunk": ([300], [37], 8, 2, 128, 16, BF, 0),
    "prompt": ([257], [257], 4, 2, 64, 128, HF, 0),
    "prompt wide": ([150], [150], 2, 1, 256, 32, BF, 0),
    "mixed": ([700, 64, 5, 1, 333], [130, 64, 1, 1, 33], 8, 4, 128, 32, BF, 0),
    "no tokens": ([100, 50, 20], [1, 0, 2], 4, 2, 64, 16, BF, 0),
    "empty rows": ([5, 0, 3], [8, 4, 3], 4, 2, 128, 16, BF, 0),
    "window": ([1000, 40, 257], [1, 1, 1], 8, 2, 128, 16, BF, 100),
    "window of one": ([77, 16], [5, 1], 4, 2, 64, 16, HF, 1),
    "window chunk": ([600, 130], [150, 130], 4, 1, 128, 16, BF, 64),
    "window wide": ([400], [90], 2, 2, 256, 64, BF, 33),
    "large page": ([1000, 300], [1, 20], 4, 2, 128, 1024, BF, 0),
    "page of 48": ([100, 49, 48, 47], [3, 2, 48, 1], 6, 2, 64, 48, HF, 0),
    "many tiny": ([i % 40 + 1 for i in range(300)], [1] * 300, 4, 2, 64, 16, BF, 0),
    "chunk of 512": ([3000, 700], [512, 300], 8, 2, 128, 32, BF, 0),
    "prompt of 1000": ([1000], [1000], 14, 2, 64, 16, BF, 0),
    "prompt of 700 wide": ([700, 20], [700, 3], 4, 2, 256, 128, HF, 0),
    "group of 32": ([300, 7], [1, 5], 32, 1, 64, 16, BF, 0),
    "group of 128": ([150], [3], 128, 1, 128, 16, HF, 0),
    "one tile of many blocks": ([9000], [30], 8, 2, 128, 64, BF, 0),
    "tiles end in blocks": ([128, 129, 256, 257, 383, 64], [32, 33, 64, 65, 100, 64], 8, 2, 128, 128, BF, 0),
    "many chunks": ([40 * i + 20 for i in range(40)], [i + 1 for i in range(40)], 8, 4, 64, 16, HF, 0),
    "chunk window": ([5000, 1500], [300, 700], 4, 2, 128, 16, HF, 700),
}


@pytest.mark.parametrize("name", ATTENTION)
def test_attention(name):
    lens, news, heads, kv, dim, page, dtype, window = ATTENTION[name]
    b = Batch(lens, news, heads, kv, dim, page, dtype, seed=len(name), window=window, extra_rows=2)
    out = torch.full((b.tokens + 2, heads, dim), 7.0, dtype=dtype, device="cuda")
    b.call(nb, window=window, max_q=max(news), out=out)
    check_attention(out, b, window)
    assert (out[b.tokens:] == 7).all(), "rows behind the last sequence were written"
    assert nb.take_device_error() == 0


@pytest.mark.parametrize("max_q", [1, 16, None, 10000])
def test_any_max_q_gives_the_result(max_q):
    """max_q selects a kernel; results hold whatever it says."""
    b = Batch([400, 90, 2], [100, 1, 2], 8, 2, 128, 16, BF, seed=3)
    check_attention(b.call(nb, max_q=max_q), b)


@pytest.mark.parametrize("news", [[1, 1], [3, 40]])
def test_an_unknown_max_q_with_the_workspace_of_any(news):
    b = Batch([700, 1900], news, 8, 2, 128, 16, torch.bfloat16, seed=8)
    size = nb.paged_attention_workspace_size(8, 2, 128, 0, b.table.shape[1] * b.page)
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")
    check_attention(b.call(nb, max_q=0, workspace=ws), b)
    check_attention(b.call(nb, max_q=0), b)
    check_attention(b.call(nb, max_q=1 << 62, workspace=ws), b)


@pytest.mark.parametrize("dtype", [BF, HF])
def test_scale_and_strided_cache(dtype):
    """Keys and values side by side in one tensor; a scale of the caller's."""
    b = Batch([300, 17], [1, 9], 8, 4, 128, 32, dtype, seed=4, interleaved=True)
    check_attention(b.call(nb, scale=0.3), b, scale=0.3)


@pytest.mark.parametrize("news", [[1, 1], [70, 200]])
def test_large_scores_and_equal_scores(news):
    """Scores of thousands (one key takes all) and rows of equal scores."""
    b = Batch([500, 333], news, 4, 2, 64, 16, BF, seed=5)
    check_attention(b.call(nb, scale=40.0), b, scale=40.0)
    b.q.zero_()
    check_attention(b.call(nb), b)


def test_infinite_keys_behind_the_mask():
    """Keys that a chunk's earlier tokens do not see may be infinite or NaN for them."""
    b = Batch([64], [8], 4, 2, 64, 16, BF, seed=6)
    page, slot = int(b.table[b.rows[0], 3]), 63 % 16
    b.k[page, :, slot] = float("inf")
    got = b.call(nb)[:7]
    b.dense[0][0][63] = 0
    want, bound = attention64(b)
    assert ((got.double() - want[:7]).abs() <= bound[:7] + 1e-12).all()


@pytest.mark.parametrize("news", [1, 40])
def test_offsets_past_32_bits(news):
    """The used pages lie more than 2^32 bytes into the cache."""
    page_elems = 8 * 256 * 128
    n_pages = (1 << 32) // (2 * page_elems) + (1 << 31) // (2 * page_elems) + 8
    b = Batch([600, 100], [news, 1], 8, 8, 128, 256, BF, seed=7, n_pages=n_pages)
    assert int(b.table.max()) * page_elems > 1 << 31
    check_attention(b.call(nb), b)


@pytest.mark.parametrize("news", [[1, 1, 1], [50, 1, 130]])
def test_padding_entries_are_skipped(news):
    b = Batch([90, 300, 200], news, 8, 2, 128, 16, BF, seed=8)
    want = b.call(nb)
    seqs, starts = b.seqs.clone(), b.starts
    seqs[1] = -1
    out = torch.full_like(want, 5.0)
    nb.paged_attention(b.q, b.k, b.v, b.table, b.row_lens, q_starts=starts, seqs=seqs, out=out)
    lo, hi = starts[1].item(), starts[2].item()
    keep = torch.ones(len(out), dtype=torch.bool)
    keep[lo:hi] = False
    assert torch.allclose(out[keep].float(), want[keep].float(), rtol=2 ** -6, atol=2 ** -8)
    assert (out[lo:hi] == 5).all()
    assert nb.take_device_error() == 0


@pytest.mark.parametrize("window", [1 << 20, 1 << 31, 1 << 62])
@pytest.mark.parametrize("news", [[1, 1], [40, 9]])
def test_a_window_longer_than_the_table(window, news):
    b = Batch([300, 9], news, 8, 2, 128, 16, BF, seed=14)
    assert torch.equal(b.call(nb, window=window), b.call(nb))


@pytest.mark.parametrize("news", [[1, 1, 1], [70, 1, 9]])
def test_strided_table_rows_and_queries(news):
    """A table that is a part of a wider one, queries and results in rows of others."""
    b = Batch([200, 90, 700], news, 8, 2, 64, 32, HF, seed=15)
    wide = torch.full((b.table.shape[0], b.table.shape[1] + 5), 1 << 20, dtype=torch.int32,
                      device="cuda")
    wide[:, :b.table.shape[1]] = b.table
    want = b.call(nb)
    room = torch.full((b.tokens, 3, 8, 64), 2.0, dtype=HF, device="cuda")
    got = nb.paged_attention(b.q, b.k, b.v, wide[:, :b.table.shape[1]], b.row_lens,
                             q_starts=b.starts, seqs=b.seqs, out=room[:, 1])
    assert torch.equal(got, want)
    assert (room[:, 0] == 2).all() and (room[:, 2] == 2).all()
    assert nb.take_device_error() == 0


def test_a_long_prompt_beside_many_steps():
    """More than 32 sequences, a prompt of several tiles among them."""
    lens = [700] + [17 * i % 600 + 1 for i in range(70)]
    b = Batch(lens, [700] + [1] * 70, 4, 2, 64, 32, BF, seed=16)
    check_attention(b.call(nb, max_q=700), b)


def test_two_streams_at_once():
    """Calls on two streams whose workspaces are torch's: each gets its own result."""
    bs = [Batch([3000, 40], [n, 1], 8, 2, 128, 16, BF, seed=17 + n) for n in (1, 50)]
    want = [b.call(nb).clone() for b in bs]
    streams = [torch.cuda.Stream() for _ in bs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, (b, s) in enumerate(zip(bs, streams)):
            with torch.cuda.stream(s):
                got[i].append(b.call(nb))
    torch.cuda.synchronize()
    for w, outs in zip(want, got):
        assert all(torch.equal(w, o) for o in outs)


def test_without_q_starts_and_seqs():
    b = Batch([90, 300, 200], [1, 1, 1], 8, 2, 128, 16, BF, seed=9)
    q = torch.empty_like(b.q)
    for i, r in enumerate(b.rows):
        q[r] = b.q[i]
    got = nb.paged_attention(q, b.k, b.v, b.table, b.row_lens)
    check_attention(torch.stack([got[r] for r in b.rows]), b)


@pytest.mark.parametrize("news", [[1, 1], [30, 200]])
def test_bad_tables_read_nothing_and_tell(news):
    """A missing page, one past the pool, a length past the table, a row past the table:
    the result is some number, the error word is raised."""
    b = Batch([300, 250], news, 8, 2, 128, 16, BF, seed=10)
    for spoil in ("missing", "past", "length", "row", "starts"):
        table, lens, seqs, starts = (t.clone() for t in (b.table, b.row_lens, b.seqs, b.starts))
        if spoil == "missing":
            table[:, 2] = -1
        elif spoil == "past":
            table[:, 0] = b.n_pages
        elif spoil == "length":
            lens[0] = 1 << 30
        elif spoil == "row":
            seqs[0] = 99
        else:
            starts[2] = 1 << 20
        out = nb.paged_attention(b.q, b.k, b.v, table, lens, q_starts=starts, seqs=seqs, max_q=300)
        assert out.shape == b.q.shape
        torch.cuda.synchronize()
        assert nb.take_device_error() == 2, spoil
    check_attention(b.call(nb), b)


def test_python_refusals():
    b = Batch([900, 30], [1, 1], 8, 2, 128, 16, BF, seed=11)  # (long enough for a workspace)
    ok = dict(q=b.q, k_pages=b.k, v_pages=b.v, table=b.table, kv_lens=b.row_lens)
    bad = [dict(q=b.q.half()), dict(q=b.q[:, :, :64]), dict(q=b.q.transpose(0, 1)),
           dict(q=b.q[:, :7]), dict(k_pages=b.k.float(), v_pages=b.v.float()),
           dict(v_pages=b.v[:-1]), dict(k_pages=b.k[..., ::2], v_pages=b.v[..., ::2]),
           dict(table=b.table.long()), dict(table=b.table.t()), dict(table=b.table.cpu()),
           dict(kv_lens=b.row_lens[:1]), dict(kv_lens=b.row_lens.float()),
           dict(q_starts=b.starts[:2], seqs=b.seqs), dict(seqs=b.seqs.long()), dict(scale=0.0),
           dict(window=-1), dict(out=torch.empty_like(b.q[:1])), dict(out=b.q.float()),
           dict(workspace=torch.empty(16, dtype=torch.uint8, device="cuda")),
           dict(q=b.q.cpu()), dict(max_q=-1, q_starts=b.starts)]
    for kw in bad:
        with pytest.raises(nb.NQError):
            nb.paged_attention(**{**ok, **kw})
    nb.paged_attention(**ok)


@pytest.mark.parametrize("news", [[1, 1, 1], [33, 1, 140]])
def test_attention_on_a_stream_and_in_a_graph(news):
    """A captured call with a workspace of its own replays on new inputs; two streams
    with a workspace each do not disturb one another."""
    b = Batch([400, 900, 200], news, 8, 2, 128, 16, BF, seed=12)
    want = b.call(nb, max_q=max(news)).clone()
    size = nb.paged_attention_workspace_size(8, 2, 128, max(news), b.table.shape[1] * 16)
    ws = [torch.empty(size, dtype=torch.uint8, device="cuda") for _ in range(2)]
    outs = [torch.zeros_like(want) for _ in range(2)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        b.call(nb, max_q=max(news), out=outs[0], workspace=ws[0])
    for _ in range(3):
        graph.replay()
        with torch.cuda.stream(s):
            b.call(nb, max_q=max(news), out=outs[1], workspace=ws[1])
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want) and torch.equal(outs[1], want)
    b.row_lens -= 1
    other = b.call(nb, max_q=max(news)).clone()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], other) and not torch.equal(other, want)


def test_attention_is_deterministic():
    b = Batch([3000, 100, 2000], [1, 90, 1], 8, 1, 128, 16, BF, seed=13)
    first = b.call(nb)
    assert all(torch.equal(first, b.call(nb)) for _ in range(5))


# ------------------------------------------------------------------- append

@pytest.mark.parametrize("group", [33, 7, 65])
def test_rows_that_fill_no_tile_do_not_see_what_ran_before(group):
    """128 / group tokens leave rows of a tile of 128 unused; another call's queries in their
    place must not change a bit of the result."""
    b = Batch([500], [500], group, 1, 128, 256, HF, seed=12)
    want = b.call(nb, max_q=500).clone()
    check_attention(want, b)
    other = Batch([600], [600], 128, 1, 128, 16, HF, seed=13)
    q = other.q.clone()
    for factor in (0.0, 5.0, 40.0, 400.0):
        other.q.copy_(q * factor)
        other.call(nb, max_q=600)
        assert torch.equal(b.call(nb, max_q=500), want)


def rotate64(x, pos, freqs):
    f = freqs.numel()
    a = pos.double()[:, None] * freqs.double()
    c, s = a.cos()[:, None], a.sin()[:, None]
    x = x.double()
    x1, x2 = x[..., :f], x[..., f:2 * f]
    return torch.cat([x1 * c - x2 * s, x1 * s + x2 * c, x[..., 2 * f:]], dim=-1)


APPEND = [([1], [1], 4, 4, 64, 16, BF, 32), ([200, 17, 64, 1], [1, 1, 1, 1], 32, 8, 128, 16, BF, 64),
          ([300, 50, 5], [130, 50, 2], 8, 2, 128, 32, HF, 64), ([33, 900], [33, 7], 6, 2, 256, 48, BF, 128),
          ([70], [20], 4, 1, 128, 64, BF, 16), ([40, 0, 9], [4, 0, 9], 4, 2, 64, 16, HF, 0),
          ([500000], [100], 2, 1, 64, 256, BF, 32)]


@pytest.mark.parametrize("i", range(len(APPEND)))
@pytest.mark.parametrize("in_place", [False, True])
def test_append(i, in_place):
    """q and k: the turn's rounding (u |x|) and fp32's: four roundings of 2^-24 on
    |x1| + |x2| and the angle's 2^-22."""
    lens, news, heads, kv, dim, page, dtype, nf = APPEND[i]
    b = Batch(lens, news, heads, kv, dim, page, dtype, seed=i, extra_rows=1)
    g = torch.Generator(device="cuda").manual_seed(i)
    kn = torch.randn((b.tokens + 1, kv, dim), device="cuda", generator=g).to(dtype)
    vn = torch.randn((b.tokens + 1, kv, dim), device="cuda", generator=g).to(dtype)
    freqs = nb.rope_frequencies(2 * nf, 500000.0) if nf else None
    k0, v0, q0 = b.k.clone(), b.v.clone(), b.q.clone()
    q_out = b.q if in_place else torch.full_like(b.q, 9.0)
    assert nb.paged_append(b.q, kn, vn, b.k, b.v, b.table, b.row_lens, q_starts=b.starts, seqs=b.seqs,
                           freqs=freqs, q_out=q_out) is q_out
    assert nb.take_device_error() == 0
    u = torch.finfo(dtype).eps / 2
    f = freqs if nf else torch.zeros(0, device="cuda")
    kt, vt = k0.clone(), v0.clone()
    kb = torch.zeros(k0.shape, dtype=torch.float64, device="cuda")
    kw = k0.double()
    at = 0
    for e, (n, m) in enumerate(zip(lens, news)):
        pos = torch.arange(n - m, n, device="cuda")
        pages = b.table[b.rows[e]].long()[pos // page]
        for x, is_q in ((q0[at:at + m], True), (kn[at:at + m], False)):
            want = rotate64(x, pos, f)
            mag = x.double().abs()
            mag = torch.cat([mag[..., :nf] + mag[..., nf:2 * nf]] * 2 + [mag[..., 2 * nf:] * 0], dim=-1)
            bound = u * want.abs() + (4 * 2.0 ** -24 + 2.0 ** -22) * mag * (1 + u)
            if is_q:
                assert ((q_out[at:at + m].double() - want).abs() <= bound).all()
            else:
                kw[pages, :, pos % page] = want
                kb[pages, :, pos % page] = bound
        vt[pages, :, pos % page] = vn[at:at + m]
        at += m
    same = lambda x, y: torch.equal(torch.nan_to_num(x, 77.0), torch.nan_to_num(y, 77.0))  # noqa: E731
    assert same(b.v, vt)
    diff = (b.k.double() - kw).abs()
    assert (torch.isnan(diff) | (diff <= kb)).all()
    assert torch.equal(torch.isnan(b.k), torch.isnan(kw))
    assert torch.equal(q_out[b.tokens:], q0[b.tokens:] if in_place else torch.full_like(q0[b.tokens:], 9.0))


def test_append_tells_what_it_cannot_store():
    b = Batch([20, 3], [4, 5], 4, 2, 64, 16, BF, seed=2)
    kn = torch.randn((b.tokens, 2, 64), device="cuda").to(BF)
    before = b.v.clone()
    nb.paged_append(b.q, kn, kn, b.k, b.v, b.table, b.row_lens, q_starts=b.starts, seqs=b.seqs)
    assert nb.take_device_error() == 2  # the second entry's first two tokens have no position
    table = torch.full_like(b.table, b.n_pages)
    b.v.copy_(before)
    nb.paged_append(b.q, kn, kn, b.k, b.v, table, b.row_lens, q_starts=b.starts, seqs=b.seqs)
    assert nb.take_device_error() == 2
    assert torch.equal(torch.nan_to_num(b.v, 7.0), torch.nan_to_num(before, 7.0))
    for kw in (dict(k=kn[:1]), dict(v=kn.half()), dict(freqs=torch.zeros(32, device="cuda").half()),
               dict(freqs=torch.zeros(40, device="cuda")), dict(freqs=torch.zeros(12, device="cuda")),
               dict(q_out=b.q[:1]), dict(k=kn[:, :1])):
        with pytest.raises(nb.NQError):
            nb.paged_append(**{**dict(q=b.q, k=kn, v=kn, k_pages=b.k, v_pages=b.v, table=b.table,
                                      kv_lens=b.row_lens, q_starts=b.starts, seqs=b.seqs), **kw})


# --------------------------------------------------------------- page pool

class Device:
    """A pool on the device beside its model; every page's contents are its own number
    until a copy."""

    def __init__(self, n_pages, rows, width, page=16, layers=3, kv=2, dim=64, dtype=BF):
        self.model = Pool(n_pages, rows, width, page)
        self.pool = torch.zeros((layers, 2, n_pages, kv, page, dim), dtype=dtype, device="cuda")
        self.pool += torch.arange(n_pages, device="cuda").view(1, 1, -1, 1, 1, 1) % 200
        self.refs = torch.zeros(n_pages, dtype=torch.int32, device="cuda")
        self.table = torch.full((rows, width), -1, dtype=torch.int32, device="cuda")
        self.lens = torch.zeros(rows, dtype=torch.int32, device="cuda")
        self.content = [p % 200 for p in range(n_pages)]

    def ids(self, x):
        return torch.tensor(x, dtype=torch.int32, device="cuda")

    def free(self, seqs):
        self.model.free(seqs)
        nb.pages_free(self.refs, self.table, self.lens, self.ids(seqs))

    def fork(self, parents, children):
        self.model.fork(parents, children)
        nb.pages_fork(self.refs, self.table, self.lens, self.ids(parents), self.ids(children))

    def reserve(self, seqs, lens):
        for a, b in self.model.reserve(seqs, lens):
            self.content[b] = self.content[a]
        nb.pages_reserve(self.pool, self.refs, self.table, self.lens, self.ids(seqs), self.ids(lens))

    def compact(self):
        for a, b in self.model.compact():
            self.content[b] = self.content[a]
        nb.pages_compact(self.pool, self.refs, self.table)

    def check(self):
        assert self.refs.tolist() == self.model.refs
        assert self.table.tolist() == self.model.table
        assert self.lens.tolist() == self.model.lens
        want = torch.tensor(self.content, dtype=self.pool.dtype, device="cuda").view(1, 1, -1, 1, 1, 1)
        assert (self.pool == want).all()
        assert nb.take_device_error() == self.model.errors
        self.model.errors = 0


def test_pool_step_by_step():
    d = Device(40, 8, 6)
    d.reserve([0, 1, 2], [20, 16, 1])
    d.check()
    d.fork([0, 0, 1], [3, 4, 5])
    d.check()
    d.reserve([0, 3, 4, 5], [21, 40, 20, 17])  # 4 keeps its length: no copy
    d.check()
    d.reserve([4], [22])                        # the only holder left: no copy
    d.check()
    d.free([0, -1, 0, 3])
    d.check()
    d.compact()
    d.check()
    d.compact()
    d.check()


def test_all_holders_of_a_page_grow_at_once():
    d = Device(64, 12, 4)
    d.reserve([0], [5])
    d.fork([0] * 5, [1, 2, 3, 4, 5])
    d.reserve([5, 0, 3, 1, 2, 4], [6, 6, 6, 6, 6, 6])  # the last of the list keeps the page
    d.check()
    assert d.table[4, 0].item() == 0


def test_refused_requests_leave_everything():
    d = Device(6, 5, 3)
    d.reserve([0], [40])
    d.check()
    for seqs, lens in (([1, 2], [48, 16]), ([0], [39]), ([1], [49]), ([1, 1], [1, 2]), ([7], [1]),
                       ([1, 0], [10, 3])):
        d.reserve(seqs, lens)
        assert d.model.errors == 4
        d.check()
    d.fork([0, 0, 1, 0, 9, -1], [1, 1, 2, 0, 3, 4])
    assert d.model.errors == 4
    d.check()
    d.free([9])
    assert d.model.errors == 4
    d.check()
    d.reserve([-1, 2, -1], [5, 16, 0])  # padding
    d.check()
    d.fork([-1], [-1])
    d.check()


@pytest.mark.parametrize("seed", range(6))
def test_pool_at_random(seed):
    rng = random.Random(seed)
    rows, page = rng.choice([8, 70]), rng.choice([16, 32])
    d = Device(rng.choice([50, 400, 2500]), rows, rng.choice([5, 40]), page=page,
               dtype=rng.choice([BF, HF]))
    for _ in range(25):
        op = rng.choice(["reserve", "reserve", "fork", "free", "compact"])
        some = rng.sample(range(rows), rng.randint(1, rows // 2))
        if op == "reserve":
            d.reserve(some, [d.model.lens[s] + rng.choice([0, 1, 3, 2 * page]) for s in some])
        elif op == "fork":
            d.fork([rng.randrange(rows) for _ in some], some)
        elif op == "free":
            d.free([s for s in some if rng.random() < 0.6] or [-1])
        else:
            d.compact()
        d.check()


def test_many_sequences_and_pages():
    d = Device(9000, 1500, 7, layers=1, kv=1)
    order = list(range(1500))
    random.Random(1).shuffle(order)
    d.reserve(order, [random.Random(s).randint(1, 90) for s in order])
    d.check()
    d.free(order[::3])
    d.compact()
    d.check()


def test_copy_pages():
    d = Device(30, 2, 2)
    nb.copy_pages(d.pool, d.ids([3, 3, 7, -1, 9]), d.ids([0, 1, 20, -1, 9]))
    for a, b in ((3, 0), (3, 1), (7, 20)):
        d.content[b] = d.content[a]
    d.check()
    # a target that is a source, or listed before, or out of range: that move is not made
    nb.copy_pages(d.pool, d.ids([5, 6, 8, 30, 11]), d.ids([6, 12, 12, 13, 14]))
    d.content[12], d.content[14] = d.content[6], d.content[11]
    d.model.errors = 4
    d.check()


def test_pool_refusals():
    d = Device(8, 4, 4)
    one = d.ids([1])
    for call in (lambda: nb.pages_free(d.refs.long(), d.table, d.lens, one),
                 lambda: nb.pages_free(d.refs, d.table, d.lens[:2], one),
                 lambda: nb.pages_free(d.refs, d.table, d.lens, one.cpu()),
                 lambda: nb.pages_free(d.refs.cpu(), d.table.cpu(), d.lens.cpu(), one.cpu()),
                 lambda: nb.pages_fork(d.refs, d.table, d.lens, one, d.ids([1, 2])),
                 lambda: nb.pages_reserve(d.pool[:, :, :7], d.refs, d.table, d.lens, one, one),
                 lambda: nb.pages_reserve(d.pool[:, :, :7].contiguous(), d.refs, d.table, d.lens, one, one),
                 lambda: nb.pages_reserve(d.pool, d.refs, d.table, d.lens, one, d.ids([1, 2])),
                 lambda: nb.pages_reserve(d.pool, d.refs, d.table, d.lens, one, one,
                                          workspace=torch.empty(256, dtype=torch.uint8, device="cuda")),
                 lambda: nb.pages_compact(d.pool.cpu(), d.refs, d.table),
                 lambda: nb.copy_pages(d.pool, one, d.ids([1, 2])),
                 lambda: nb.copy_pages(d.pool, one.long(), one.long())):
        with pytest.raises(nb.NQError):
            call()
    d.check()


def test_pool_calls_in_a_graph():
    """A decode step's bookkeeping, captured once and replayed: lengths advance on the
    device, pages appear as they are needed."""
    d = Device(60, 4, 10)
    seqs = d.ids([0, 1, -1])
    new = d.ids([30, 16, 0])
    ws = torch.empty(1 << 16, dtype=torch.uint8, device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        nb.pages_reserve(d.pool, d.refs, d.table, d.lens, seqs, new, workspace=ws)
        new += 1
    for step in range(20):
        graph.replay()
        d.model.reserve([0, 1, -1], [30 + step, 16 + step, 0])
    d.check()


# ----------------------------------------------------------- all of them together

@pytest.mark.parametrize("dtype,dim,heads,kv,page", [(BF, 128, 8, 2, 16), (HF, 64, 6, 3, 32)])
def test_serving_run(dtype, dim, heads, kv, page):
    """Prompts in chunks, a fork, single steps, an end, a compaction: after every step the
    attention of every new token is held against 64 bits over the keys as they were
    appended."""
    g = torch.Generator(device="cuda").manual_seed(1)
    rows, width, n_pages = 6, 24, 90
    pool = torch.full((1, 2, n_pages, kv, page, dim), float("nan"), dtype=dtype, device="cuda")
    refs = torch.zeros(n_pages, dtype=torch.int32, device="cuda")
    table = torch.full((rows, width), -1, dtype=torch.int32, device="cuda")
    lens = torch.zeros(rows, dtype=torch.int32, device="cuda")
    freqs = nb.rope_frequencies(dim, 10000.0, device="cuda")
    ids = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    hist = {}

    def step(seqs, news):
        now = [len(hist.get(s, (torch.zeros(0),))[0]) + m for s, m in zip(seqs, news)]
        nb.pages_reserve(pool, refs, table, lens, ids(seqs), ids(now))
        n = sum(news)
        q = torch.randn((n, heads, dim), device="cuda", generator=g).to(dtype)
        k = torch.randn((n, kv, dim), device="cuda", generator=g).to(dtype)
        v = torch.randn((n, kv, dim), device="cuda", generator=g).to(dtype)
        starts = ids([sum(news[:i]) for i in range(len(news) + 1)])
        kw = dict(q_starts=starts, seqs=ids(seqs))
        qr = nb.paged_append(q, k, v, pool[0, 0], pool[0, 1], table, lens, freqs=freqs, **kw)
        out = nb.paged_attention(qr, pool[0, 0], pool[0, 1], table, lens, max_q=max(news), **kw)
        b = Batch.__new__(Batch)
        b.lens, b.news, b.heads, b.kv_heads, b.dim, b.dtype = now, news, heads, kv, dim, dtype
        b.tokens, b.q, b.dense = n, qr, []
        at = 0
        for s, m, full in zip(seqs, news, now):
            pos = torch.arange(full - m, full, device="cuda")
            kk = rotate64(k[at:at + m], pos, freqs).to(dtype)
            old = hist.get(s, (k[:0], v[:0]))
            hist[s] = (torch.cat([old[0], kk]), torch.cat([old[1], v[at:at + m]]))
            b.dense.append(hist[s])
            at += m
        # the cache's keys may differ from these by one rounding: allow for it as for the
        # scores' own error (u |q| |k| in the exponent, on numerator and denominator)
        want, bound = attention64(b)
        u = torch.finfo(dtype).eps / 2
        diff = (out.double() - want).abs()
        assert torch.isfinite(out).all()
        rare = diff > bound + 1e-12
        assert rare.float().mean() < 0.01 and (diff <= bound + 2 * u * 8).all()

    step([0, 2], [70, 33])
    step([0, 2, 3], [150, 1, 5])
    nb.pages_fork(refs, table, lens, ids([0, 0]), ids([1, 4]))
    hist[1], hist[4] = hist[0], hist[0]
    for _ in range(3):
        step([0, 1, 2, 3, 4], [1, 1, 1, 1, 1])
    nb.pages_free(refs, table, lens, ids([0, 3]))
    del hist[0], hist[3]
    nb.pages_compact(pool, refs, table)
    step([4, 5, 1, 2], [20, 40, 1, 1])
    step([1, 2, 4, 5], [1, 1, 1, 1])
    used = int((refs > 0).sum())
    assert (refs[:used] > 0).all() or used <= n_pages
    assert nb.take_device_error() == 0


# ------------------------------------------------------------- workspaces

@pytest.mark.parametrize("byte", [0, 1, 0x7f, 0xff])
@pytest.mark.parametrize("lens,news", [([3000, 40], [1, 1]), ([1500, 700], [1, 90]),
                                       ([1400], [1400])])
def test_what_a_workspace_holds_does_not_matter(lens, news, byte):
    """Cut tiles, and CTAs without a tile of their own, beside any bytes."""
    b = Batch(lens, news, 8, 2, 128, 16, BF, seed=31)
    want = b.call(nb, max_q=max(news)).clone()
    size = nb.paged_attention_workspace_size(8, 2, 128, max(news), b.table.shape[1] * 16)
    assert size > 0
    ws = torch.full((size,), byte, dtype=torch.uint8, device="cuda")
    out = torch.full((b.tokens + 1, 8, 128), 3.0, dtype=BF, device="cuda")
    b.q = torch.cat([b.q, b.q[:1]])
    got = b.call(nb, max_q=max(news), workspace=ws, out=out)
    assert torch.equal(got[:b.tokens], want)
    assert (got[b.tokens:] == 3).all()
    assert nb.take_device_error() == 0


# -------------------------------------------------------------------- NaN

@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("lens,news", [([200, 40], [1, 1]), ([6000, 40], [1, 1]), ([900, 700], [3, 1]),
                                       ([2000, 700], [150, 1])])
def test_nan_reaches_its_row_alone(lens, news, dtype):
    """A NaN in a query makes that head's row NaN, however the keys are split over the CTAs, and
    one in a key the rows that see it; the other rows stay right."""
    b = Batch(lens, news, 8, 2, 128, 16, dtype, seed=41)
    want, bound = attention64(b)
    right = lambda x, rows: ((x.double() - want).abs() <= bound + 1e-12)[rows].all()  # noqa: E731
    q = b.q.clone()
    b.q = q.clone()
    b.q[0, 5, 17] = float("nan")
    got = b.call(nb, max_q=max(news))
    assert torch.isnan(got[0, 5]).all()
    other = torch.ones(got.shape[:2], dtype=torch.bool, device="cuda")
    other[0, 5] = False
    assert right(got, other)
    # a key of the first sequence's second head that all of its new tokens see
    b.q = q
    at = lens[0] - news[0] - 3
    b.k[int(b.table[b.rows[0], at // 16]), 1, at % 16, 9] = float("nan")
    got = b.call(nb, max_q=max(news))
    assert torch.isnan(got[:news[0], 4:]).all()
    other[:] = True
    other[:news[0], 4:] = False
    assert right(got, other)
    assert nb.take_device_error() == 0


@pytest.mark.parametrize("page,width", [(16, 40), (128, 9)])
def test_a_step_in_the_workspace_of_a_chunk(page, width):
    """The workspace of a larger max_q, through the C call without q_starts too."""
    import ctypes
    from neurons_b200 import paged
    from neurons_b200._lib import lib
    b = Batch([600, 90, 300], [1, 1, 1], 8, 2, 128, page, BF, seed=51)
    table = torch.full((3, width), -1, dtype=torch.int32, device="cuda")
    table[:, :b.table.shape[1]] = b.table[:, :width]
    b.table = table
    size = nb.paged_attention_workspace_size(8, 2, 128, 512, width * page)
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")
    want = b.call(nb, max_q=1)
    check_attention(want, b)
    assert torch.equal(b.call(nb, max_q=1, workspace=ws), want)
    out = torch.zeros_like(want)
    cache = paged.Cache(b.k.data_ptr(), b.v.data_ptr(), b.n_pages, b.k.stride(0), 2, page, 128, 1)
    batch = paged.Batch(table.data_ptr(), width, width, 3, b.row_lens.data_ptr(), b.seqs.data_ptr(),
                        None, 3, 3)
    assert lib().nq_paged_attention(b.q.data_ptr(), b.q.stride(0), 8, ctypes.byref(cache),
                                    ctypes.byref(batch), 512, 128 ** -0.5, 0, ws.data_ptr(), size,
                                    out.data_ptr(), out.stride(0), None) == 0
    torch.cuda.synchronize()
    assert torch.equal(out, want)


@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("spoil", ["length", "row", "starts"])
def test_append_leaves_out_an_entry_that_is_out_of_range(spoil, new):
    """Its tokens have no position: nothing is written over the keys that are there."""
    g = torch.Generator(device="cuda").manual_seed(5)
    draw = lambda *shape: torch.randn(shape, device="cuda", generator=g).to(BF)  # noqa: E731
    k, v = draw(16, 2, 16, 64), draw(16, 2, 16, 64)
    table = torch.randperm(16, device="cuda", generator=g).to(torch.int32).view(2, 8)  # all full
    lens = torch.tensor([128, 100], dtype=torch.int32, device="cuda")
    seqs = torch.tensor([1, 0], dtype=torch.int32, device="cuda")
    starts = torch.tensor([0, 3, 3 + new], dtype=torch.int32, device="cuda")
    q, kn, vn = draw(3 + new, 4, 64), draw(3 + new, 2, 64), draw(3 + new, 2, 64)
    want = [x.clone() for x in (k, v, q)]
    for t in range(3):  # the entry before it is stored as ever
        page, slot = int(table[1, (97 + t) // 16]), (97 + t) % 16
        want[0][page, :, slot], want[1][page, :, slot] = kn[t], vn[t]
    if spoil == "length":
        lens[0] = 128 + new
    elif spoil == "row":
        seqs[1] = 2
    else:
        starts[2] += 1
    q_out = torch.full_like(q, 9.0)
    nb.paged_append(q, kn, vn, k, v, table, lens, q_starts=starts, seqs=seqs, q_out=q_out)
    assert nb.take_device_error() == 2
    assert torch.equal(k, want[0]) and torch.equal(v, want[1])
    assert torch.equal(q_out[:3], q[:3]) and (q_out[3:] == 9).all()


# ------------------------------------------------------- what sits side by side

@pytest.mark.parametrize("lens,news,heads,kv,dim,page,dtype,window", [
    ([2400, 1700], [700, 90], 4, 2, 256, 16, BF, 1024),   # 32 boxes a block, a ring of one block
    ([1500], [33], 8, 4, 256, 16, HF, 300),
    ([1400, 1300], [150, 1], 8, 4, 256, 128, BF, 1024),
    ([3000], [200], 4, 1, 128, 16, HF, 1024),
    ([900, 2000], [600, 3], 4, 2, 64, 16, BF, 500),
])
def test_windows_over_many_blocks(lens, news, heads, kv, dim, page, dtype, window):
    b = Batch(lens, news, heads, kv, dim, page, dtype, seed=61, window=window)
    check_attention(b.call(nb, window=window, max_q=max(news)), b, window)
    assert nb.take_device_error() == 0


@pytest.mark.parametrize("lens,news", [([200], [1]), ([1, 17, 250, 64], [1] * 4), ([90, 300], [30, 1])])
def test_short_sequences_in_a_wide_table(lens, news):
    """A server's table has room for its longest sequence: short ones are cut and joined
    there, where a table as wide as they are leaves their tiles whole."""
    b = Batch(lens, news, 8, 2, 128, 16, BF, seed=62)
    want = b.call(nb, max_q=max(news))
    wide = torch.full((len(lens), 600), -1, dtype=torch.int32, device="cuda")
    wide[:, :b.table.shape[1]] = b.table
    b.table = wide
    got = b.call(nb, max_q=max(news))
    check_attention(got, b)
    check_attention(want, b)
    assert nb.take_device_error() == 0


@pytest.mark.parametrize("seed", range(12))
def test_attention_at_random(seed):
    """Batches of any make: group sizes that do and do not divide a tile, pages, windows,
    entries without tokens or longer than their sequence; and the same bits again."""
    rng = random.Random(1000 + seed)
    kv = rng.choice([1, 2, 3])
    group = rng.choice([1, 2, 3, 4, 5, 7, 8, 12, 16, 17, 33, 64, 100])
    dim, page = rng.choice([64, 128, 256]), rng.choice([16, 32, 48, 64, 80, 128, 144, 256])
    dtype, window = rng.choice([BF, HF]), rng.choice([0, 0, 1, 15, 64, 200, 1000])
    n = rng.choice([1, 2, 5, 40])
    lens = [rng.choice([0, 1, rng.randint(2, 70), rng.randint(100, 1500)]) for _ in range(n)]
    many = rng.choice([1, 1, 4, 40, 300])
    news = [rng.choice([0, 1, rng.randint(1, many)]) for _ in range(n)]
    news[0] = max(news[0], 1)
    if rng.random() < 0.7:  # (else some rows have no key)
        lens = [max(a, m) for a, m in zip(lens, news)]
    b = Batch(lens, news, kv * group, kv, dim, page, dtype, seed=seed, window=window)
    max_q = rng.choice([None, max(news), 1])
    got = b.call(nb, window=window, max_q=max_q)
    check_attention(got, b, window)
    assert torch.equal(b.call(nb, window=window, max_q=max_q), got)
    assert nb.take_device_error() == 0


def test_compaction_leaves_the_used_pages_in_front():
    """refs and table right after a compaction, beside shared and half-used pages."""
    d = Device(120, 10, 8)
    d.reserve([0, 1, 2, 3], [100, 40, 128, 1])
    d.fork([0, 2], [4, 5])
    d.reserve([4, 5, 6], [101, 128, 60])
    d.free([1, 0])
    nb.take_device_error()
    used = int((d.refs > 0).sum())
    assert int(d.table.max()) >= used  # (there is something to move)
    d.compact()
    assert (d.refs[:used] > 0).all() and (d.refs[used:] == 0).all()
    assert int(d.table.max()) == used - 1
    d.check()


@pytest.mark.parametrize("lens,news,heads,kv,dim,page,dtype", [
    ([200], [1], 32, 8, 128, 16, BF), ([1, 2, 1000, 37, 513], [1] * 5, 8, 1, 128, 32, BF),
    ([5000, 3], [1, 1], 4, 2, 64, 16, BF), ([700, 33], [1, 1], 8, 4, 256, 16, BF),
    ([900, 64], [4, 2], 8, 2, 128, 64, BF), ([900, 5000], [2, 1], 32, 4, 64, 64, HF)])
def test_few_rows_keep_the_weights(lens, news, heads, kv, dim, page, dtype):
    """A decode step's weights are held in two terms of the cache's type: of their rounding,
    u sum p |v| in attention64()'s bound, u^2 sum p |v| is left."""
    b = Batch(lens, news, heads, kv, dim, page, dtype, seed=71)
    want, bound = attention64(b)
    u = torch.finfo(dtype).eps / 2
    dense, b.dense = b.dense, [(k, v.abs()) for k, v in b.dense]
    bound -= (u - u * u) * attention64(b)[0]  # (its result with |v|: sum p |v| / sum p)
    b.dense = dense
    got = b.call(nb, max_q=max(news)).double()
    over = (got - want).abs() - bound
    assert (over <= 1e-12).all(), f"{over.max().item():.3e} over the bound"


@pytest.mark.parametrize("many", [1, 60])
def test_batches_of_padding_gaps_and_repeats(many):
    """Nothing but padding; rows in front of the first entry; a sequence listed twice."""
    b = Batch([900, 300], [many, many], 8, 2, 128, 16, BF, seed=81)
    want = b.call(nb, max_q=many).clone()
    kw = dict(max_q=many, scale=None)
    out = torch.full_like(want, 4.0)
    nb.paged_attention(b.q, b.k, b.v, b.table, b.row_lens, q_starts=b.starts,
                       seqs=torch.full_like(b.seqs, -1), out=out, **kw)
    assert (out == 4).all()
    # five rows of another's before the first entry
    q = torch.cat([torch.full_like(want[:1], float("nan")).repeat(5, 1, 1), b.q])
    out = torch.full((len(q), 8, 128), 4.0, dtype=BF, device="cuda")
    nb.paged_attention(q, b.k, b.v, b.table, b.row_lens, q_starts=b.starts + 5, seqs=b.seqs, out=out,
                       **kw)
    assert (out[:5] == 4).all()
    check_attention(out[5:], b)
    # each sequence twice, for the same new tokens
    starts = torch.cat([b.starts, b.starts[1:] + b.starts[-1]])
    got = nb.paged_attention(torch.cat([b.q, b.q]), b.k, b.v, b.table, b.row_lens, q_starts=starts,
                             seqs=torch.cat([b.seqs, b.seqs]), **kw)
    check_attention(got[:b.tokens], b)
    check_attention(got[b.tokens:], b)
    assert nb.take_device_error() == 0


@pytest.mark.parametrize("most", [1, 20])
def test_a_batch_of_many_sequences(most):
    """1500 entries, padding among them: more than a warp's lanes many times over."""
    rng = random.Random(9)
    lens = [rng.choice([1, 16, 40, rng.randint(1, 90)]) for _ in range(1500)]
    news = [min(n, rng.randint(1, most)) for n in lens]
    b = Batch(lens, news, 4, 2, 64, 16, BF, seed=82)
    check_attention(b.call(nb, max_q=most), b)
    check_attention(b.call(nb), b)
    want = b.call(nb, max_q=most)
    seqs = b.seqs.clone()
    gone = torch.rand(1500, device="cuda", generator=torch.Generator("cuda").manual_seed(1)) < 0.4
    seqs[gone] = -1
    out = torch.full_like(want, 4.0)
    nb.paged_attention(b.q, b.k, b.v, b.table, b.row_lens, q_starts=b.starts, seqs=seqs, max_q=most,
                       out=out)
    row_gone = gone.repeat_interleave(torch.tensor(news, device="cuda"))
    assert (out[row_gone] == 4).all()
    out[row_gone] = want[row_gone]
    check_attention(out, b)
    assert nb.take_device_error() == 0


def test_values_that_are_the_keys():
    """One tensor as keys and values, in pages of a whole sequence."""
    b = Batch([700, 1500], [1, 30], 4, 1, 128, 2048, BF, seed=83)
    b.v = b.k
    b.dense = [(k, k) for k, _ in b.dense]
    check_attention(b.call(nb), b)
    check_attention(b.call(nb, max_q=1), b)
