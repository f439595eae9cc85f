"""GPU parity of the Llama paths over a paged cache: prompts in chunks against the
oracle's decode function (oracle/llama_oracle.py), and PagedLlama's batched steps, forks,
frees and compaction against one decoder per sequence.  Logits: normwise error <= 1e-2,
as for the decode step (tests/test_gpu_llama.py): each step's inputs differ only through
earlier bf16 rounding flips."""
import ctypes

import numpy as np
import pytest
import torch

import neurons_b200 as nb
from neurons_b200._lib import lib
from neurons_b200.llama import LlamaDecoder, PagedLlama
from test_gpu_llama import SMALL, check_logits, make_model

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def model(oracle):
    return make_model(oracle, dict(SMALL, max_context=650), 21)


def cfg():
    return dict(SMALL, max_context=650)  # (not a multiple of a page's 16 keys)


@pytest.mark.parametrize("chunk", [1, 7, 64, 300, 1000])
def test_chunked_prompt_matches_the_oracle(oracle, nqlib, model, chunk):
    from oracle.llama_oracle import LlamaOracle
    host, dev = model
    dec, ora = LlamaDecoder(cfg(), dev), LlamaOracle(cfg(), host)
    toks = np.random.default_rng(5).integers(0, SMALL["vocab"], 150).astype(np.int32)
    for t in toks:
        ref, _ = ora.step(int(t))
    dec.set_prefill_chunk(chunk)
    lg = dec.prefill(torch.from_numpy(toks).cuda())
    torch.cuda.synchronize()
    check_logits(oracle, lg, ref, f"chunk {chunk}")
    assert dec.position == 150
    # the decode step goes on over the chunks' keys, from the prompt's own next token
    token = int(lg.argmax())
    for i in range(3):
        lg, nxt = dec.step(None)
        ref, _ = ora.step(token)
        torch.cuda.synchronize()
        check_logits(oracle, lg, ref, f"chunk {chunk}, step {i}")
        token = int(nxt.item())
    assert nb.take_device_error() == 0


def test_a_second_prompt_continues_the_first(oracle, nqlib, model):
    _, dev = model
    toks = torch.randint(0, SMALL["vocab"], (200,), dtype=torch.int32, device="cuda")
    one, two = LlamaDecoder(cfg(), dev), LlamaDecoder(cfg(), dev)
    one.set_prefill_chunk(64)
    two.set_prefill_chunk(64)
    a = one.prefill(toks)
    two.prefill(toks[:100], logits=False)
    b = two.prefill(toks[100:])
    assert (a - b).norm() <= 1e-2 * a.norm()
    two.set_prefill_chunk(0)
    two.reset()
    c = two.prefill(toks)  # by the decode step, as before
    assert (a - c).norm() <= 1e-2 * a.norm()


def test_chunked_prompt_in_a_graph(nqlib, model):
    _, dev = model
    toks = torch.randint(0, SMALL["vocab"], (90,), dtype=torch.int32, device="cuda")
    dec = LlamaDecoder(cfg(), dev)
    dec.set_prefill_chunk(40)
    want = dec.prefill(toks).clone()
    dec.reset()
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        got = dec.prefill(toks)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want)
    assert nb.take_device_error() == 0


def close(a, b, what):
    err = ((a - b).norm() / b.norm()).item()
    assert err < 1e-2, f"{what}: {err:.3e}"


@pytest.mark.parametrize("page_size", [16, 128])
def test_paged_serving_matches_single_sequences(nqlib, model, page_size):
    """Prompts of several lengths in one step, a fork, single tokens, a chunk beside them, an
    end, a compaction: every sequence's logits are those of a decoder of its own."""
    _, dev = model
    g = torch.Generator().manual_seed(3)
    dec = LlamaDecoder(cfg(), dev)
    srv = PagedLlama(dec, n_pages=2400 // page_size, page_size=page_size, max_seqs=6, max_len=500)
    said = {}

    def step(seqs, news):
        toks = [torch.randint(0, SMALL["vocab"], (m,), dtype=torch.int32, generator=g) for m in news]
        lg, nxt = srv.step(seqs, torch.cat(toks).cuda(), news)
        for i, (s, t) in enumerate(zip(seqs, toks)):
            said[s] = torch.cat([said.get(s, t[:0]), t])
            own = LlamaDecoder(cfg(), dev)
            own.set_prefill_chunk(600)
            close(lg[i], own.prefill(said[s].cuda()), f"sequence {s} of {seqs}")
            assert nxt[i].item() == lg[i].argmax().item()
            own.close()
        assert srv.lens.tolist() == srv.host_lens
        assert nb.take_device_error() == 0

    step([0, 1, 2], [100, 1, 33])
    step([2, 0], [1, 1])
    srv.fork(0, [3, 4])
    said[3], said[4] = said[0], said[0]
    step([0, 1, 2, 3, 4], [1, 1, 1, 1, 1])
    step([4, 1, 3], [1, 130, 1])
    srv.free([0, 2])
    del said[0], said[2]
    srv.compact()
    step([1, 3, 4, 5], [1, 1, 1, 60])
    assert srv.lengths() == [0, len(said[1]), 0, len(said[3]), len(said[4]), len(said[5])]
    used = int((srv.refs > 0).sum())
    assert int(srv.table.max()) < used + 20


def test_serving_refusals(nqlib, model):
    _, dev = model
    dec = LlamaDecoder(cfg(), dev)
    srv = PagedLlama(dec, n_pages=6, page_size=16, max_seqs=3, max_len=64)
    t = lambda n: torch.zeros(n, dtype=torch.int32, device="cuda")  # noqa: E731
    for call in (lambda: srv.step([0, 0], t(2), [1, 1]), lambda: srv.step([3], t(1), [1]),
                 lambda: srv.step([0], t(1), [2]), lambda: srv.step([0], t(1).long(), [1]),
                 lambda: srv.step([0], t(65), [65]), lambda: srv.step([], t(0), []),
                 lambda: srv.step([0], t(0), [0]), lambda: srv.fork(0, [3]),
                 lambda: srv.free([1, 1]), lambda: PagedLlama(dec, 4, page_size=24),
                 lambda: dec.set_prefill_chunk(-1)):
        with pytest.raises(nb.NQError):
            call()
    srv.step([0, 1], t(80), [40, 40])  # six pages
    with pytest.raises(nb.NQError):
        srv.fork(0, [1])
    assert nb.take_device_error() == 0
    srv.step([2], t(16), [16])  # no page left: the device refuses
    assert nb.take_device_error() & 4
    assert srv.lengths() == [40, 40, 0]
    srv.free([0])
    srv.step([2], t(16), [16])
    assert nb.take_device_error() == 0 and srv.lengths() == [0, 40, 16]


def test_a_refused_step_leaves_the_cache(nqlib, model):
    """A step without enough free pages writes no key: all pages, those that sequences
    share among them, hold what they held, and the sequences go on as if it had not been."""
    dec = LlamaDecoder(cfg(), model[1])
    srv = PagedLlama(dec, n_pages=5, page_size=16, max_seqs=3, max_len=200)
    srv.pool.zero_()
    toks = torch.randint(0, SMALL["vocab"], (40,), dtype=torch.int32, device="cuda")
    srv.step([0], toks, [40])
    srv.fork(0, [1])
    before = srv.pool.clone()
    srv.step([0, 1], torch.cat([toks, toks]), [40, 40])  # 3 + 3 pages of 2 free ones
    assert nb.take_device_error() & 4
    assert srv.lengths() == [40, 40, 0]
    assert torch.equal(srv.pool, before)
    a, _ = srv.step([0, 1], toks[:2].contiguous(), [1, 1])
    ref = LlamaDecoder(cfg(), model[1])
    ref.set_prefill_chunk(64)
    for i in range(2):
        ref.reset()
        ref.prefill(toks, logits=False)
        close(a[i], ref.step(toks[i:i + 1])[0], f"sequence {i}")
    assert nb.take_device_error() == 0


def test_forward_refusals(nqlib, model):
    _, dev = model
    dec = LlamaDecoder(cfg(), dev)
    from neurons_b200.paged import Batch, Cache
    z = torch.zeros(1 << 20, dtype=torch.uint8, device="cuda").data_ptr()
    ok = dict(tokens=z, cache=Cache(z, z, 2, 2 * 16 * 128, 2, 16, 128, 1), stride=1 << 14,
              batch=Batch(z, 1, 1, 1, z, None, None, 1, 1), max_q=1, rows=z, n_out=1, logits=z,
              ws=z, ws_bytes=16)

    def call(**kw):
        d = {**ok, **kw}
        return lib().nq_llama_forward(dec.handle, d["tokens"], ctypes.byref(d["cache"]), d["stride"],
                                      ctypes.byref(d["batch"]), d["max_q"], d["rows"], d["n_out"],
                                      d["logits"], None, d["ws"], d["ws_bytes"], None)

    for kw in (dict(), dict(tokens=None), dict(ws=None), dict(rows=None), dict(logits=None),
               dict(max_q=-1), dict(n_out=-1), dict(stride=4), dict(stride=-8),
               dict(cache=Cache(z, z, 2, 4096, 2, 16, 128, 2)),
               dict(cache=Cache(z, z, 2, 4096, 1, 16, 128, 1)),
               dict(cache=Cache(z, z, 2, 4096, 2, 16, 64, 1))):
        assert call(**kw) == 1, kw
    assert call(batch=Batch(z, 1, 1, 1, z, None, None, 0, 0)) == 0


def serve_beside(srv, model, toks):
    """A step of sequence 0 with the token behind toks, held against a decoder that was given
    the same tokens alone."""
    lg, _ = srv.step([0], toks[-1:].contiguous(), [1])
    ref = LlamaDecoder(cfg(), model[1])
    ref.set_prefill_chunk(64)
    close(lg[0], ref.prefill(toks.contiguous()), "the step behind a refused one")
    ref.close()


def test_steps_go_on_behind_a_refused_one(nqlib, model):
    """Nobody asks for the lengths between a refused step and the next one: its tokens still
    stand right behind the last ones that were accepted, in the sequence and in its forks."""
    dec = LlamaDecoder(cfg(), model[1])
    srv = PagedLlama(dec, n_pages=4, page_size=16, max_seqs=4, max_len=64)
    srv.pool.fill_(float("nan"))
    toks = torch.randint(0, SMALL["vocab"], (24,), dtype=torch.int32, device="cuda")
    srv.step([0, 1], torch.cat([toks[:20], toks[:20]]), [20, 20])       # all four pages
    srv.step([0, 2], torch.zeros(18, dtype=torch.int32, device="cuda"), [1, 17])  # refused
    serve_beside(srv, model, toks[:21])
    srv.free([1])
    serve_beside(srv, model, toks[:22])
    srv.step([0, 1], torch.zeros(50, dtype=torch.int32, device="cuda"), [40, 10])  # refused
    srv.fork(0, [2])  # (which the step above left empty, whatever the host thought of it)
    assert nb.take_device_error() == 4
    lg, _ = srv.step([2], toks[22:23].contiguous(), [1])
    serve_beside(srv, model, toks[:23])
    ref = LlamaDecoder(cfg(), model[1])
    ref.set_prefill_chunk(64)
    close(lg[0], ref.prefill(toks[:23].contiguous()), "a fork behind a refused step")
    assert srv.lengths() == [23, 0, 23, 0]
    assert nb.take_device_error() == 0


def test_a_refused_step_does_not_use_up_max_len(nqlib, model):
    """Tokens that were refused count neither against max_len nor as a child's."""
    dec = LlamaDecoder(cfg(), model[1])
    srv = PagedLlama(dec, n_pages=3, page_size=16, max_seqs=3, max_len=64)
    t = lambda n: torch.zeros(n, dtype=torch.int32, device="cuda")  # noqa: E731
    srv.step([0], t(30), [30])
    srv.step([0, 1], t(64), [30, 34])  # 2 + 3 pages of the one that is left
    assert nb.take_device_error() == 4
    srv.step([0], t(10), [10])
    srv.step([0], t(8), [8])
    srv.fork(0, [1])
    assert srv.lengths() == [48, 48, 0]
    with pytest.raises(nb.NQError):
        srv.step([0], t(17), [17])
    with pytest.raises(nb.NQError):
        srv.fork(0, [1])
    assert nb.take_device_error() == 0


def test_a_step_that_cannot_be_made_reserves_nothing(nqlib, model):
    """Outputs that do not fit the GPU's memory: the sequences stay as they were."""
    dec = LlamaDecoder(cfg(), model[1])
    srv = PagedLlama(dec, n_pages=8, page_size=16, max_seqs=2, max_len=64)
    toks = torch.randint(0, SMALL["vocab"], (12,), dtype=torch.int32, device="cuda")
    srv.step([0], toks[:10].contiguous(), [10])
    vocab, dec.vocab = dec.vocab, 1 << 50
    with pytest.raises(RuntimeError):
        srv.step([0], toks[:1].contiguous(), [1])
    dec.vocab = vocab
    assert srv.lens.tolist() == srv.host_lens == [10, 0]
    serve_beside(srv, model, toks[:11])


def test_steps_behind_a_long_chunked_prompt(oracle, nqlib):
    """A step turns its query by the same angles as the chunks turned their keys: at position
    520000 angles in 32 bits are off by up to 0.03, and with scores of tens over as many keys a
    step shows that."""
    far = dict(SMALL, n_layers=1, max_context=520100, rope_theta=100.0)
    _, dev = make_model(oracle, far, 23)
    g = torch.Generator(device="cuda").manual_seed(4)
    for n, rows in (("q", 1024), ("k", 256), ("o", 1024)):
        w = torch.randn(rows, 1024, device="cuda", generator=g) * 0.1
        dev["layers"][0][n] = nb.quantize(w, far["group_size"], far["bits"], nb.SCHEME_MLX_AFFINE)
    n = 520000
    toks = torch.randint(0, far["vocab"], (n + 3,), dtype=torch.int32, device="cuda", generator=g)
    dec = LlamaDecoder(far, dev)
    dec.set_prefill_chunk(8192)
    want = []
    for i in range(3):
        dec.reset()
        want.append(dec.prefill(toks[:n + 1 + i]))
    dec.reset()
    dec.prefill(toks[:n], logits=False)
    for i in range(3):
        close(dec.step(toks[n + i:n + i + 1])[0], want[i], f"step {i}")
    assert nb.take_device_error() == 0


def test_compaction_between_steps(nqlib, model):
    """Right after srv.compact() the used pages are the lowest, and the next steps' logits are
    those of a decoder of each sequence's own."""
    dec = LlamaDecoder(cfg(), model[1])
    srv = PagedLlama(dec, n_pages=40, page_size=16, max_seqs=4, max_len=300)
    toks = torch.randint(0, SMALL["vocab"], (230,), dtype=torch.int32, device="cuda")
    srv.step([0, 1, 2], torch.cat([toks[:200], toks[:50], toks[:120]]), [200, 50, 120])
    srv.fork(2, [3])
    srv.free([0])
    used = int((srv.refs > 0).sum())
    assert int(srv.table.max()) >= used
    srv.compact()
    assert (srv.refs[:used] > 0).all() and (srv.refs[used:] == 0).all()
    assert int(srv.table.max()) == used - 1
    lg, _ = srv.step([1, 2, 3], torch.cat([toks[50:51], toks[120:150], toks[7:8]]), [1, 30, 1])
    ref = LlamaDecoder(cfg(), model[1])
    ref.set_prefill_chunk(300)
    for got, said in zip(lg, (toks[:51], toks[:150], torch.cat([toks[:120], toks[7:8]]))):
        ref.reset()
        close(got, ref.prefill(said.contiguous()), f"{said.numel()} tokens")
    assert nb.take_device_error() == 0


@pytest.mark.parametrize("heads,kv,dim", [(16, 4, 64), (16, 2, 64), (4, 2, 256)])
def test_other_head_dims(oracle, nqlib, heads, kv, dim):
    """Chunks, steps behind them and paged serving with heads of 64 and 256 dims."""
    from oracle.llama_oracle import LlamaOracle
    c = dict(SMALL, n_heads=heads, n_kv_heads=kv, head_dim=dim, max_context=200)
    host, dev = make_model(oracle, c, dim)
    dec, ora = LlamaDecoder(c, dev), LlamaOracle(c, host)
    toks = np.random.default_rng(6).integers(0, c["vocab"], 41).astype(np.int32)
    td = torch.from_numpy(toks).cuda()
    refs = [ora.step(int(t))[0] for t in toks]
    dec.set_prefill_chunk(24)
    check_logits(oracle, dec.prefill(td[:40].contiguous()), refs[39], "chunks")
    check_logits(oracle, dec.step(td[40:])[0], refs[40], "step")
    srv = PagedLlama(dec, n_pages=10, page_size=16, max_seqs=2, max_len=64)
    lg, _ = srv.step([0, 1], torch.cat([td[:40], td[:3]]), [40, 3])
    check_logits(oracle, lg[0], refs[39], "paged prompt")
    check_logits(oracle, lg[1], refs[2], "short paged prompt")
    lg, _ = srv.step([0, 1], torch.cat([td[40:], td[3:4]]), [1, 1])
    check_logits(oracle, lg[0], refs[40], "paged step")
    check_logits(oracle, lg[1], refs[3], "short paged step")
    assert nb.take_device_error() == 0
