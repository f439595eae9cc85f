"""Llama decode step on the GPU (libnq.so, nq_llama_*): the quantized
matmuls of the reference's LlamaModel decode function
(compute/src/compute/model/llama_model.cpp:355-509) with RMSNorm, RoPE, GQA
attention over a KV cache and greedy argmax around them, and its pipelined
generation (:713-812) as back-to-back steps that feed each other's token on
the device.

    dec = LlamaDecoder(cfg, weights)      # weights: torch CUDA tensors
    dec.set_prefill_chunk(512)            # the prompt in chunks (default: by the step)
    dec.prefill(prompt_ids)               # int32 CUDA tensor
    ids = dec.generate(64)                # int32 CUDA tensor of 64 tokens

PagedLlama serves many sequences with the same weights over one page pool:

    srv = PagedLlama(dec, n_pages=4096, page_size=64, max_seqs=64, max_len=8192)
    logits, tok = srv.step([0, 1], prompts, [len0, len1])   # chunks of any lengths
    logits, tok = srv.step([0, 1], tok, [1, 1])             # one token each
    srv.fork(0, [2, 3]); srv.free([1]); srv.compact()
"""
import ctypes

import torch

from . import ops, paged
from ._lib import NQError, check, lib

P = ctypes.c_void_p


class QWeight(ctypes.Structure):
    _fields_ = [("w", P), ("scales", P), ("biases", P)]


class LlamaConfig(ctypes.Structure):
    _fields_ = [("n_layers", ctypes.c_int), ("hidden", ctypes.c_int), ("n_heads", ctypes.c_int),
                ("n_kv_heads", ctypes.c_int), ("head_dim", ctypes.c_int),
                ("intermediate", ctypes.c_int), ("vocab", ctypes.c_int), ("bits", ctypes.c_int),
                ("group_size", ctypes.c_int), ("max_context", ctypes.c_int),
                ("rms_eps", ctypes.c_float), ("rope_theta", ctypes.c_float)]


class LlamaLayer(ctypes.Structure):
    _fields_ = [("input_norm", P), ("post_norm", P)] + [
        (n, QWeight) for n in ("q", "k", "v", "o", "gate", "up", "down")]


CONFIG_KEYS = [f for f, _ in LlamaConfig._fields_]
PROJ = ("q", "k", "v", "o", "gate", "up", "down")


def _qw(t):
    if t is None:
        return QWeight(None, None, None)
    w, s, b = t
    return QWeight(P(w.data_ptr()), P(s.data_ptr()) if s is not None else None,
                   P(b.data_ptr()) if b is not None else None)


class LlamaDecoder:
    """cfg: dict with the LlamaConfig fields.  weights: dict with 'embed'
    (wq, scales, biases), 'final_norm' (bf16), optional 'lm_head' (wq, s, b) and
    'layers': a list of dicts with 'input_norm', 'post_norm' and the seven
    projections as (wq, scales, biases), all CUDA tensors (kept referenced)."""

    def __init__(self, cfg, weights):
        self.cfg = dict(cfg)
        self._keep = weights
        c = LlamaConfig(**{k: self.cfg[k] for k in CONFIG_KEYS})
        layers = (LlamaLayer * cfg["n_layers"])()
        for i, L in enumerate(weights["layers"]):
            layers[i].input_norm = P(L["input_norm"].data_ptr())
            layers[i].post_norm = P(L["post_norm"].data_ptr())
            for n in PROJ:
                setattr(layers[i], n, _qw(L[n]))
        embed = _qw(weights["embed"])
        head = _qw(weights.get("lm_head"))
        self.handle = P()
        check(lib().nq_llama_create(ctypes.byref(self.handle), ctypes.byref(c), layers,
                                    P(weights["final_norm"].data_ptr()), ctypes.byref(embed),
                                    ctypes.byref(head) if head.w else None))
        self.vocab = cfg["vocab"]

    def close(self):
        if self.handle:
            lib().nq_llama_destroy(self.handle)
            self.handle = P()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    @property
    def position(self):
        return int(lib().nq_llama_position(self.handle))

    def set_prefill_chunk(self, chunk):
        """Prompts in chunks of up to `chunk` tokens (0: one position per step).  Before a
        sequence's first token: from here on steps take their angles in 64 bits, as chunks do."""
        check(lib().nq_llama_set_prefill_chunk(self.handle, int(chunk)))

    def reset(self):
        check(lib().nq_llama_reset(self.handle, ops._stream()))

    def step(self, token=None, logits=True):
        """One step on `token` (int32 CUDA tensor of 1; None: the last argmax).
        Returns (logits fp32 [vocab] or None, next token int32 [1])."""
        lg = torch.empty(self.vocab, dtype=torch.float32, device="cuda") if logits else None
        nxt = torch.empty(1, dtype=torch.int32, device="cuda")
        check(lib().nq_llama_step(self.handle, P(token.data_ptr()) if token is not None else None,
                                  P(lg.data_ptr()) if lg is not None else None,
                                  P(nxt.data_ptr()), ops._stream()))
        return lg, nxt

    def prefill(self, tokens, logits=True):
        """The prompt (int32 CUDA tensor) through the decoder, one position per
        step or in chunks (set_prefill_chunk); returns the last position's logits
        (fp32) or None."""
        if tokens.dtype != torch.int32 or not tokens.is_cuda:
            raise NQError(1, "prefill: tokens must be an int32 CUDA tensor")
        lg = torch.empty(self.vocab, dtype=torch.float32, device="cuda") if logits else None
        check(lib().nq_llama_prefill(self.handle, P(tokens.data_ptr()), tokens.numel(),
                                     P(lg.data_ptr()) if lg is not None else None,
                                     ops._stream()))
        return lg

    def generate(self, n, token=None, out=None):
        """n greedy steps, pipelined on the device; returns the n tokens."""
        out = out if out is not None else torch.empty(n, dtype=torch.int32, device="cuda")
        check(lib().nq_llama_generate(self.handle,
                                      P(token.data_ptr()) if token is not None else None, n,
                                      P(out.data_ptr()), ops._stream()))
        return out


class PagedLlama:
    """Continuous batching over a LlamaDecoder's weights: sequences 0 .. max_seqs - 1 of up
    to max_len tokens in a pool of n_pages pages.  The page table, lengths and
    reference counts live on the device, where a step takes the lengths from.  A refused
    step leaves the host's own lengths too large until lengths() is called, which a call
    that they would refuse does first."""

    def __init__(self, decoder, n_pages, page_size=64, max_seqs=64, max_len=4096):
        c = decoder.cfg
        if n_pages <= 0 or page_size <= 0 or page_size % 16 or max_seqs <= 0 or max_len <= 0:
            raise NQError(1, "PagedLlama: sizes must be positive, page_size a multiple of 16")
        self.decoder, self.max_len = decoder, max_len
        self.pool = torch.empty((c["n_layers"], 2, n_pages, c["n_kv_heads"], page_size,
                                 c["head_dim"]), dtype=torch.bfloat16, device="cuda")
        width = -(-max_len // page_size)
        self.refs = torch.zeros(n_pages, dtype=torch.int32, device="cuda")
        self.table = torch.full((max_seqs, width), -1, dtype=torch.int32, device="cuda")
        self.lens = torch.zeros(max_seqs, dtype=torch.int32, device="cuda")
        self.host_lens = [0] * max_seqs

    def _ids(self, x):
        return torch.tensor(x, dtype=torch.int32, device="cuda")

    def _check(self, seqs):
        if any(s < 0 or s >= len(self.host_lens) for s in seqs) or len(set(seqs)) < len(seqs):
            raise NQError(1, f"sequences must be different numbers below {len(self.host_lens)}")

    def _holds(self, test):
        """test() by the host's lengths, or else by the device's."""
        if test():
            return True
        self.lengths()
        return test()

    def step(self, seqs, tokens, news, logits=True):
        """news[i] new tokens of sequence seqs[i], one sequence after another in `tokens`
        (int32 CUDA tensor).  Returns the last positions' logits (fp32 [n, vocab], or None)
        and argmax (int32 [n]).  Too few free pages leave the sequences as they were and
        raise bit 2 of take_device_error(); the step's outputs mean nothing then, the next
        step goes on behind the tokens that were accepted, and lengths() tells the
        sequences' lengths."""
        self._check(seqs)
        n, total = len(seqs), sum(news)
        if len(news) != n or n == 0 or min(news) < 1 or tokens.dtype != torch.int32 or \
                not tokens.is_cuda or not tokens.is_contiguous() or tokens.numel() != total:
            raise NQError(1, "step: tokens must be int32 CUDA, news[i] >= 1 of them for each sequence")
        if not self._holds(lambda: all(self.host_lens[s] + m <= self.max_len
                                       for s, m in zip(seqs, news))):
            raise NQError(1, f"step: a sequence would pass max_len {self.max_len}")
        # Everything that can fail on the host comes before the reserve: a sequence that has
        # grown and whose tokens are not appended would keep a hole.
        d, pool, table = self.decoder, self.pool, self.table
        lg = torch.empty((n, d.vocab), dtype=torch.float32, device="cuda") if logits else None
        nxt = torch.empty(n, dtype=torch.int32, device="cuda")
        most = max(news)
        f = lib()
        need = f.nq_llama_forward_workspace_size(d.handle, total, n, most,
                                                 table.shape[1] * pool.shape[-2])
        ws = torch.empty(need, dtype=torch.uint8, device="cuda")
        starts = [0]
        for m in news:
            starts.append(starts[-1] + m)
        meta = self._ids(list(seqs) + list(news) + starts + [e - 1 for e in starts[1:]])
        ids, more, q_starts, rows = meta.split([n, n, n + 1, n])
        lens = self.lens.index_select(0, ids) + more
        paged.pages_reserve(pool, self.refs, table, self.lens, ids, lens)
        for s, m in zip(seqs, news):
            self.host_lens[s] += m
        # (refused: the sequences have their old lengths, and the new tokens would be
        # written over their last ones; they are padding then)
        ids = torch.where(self.lens.index_select(0, ids) == lens, ids, -1)
        cache = paged.Cache(pool.data_ptr(), pool[0, 1].data_ptr(), pool.shape[2], pool.stride(2),
                            *pool.shape[3:], 1)
        batch = paged.Batch(table.data_ptr(), table.shape[1], table.shape[1], table.shape[0],
                            self.lens.data_ptr(), ids.data_ptr(), q_starts.data_ptr(), n, total)
        check(f.nq_llama_forward(d.handle, tokens.data_ptr(), ctypes.byref(cache),
                                 pool.stride(0), ctypes.byref(batch), most, rows.data_ptr(), n,
                                 lg.data_ptr() if logits else None, nxt.data_ptr(), ws.data_ptr(),
                                 need, ops._stream()))
        return lg, nxt

    def fork(self, parent, children):
        """children (empty so far) continue from parent's tokens, sharing its pages."""
        self._check([parent] + list(children))
        if not self._holds(lambda: not any(self.host_lens[c] for c in children)):
            raise NQError(1, "fork: a child has tokens")
        paged.pages_fork(self.refs, self.table, self.lens, self._ids([parent] * len(children)),
                         self._ids(list(children)))
        for c in children:
            self.host_lens[c] = self.host_lens[parent]

    def free(self, seqs):
        self._check(seqs)
        paged.pages_free(self.refs, self.table, self.lens, self._ids(list(seqs)))
        for s in seqs:
            self.host_lens[s] = 0

    def compact(self):
        """The used pages move to the pool's low end."""
        paged.pages_compact(self.pool, self.refs, self.table)

    def lengths(self):
        """The lengths as the device has them (waits for it); the host's follow."""
        self.host_lens = self.lens.tolist()
        return list(self.host_lens)
