"""The key/value cache in pages, over the C ABI (nq_paged_*, nq_pages_*).

    paged_append(q, k, v, k_pages, v_pages, table, kv_lens, ...)   rotary positions, store
    paged_attention(q, k_pages, v_pages, table, kv_lens, ...)      attention of new tokens
    pages_reserve / pages_fork / pages_free / pages_compact        the page pool
    copy_pages(pool, src, dst)

A pool is a tensor [layers, 2, pages, kv heads, page size, head dim] (bf16 or
fp16); layer l's keys are pool[l, 0] and its values pool[l, 1].  table
[rows, width] (int32, -1: no page) lists the pages of each sequence, kv_lens
[rows] their lengths, new tokens included, refs [pages] how many sequences hold
a page.  A step's batch is its sequences' new tokens one after another: those
of entry b are rows q_starts[b] .. q_starts[b + 1] (one each without q_starts),
its table row seqs[b] (b without seqs; negative: padding).

Every call is asynchronous on torch's current stream, reads its index tensors
on the device only, and may be captured in a CUDA graph.  Arguments that can
be seen to be wrong raise NQError; what the index tensors say wrong raises bits
of take_device_error() (include/nq.h).
"""
import ctypes

import torch

from ._lib import lib

P, I64, I = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int


class Cache(ctypes.Structure):
    """nq_paged_cache_t"""
    _fields_ = [("k", P), ("v", P), ("n_pages", I64), ("page_stride", I64), ("n_kv_heads", I),
                ("page_size", I), ("head_dim", I), ("dtype", I)]


class Batch(ctypes.Structure):
    """nq_paged_batch_t"""
    _fields_ = [("table", P), ("table_ld", I64), ("table_width", I64), ("n_rows", I64),
                ("kv_lens", P), ("seqs", P), ("q_starts", P), ("n_seqs", I64), ("n_tokens", I64)]


class PageTable(ctypes.Structure):
    """nq_page_table_t"""
    _fields_ = [("refs", P), ("table", P), ("lens", P), ("n_pages", I64), ("n_rows", I64),
                ("table_ld", I64), ("table_width", I64), ("page_size", I)]


class PagePool(ctypes.Structure):
    """nq_page_pool_t"""
    _fields_ = [("data", P), ("outer", I64), ("n_pages", I64), ("page_bytes", I64)]


_module = None


def _native():
    """The torch binding (binding/paged_torch.cpp), which checks the arguments."""
    global _module
    if _module is None:
        lib()
        try:
            from . import _paged
        except ImportError as e:
            raise ImportError("neurons_b200: _paged.so is missing or does not fit the installed "
                              "torch -- build it with `python -m neurons_b200.build --force`") from e
        _module = _paged
    return _module


def rope_frequencies(dims, base=10000.0, device="cuda"):
    """base^(-2 i / dims) for i < dims / 2 (radians per position), fp32: the `freqs` of
    paged_append for a plain rotary embedding over the first `dims` dims of a head."""
    f = [float(base) ** (-2.0 * i / dims) for i in range(dims // 2)]
    return torch.tensor(f, dtype=torch.float64).to(torch.float32).to(device)


def paged_attention_workspace_size(n_heads, n_kv_heads, head_dim, max_q, max_keys):
    """Bytes of a paged_attention call; max_keys: the table's width times the page size."""
    return int(lib().nq_paged_attention_workspace_size(n_heads, n_kv_heads, head_dim, max_q,
                                                       max_keys))


def paged_attention(q, k_pages, v_pages, table, kv_lens, q_starts=None, max_q=None, window=0,
                    scale=None, seqs=None, out=None, workspace=None):
    """Attention of the new tokens q [tokens, heads, head dim] over their sequences' pages;
    token t of an entry's n stands at position kv_len - n + t and sees the keys up to it
    (and only the last `window` of them when window > 0).  scale: 1 / sqrt(head dim)
    unless given.  max_q: the longest entry's number of new tokens (the kernel is chosen
    by it; without it, the number of rows).  out: as q, or a new tensor."""
    return (_module or _native()).attention(q, k_pages, v_pages, table, kv_lens, q_starts, max_q,
                                            window, scale, seqs, out, workspace)


def paged_append(q, k, v, k_pages, v_pages, table, kv_lens, q_starts=None, freqs=None, seqs=None,
                 q_out=None):
    """Turns the new tokens' queries and keys by their positions (freqs: fp32, radians per
    position of each pair of dims; None: no turn) and stores keys and values in their pages.
    Returns the queries: in q_out (may be q), or a new tensor."""
    return (_module or _native()).append(q, k, v, k_pages, v_pages, table, kv_lens, q_starts, freqs,
                                         seqs, q_out)


def pages_free(refs, table, lens, seqs):
    """The sequences give their pages back: one holder less each, length 0."""
    (_module or _native()).free(refs, table, lens, seqs)


def pages_fork(refs, table, lens, parents, children):
    """children[i] (empty so far) becomes a copy of parents[i] that shares its pages."""
    (_module or _native()).fork(refs, table, lens, parents, children)


def pages_workspace_size(n_pages, n):
    """Bytes that pages_reserve (n sequences) and pages_compact (n_pages pages) need."""
    return int(lib().nq_pages_workspace_size(n_pages, n))


def pages_reserve(pool, refs, table, lens, seqs, new_lens, workspace=None):
    """The sequences grow to new_lens tokens: shared last pages that are not full are
    copied, free pages added.  All or nothing; after a refusal lens is as it was, and an
    append of the new tokens must leave these sequences out (see include/nq.h)."""
    (_module or _native()).reserve(pool, refs, table, lens, seqs, new_lens, workspace)


def pages_compact(pool, refs, table, workspace=None):
    """The used pages move to the pool's low end; refs and table follow."""
    (_module or _native()).compact(pool, refs, table, workspace)


def copy_pages(pool, src, dst):
    """Copies page src[i] to dst[i] in every layer; a target may not also be a source or
    an earlier target (that move is refused)."""
    (_module or _native()).copy(pool, src, dst)
