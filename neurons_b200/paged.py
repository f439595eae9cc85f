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

from ._lib import NQError, check, lib

P, I64, I = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int

_DTYPES = {torch.bfloat16: 1, torch.float16: 2}


class _Cache(ctypes.Structure):
    _fields_ = [("k", P), ("v", P), ("n_pages", I64), ("page_stride", I64), ("n_kv_heads", I),
                ("page_size", I), ("head_dim", I), ("dtype", I)]


class _Batch(ctypes.Structure):
    _fields_ = [("table", P), ("table_ld", I64), ("table_width", I64), ("n_rows", I64),
                ("kv_lens", P), ("seqs", P), ("q_starts", P), ("n_seqs", I64), ("n_tokens", I64)]


class _Table(ctypes.Structure):
    _fields_ = [("refs", P), ("table", P), ("lens", P), ("n_pages", I64), ("n_rows", I64),
                ("table_ld", I64), ("table_width", I64), ("page_size", I)]


class _Pool(ctypes.Structure):
    _fields_ = [("data", P), ("outer", I64), ("n_pages", I64), ("page_bytes", I64)]


# the stream's handle without an object around it (a torch.cuda.Stream costs more than
# a small kernel)
_raw_stream = torch._C._cuda_getCurrentRawStream
_device = torch.cuda.current_device
_INT32 = torch.int32


def _index(t, name, device, dim=1):
    """An int32 index tensor on `device`, its last axis contiguous."""
    st = t.stride()
    if t.dtype is not _INT32 or len(st) != dim or t.get_device() != device or \
            (st[-1] != 1 and t.numel() > 1):
        raise NQError(1, f"{name} must be a contiguous int32 tensor with {dim} axes on the cache's "
                         "device")
    return t.data_ptr()


def _rows(t, name, heads, dim, dtype, device):
    """Rows [tokens, heads, dim] whose heads lie one after another: address, distance."""
    shape, st = t.shape, t.stride()
    if t.dtype is not dtype or len(shape) != 3 or t.get_device() != device:
        raise NQError(1, f"{name} must be [tokens, heads, head dim], of the cache's type and on its "
                         "device")
    if shape[2] != dim or (heads is not None and shape[1] != heads):
        raise NQError(1, f"{name} has shape {tuple(shape)}, expected [tokens, "
                         f"{heads if heads is not None else 'heads'}, {dim}]")
    if st[2] != 1 or (st[1] != dim and shape[1] > 1):
        raise NQError(1, f"{name}: the heads of a token must lie one after another")
    return t.data_ptr(), st[0] if shape[0] > 1 else shape[1] * dim


def _cache(k, v):
    """The cache's structure, heads, head dim, page size and device."""
    shape, st, device = k.shape, k.stride(), k.get_device()
    dtype = _DTYPES.get(k.dtype)
    if dtype is None or len(shape) != 4 or device < 0:
        raise NQError(1, "k_pages must be a bf16 or fp16 CUDA tensor "
                         "[pages, kv heads, page size, head dim]")
    if v.dtype is not k.dtype or v.shape != shape or v.stride() != st or v.get_device() != device:
        raise NQError(1, "v_pages must match k_pages in type, shape, strides and device")
    n, heads, size, dim = shape
    if (st[3] != 1 or st[2] != dim or (st[1] != size * dim and heads > 1)) and k.numel() > 0:
        raise NQError(1, "a page must be contiguous")
    if device != _device():
        raise NQError(1, "the cache is not on the current device")
    return (_Cache(k.data_ptr(), v.data_ptr(), n, st[0] if n > 1 else heads * size * dim, heads,
                   size, dim, dtype), heads, dim, size, device)


def _batch(table, kv_lens, seqs, q_starts, tokens, device):
    tp, lp = _index(table, "table", device, 2), _index(kv_lens, "kv_lens", device)
    rows, width = table.shape
    if kv_lens.shape[0] != rows:
        raise NQError(1, f"kv_lens has {kv_lens.shape[0]} entries for {rows} table rows")
    sp = qp = None
    if seqs is not None:
        sp, n = _index(seqs, "seqs", device), seqs.shape[0]
        if q_starts is not None and q_starts.shape[0] != n + 1:
            raise NQError(1, f"q_starts must have {n + 1} entries")
    elif q_starts is not None:
        n = q_starts.shape[0] - 1
    else:
        n = min(rows, tokens)
    if q_starts is not None:
        qp = _index(q_starts, "q_starts", device)
    return _Batch(tp, table.stride(0) if rows > 1 else width, width, rows, lp, sp, qp, n, tokens)


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
    c, kv_heads, dim, size, device = _cache(k_pages, v_pages)
    dtype = k_pages.dtype
    qp, q_ld = _rows(q, "q", None, dim, dtype, device)
    tokens, heads, _ = q.shape
    b = _batch(table, kv_lens, seqs, q_starts, tokens, device)
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        op, out_ld = out.data_ptr(), heads * dim
    elif out.shape != q.shape:
        raise NQError(1, "out must have q's shape")
    else:
        op, out_ld = _rows(out, "out", heads, dim, dtype, device)
    if q_starts is None:
        max_q = 1
    elif max_q is None:
        max_q = tokens
    f = lib()
    if workspace is None:
        n = f.nq_paged_attention_workspace_size(heads, kv_heads, dim, max_q, table.shape[1] * size)
        if n > 0:
            workspace = q.new_empty(n, dtype=torch.uint8)
        wp = workspace.data_ptr() if n > 0 else None
    elif workspace.get_device() != device or not workspace.is_contiguous():
        raise NQError(1, "workspace must be contiguous, on the cache's device")
    else:
        wp, n = workspace.data_ptr(), workspace.numel() * workspace.element_size()
    check(f.nq_paged_attention(qp, q_ld, heads, ctypes.byref(c), ctypes.byref(b), max_q,
                               scale if scale is not None else dim ** -0.5, window, wp, n, op,
                               out_ld, _raw_stream(device)))
    return out


def paged_append(q, k, v, k_pages, v_pages, table, kv_lens, q_starts=None, freqs=None, seqs=None,
                 q_out=None):
    """Turns the new tokens' queries and keys by their positions (freqs: fp32, radians per
    position of each pair of dims; None: no turn) and stores keys and values in their pages.
    Returns the queries: in q_out (may be q), or a new tensor."""
    c, kv_heads, dim, _, device = _cache(k_pages, v_pages)
    dtype = k_pages.dtype
    qp, q_ld = _rows(q, "q", None, dim, dtype, device)
    tokens, heads, _ = q.shape
    kp, k_ld = _rows(k, "k", kv_heads, dim, dtype, device)
    vp, v_ld = _rows(v, "v", kv_heads, dim, dtype, device)
    if k.shape[0] != tokens or v.shape[0] != tokens:
        raise NQError(1, "q, k and v differ in tokens")
    b = _batch(table, kv_lens, seqs, q_starts, tokens, device)
    if q_out is None:
        q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
    elif q_out.shape != q.shape:
        raise NQError(1, "q_out must have q's shape")
    op, out_ld = _rows(q_out, "q_out", heads, dim, dtype, device)
    fp, nf = None, 0
    if freqs is not None:
        if freqs.dtype is not torch.float32 or freqs.dim() != 1 or \
                freqs.get_device() != device or not freqs.is_contiguous():
            raise NQError(1, "freqs must be a contiguous fp32 vector on the cache's device")
        fp, nf = freqs.data_ptr(), freqs.shape[0]
    check(lib().nq_paged_append(qp, q_ld, kp, k_ld, vp, v_ld, heads, ctypes.byref(c),
                                ctypes.byref(b), fp, nf, op, out_ld, _raw_stream(device)))
    return q_out


def _table(refs, table, lens, page_size):
    device = refs.get_device()
    if device < 0 or device != _device():
        raise NQError(1, "refs must be a CUDA tensor on the current device")
    rp, tp = _index(refs, "refs", device), _index(table, "table", device, 2)
    rows, width = table.shape
    lp = rp
    if lens is not None:
        lp = _index(lens, "lens", device)
        if lens.shape[0] != rows:
            raise NQError(1, f"lens has {lens.shape[0]} entries for {rows} table rows")
    return _Table(rp, tp, lp, refs.shape[0], rows, table.stride(0) if rows > 1 else width, width,
                  page_size), device


def _pool(pool, device):
    shape = pool.shape
    if pool.get_device() != device or len(shape) < 4 or not pool.is_contiguous():
        raise NQError(1, "pool must be a contiguous CUDA tensor [..., pages, kv heads, page size, "
                         "head dim] on the current device")
    n, page = shape[-4], shape[-3] * shape[-2] * shape[-1]
    if pool.numel() == 0:
        raise NQError(1, "the pool is empty")
    return _Pool(pool.data_ptr(), pool.numel() // (n * page), n, page * pool.element_size())


def _list(t, name, n, device):
    p = _index(t, name, device)
    if t.shape[0] != n:
        raise NQError(1, f"{name} must have {n} entries")
    return p


def _workspace(ws, need, like):
    if ws is None:
        ws = like.new_empty(need, dtype=torch.uint8)
    elif ws.device != like.device or not ws.is_contiguous():
        raise NQError(1, "workspace must be contiguous, on the pool's device")
    return ws.data_ptr(), ws.numel() * ws.element_size(), ws


def pages_free(refs, table, lens, seqs):
    """The sequences give their pages back: one holder less each, length 0."""
    t, device = _table(refs, table, lens, 1)
    check(lib().nq_pages_free(ctypes.byref(t), _index(seqs, "seqs", device), seqs.shape[0],
                              _raw_stream(device)))


def pages_fork(refs, table, lens, parents, children):
    """children[i] (empty so far) becomes a copy of parents[i] that shares its pages."""
    t, device = _table(refs, table, lens, 1)
    n = parents.shape[0]
    check(lib().nq_pages_fork(ctypes.byref(t), _index(parents, "parents", device),
                              _list(children, "children", n, device), n, _raw_stream(device)))


def pages_workspace_size(n_pages, n):
    """Bytes that pages_reserve (n sequences) and pages_compact (n_pages pages) need."""
    return int(lib().nq_pages_workspace_size(n_pages, n))


def pages_reserve(pool, refs, table, lens, seqs, new_lens, workspace=None):
    """The sequences grow to new_lens tokens: shared last pages that are not full are
    copied, free pages added.  All or nothing (see include/nq.h)."""
    t, device = _table(refs, table, lens, pool.shape[-2])
    p = _pool(pool, device)
    n = seqs.shape[0]
    f = lib()
    wp, wn, keep = _workspace(workspace, f.nq_pages_workspace_size(0, n), pool)
    check(f.nq_pages_reserve(ctypes.byref(t), ctypes.byref(p), _index(seqs, "seqs", device),
                             _list(new_lens, "new_lens", n, device), n, wp, wn,
                             _raw_stream(device)))


def pages_compact(pool, refs, table, workspace=None):
    """The used pages move to the pool's low end; refs and table follow."""
    t, device = _table(refs, table, None, pool.shape[-2])
    p = _pool(pool, device)
    f = lib()
    wp, wn, keep = _workspace(workspace, f.nq_pages_workspace_size(t.n_pages, 0), pool)
    check(f.nq_pages_compact(ctypes.byref(t), ctypes.byref(p), wp, wn, _raw_stream(device)))


def copy_pages(pool, src, dst):
    """Copies page src[i] to dst[i] in every layer; a target may not also be a source or
    an earlier target (that move is refused)."""
    device = _device()
    p = _pool(pool, device)
    n = src.shape[0]
    check(lib().nq_pages_copy(ctypes.byref(p), _index(src, "src", device),
                              _list(dst, "dst", n, device), n, _raw_stream(device)))
