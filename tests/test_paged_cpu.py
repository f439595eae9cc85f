"""Refusals of the paged cache's C entry points: bad arguments return InvalidInput with a
message before a device is touched."""
import ctypes
import os
import subprocess

import pytest

from neurons_b200.paged import Batch, Cache, PagePool, PageTable

A = 1 << 20  # an aligned address that validation never reads


def cache(**kw):
    d = dict(k=A, v=A, n_pages=8, page_stride=2 * 16 * 64, n_kv_heads=2, page_size=16, head_dim=64,
             dtype=1)
    d.update(kw)
    return Cache(**d)


def batch(**kw):
    d = dict(table=A, table_ld=4, table_width=4, n_rows=2, kv_lens=A, seqs=None, q_starts=A,
             n_seqs=2, n_tokens=6)
    d.update(kw)
    return Batch(**d)


def attend(lib, c=None, b=None, heads=4, q=A, q_ld=256, max_q=4, scale=0.1, window=0, ws=A,
           ws_bytes=1 << 40, out=A, out_ld=256):
    c, b = c or cache(), b or batch()
    return lib.nq_paged_attention(q, q_ld, heads, ctypes.byref(c), ctypes.byref(b), max_q, scale,
                                  window, ws, ws_bytes, out, out_ld, None)


def append(lib, c=None, b=None, heads=4, q=A, k=A, v=A, ld=512, freqs=A, n=32, out=A):
    c, b = c or cache(), b or batch()
    return lib.nq_paged_append(q, ld, k, ld, v, ld, heads, ctypes.byref(c), ctypes.byref(b), freqs, n,
                               out, ld, None)


BAD_CACHES = [dict(head_dim=96), dict(dtype=0), dict(page_size=8), dict(page_size=0),
              dict(n_kv_heads=0), dict(n_kv_heads=3), dict(n_pages=-1), dict(n_pages=0),
              dict(k=None), dict(v=None), dict(k=A + 8), dict(v=A + 2), dict(page_stride=100),
              dict(page_stride=2 * 16 * 64 + 4)]
BAD_BATCHES = [dict(table=None), dict(kv_lens=None), dict(n_seqs=-1), dict(n_tokens=-1),
               dict(n_rows=0), dict(table_width=0), dict(table_ld=3),
               dict(table_width=1 << 28, table_ld=1 << 28), dict(n_seqs=3),
               dict(q_starts=None, n_seqs=2, n_tokens=1)]


@pytest.mark.parametrize("call", [attend, append])
@pytest.mark.parametrize("bad", BAD_CACHES)
def test_bad_caches_are_refused(nqlib, call, bad):
    assert call(nqlib, c=cache(**bad)) == 1
    assert nqlib.nq_last_error()


@pytest.mark.parametrize("call", [attend, append])
@pytest.mark.parametrize("bad", BAD_BATCHES)
def test_bad_batches_are_refused(nqlib, call, bad):
    assert call(nqlib, b=batch(**bad)) == 1
    assert nqlib.nq_last_error()


@pytest.mark.parametrize("bad", [dict(heads=0), dict(heads=5), dict(scale=0.0), dict(scale=-1.0),
                                 dict(scale=float("nan")), dict(scale=float("inf")),
                                 dict(window=-1), dict(max_q=-1), dict(q=None), dict(out=None),
                                 dict(q=A + 4), dict(out=A + 8), dict(q_ld=255), dict(q_ld=260),
                                 dict(out_ld=128)])
def test_bad_attention_arguments_are_refused(nqlib, bad):
    assert attend(nqlib, **bad) == 1
    assert nqlib.nq_last_error()


@pytest.mark.parametrize("bad", [dict(q=None), dict(k=None), dict(v=None), dict(out=None),
                                 dict(k=A + 4), dict(ld=516), dict(ld=64), dict(n=33), dict(n=40),
                                 dict(n=-8), dict(freqs=None)])
def test_bad_append_arguments_are_refused(nqlib, bad):
    assert append(nqlib, **bad) == 1
    assert nqlib.nq_last_error()


def test_null_structures_are_refused(nqlib):
    c, b = cache(), batch()
    assert nqlib.nq_paged_attention(A, 256, 4, None, ctypes.byref(b), 4, 0.1, 0, A, 1 << 40, A, 256,
                                    None) == 1
    assert nqlib.nq_paged_attention(A, 256, 4, ctypes.byref(c), None, 4, 0.1, 0, A, 1 << 40, A, 256,
                                    None) == 1
    assert nqlib.nq_paged_append(A, 512, A, 512, A, 512, 4, None, None, None, 0, A, 512, None) == 1


def test_empty_batches_are_no_ops(nqlib):
    for b in (batch(n_seqs=0), batch(n_tokens=0)):
        assert attend(nqlib, b=b, q=None, out=None, ws=None) == 0
        assert append(nqlib, b=b, q=None, k=None, v=None, out=None) == 0


def test_workspace_size_of_bad_shapes_is_zero(nqlib):
    size = nqlib.nq_paged_attention_workspace_size
    assert size(5, 2, 64, 1, 4096) == size(4, 2, 80, 1, 4096) == size(4, 2, 64, -1, 4096) == 0
    assert size(4, 2, 64, 1, 64) == 0  # short tables need none
    assert size(4, 2, 64, 1, 4096) > 0
    assert nqlib.nq_pages_workspace_size(-1, 0) == 0
    assert nqlib.nq_pages_workspace_size(0, 0) > 0


def test_workspace_size_without_a_known_max_q_is_the_largest(nqlib):
    size = nqlib.nq_paged_attention_workspace_size
    for heads, kv_heads, keys in ((32, 8, 8192), (4, 2, 1024), (64, 1, 512), (8, 8, 16)):
        most = max(size(heads, kv_heads, 128, q, keys) for q in (1, 2, 4, 16, 17, 129, 4096))
        assert size(heads, kv_heads, 128, 0, keys) == most
        assert size(heads, kv_heads, 128, 1 << 62, keys) == size(heads, kv_heads, 128, 4096, keys)


@pytest.mark.parametrize("heads,kv_heads,dim", [(32, 8, 128), (4, 2, 64), (64, 1, 256), (8, 8, 128),
                                                (16, 1, 64), (128, 1, 128)])
@pytest.mark.parametrize("keys", [16, 256, 272, 1024, 1280, 1296, 1 << 20])
def test_a_workspace_serves_every_smaller_max_q(nqlib, heads, kv_heads, dim, keys):
    """max_q is a bound: a workspace of its size fits calls with fewer new tokens, those
    without q_starts (one token each) among them."""
    size = nqlib.nq_paged_attention_workspace_size
    qs = [1, 2, 3, 4, 8, 15, 16, 17, 64, 300, 4096]
    sizes = [size(heads, kv_heads, dim, q, keys) for q in qs]
    assert sizes == sorted(sizes) and sizes[-1] == size(heads, kv_heads, dim, 0, keys)


def table(**kw):
    d = dict(refs=A, table=A, lens=A, n_pages=8, n_rows=4, table_ld=4, table_width=4, page_size=16)
    d.update(kw)
    return PageTable(**d)


def pool(**kw):
    d = dict(data=A, outer=2, n_pages=8, page_bytes=64)
    d.update(kw)
    return PagePool(**d)


BAD_TABLES = [dict(refs=None), dict(table=None), dict(lens=None), dict(n_pages=0), dict(n_rows=0),
              dict(n_rows=1 << 40), dict(table_width=0), dict(table_ld=3), dict(page_size=0),
              dict(page_size=-16)]


@pytest.mark.parametrize("bad", BAD_TABLES)
def test_bad_tables_are_refused(nqlib, bad):
    t, p = table(**bad), pool()
    t_, p_ = ctypes.byref(t), ctypes.byref(p)
    assert nqlib.nq_pages_free(t_, A, 1, None) == 1
    assert nqlib.nq_pages_fork(t_, A, A, 1, None) == 1
    assert nqlib.nq_pages_reserve(t_, p_, A, A, 1, A, 1 << 30, None) == 1
    assert nqlib.nq_pages_compact(t_, p_, A, 1 << 30, None) == 1
    assert nqlib.nq_last_error()


@pytest.mark.parametrize("bad", [dict(data=None), dict(data=A + 8), dict(outer=0), dict(n_pages=0),
                                 dict(page_bytes=0), dict(page_bytes=24), dict(n_pages=9)])
def test_bad_pools_are_refused(nqlib, bad):
    t, p = table(), pool(**bad)
    t_, p_ = ctypes.byref(t), ctypes.byref(p)
    assert nqlib.nq_pages_reserve(t_, p_, A, A, 1, A, 1 << 30, None) == 1
    assert nqlib.nq_pages_compact(t_, p_, A, 1 << 30, None) == 1
    if "n_pages" not in bad or bad["n_pages"] == 0:
        assert nqlib.nq_pages_copy(p_, A, A, 1, None) == 1


def test_a_list_that_could_ask_for_2_31_pages_is_refused(nqlib):
    t, p = table(table_width=1 << 16, table_ld=1 << 16, n_rows=1 << 16), pool()
    t_, p_ = ctypes.byref(t), ctypes.byref(p)
    assert nqlib.nq_pages_reserve(t_, p_, A, A, 1 << 15, A, 1 << 40, None) == 1


def test_lists_whose_checks_would_take_minutes_are_refused(nqlib):
    t, p = table(table_width=1, table_ld=1), pool()
    t_, p_ = ctypes.byref(t), ctypes.byref(p)
    for n in ((1 << 16) + 1, 1 << 30):
        assert nqlib.nq_pages_reserve(t_, p_, A, A, n, A, 1 << 60, None) == 1
        assert b"entries" in nqlib.nq_last_error()
    for n in ((1 << 20) + 1, 1 << 30, 1 << 62):
        for rc in (nqlib.nq_pages_free(t_, A, n, None), nqlib.nq_pages_fork(t_, A, A, n, None),
                   nqlib.nq_pages_copy(p_, A, A, n, None)):
            assert rc == 1 and b"entries" in nqlib.nq_last_error()
    if nqlib.nq_device_count() == 0:  # (without a device, the longest lists that are taken get as far as that)
        for rc in (nqlib.nq_pages_reserve(t_, p_, A, A, 1 << 16, A, 1 << 60, None),
                   nqlib.nq_pages_free(t_, A, 1 << 20, None),
                   nqlib.nq_pages_copy(p_, A, A, 1 << 20, None)):
            assert rc not in (0, 1)


def test_sizes_whose_products_pass_64_bits_are_refused(nqlib):
    for call in (attend, append):
        for c, b in ((cache(), batch(table_width=1 << 60, table_ld=1 << 60)),
                     (cache(), batch(table_width=(1 << 60) + 4, table_ld=1 << 61)),
                     (cache(n_kv_heads=1 << 30, page_size=1 << 28), batch(table_width=1))):
            heads = c.n_kv_heads
            assert call(nqlib, c=c, b=b, heads=heads) == 1
            assert b"too large" in nqlib.nq_last_error()
    for width in (1 << 60, (1 << 60) + 4):
        t, p = table(table_width=width, table_ld=width), pool()
        t_, p_ = ctypes.byref(t), ctypes.byref(p)
        for rc in (nqlib.nq_pages_free(t_, A, 1, None), nqlib.nq_pages_fork(t_, A, A, 1, None),
                   nqlib.nq_pages_reserve(t_, p_, A, A, 1, A, 1 << 40, None),
                   nqlib.nq_pages_compact(t_, p_, A, 1 << 40, None)):
            assert rc == 1 and b"too large" in nqlib.nq_last_error()


def test_page_lists_and_counts_are_checked(nqlib):
    t, p = table(), pool()
    t_, p_ = ctypes.byref(t), ctypes.byref(p)
    assert nqlib.nq_pages_free(t_, None, 1, None) == 1
    assert nqlib.nq_pages_free(t_, A, -1, None) == 1
    assert nqlib.nq_pages_fork(t_, None, A, 1, None) == 1
    assert nqlib.nq_pages_fork(t_, A, None, 1, None) == 1
    assert nqlib.nq_pages_copy(p_, None, A, 1, None) == 1
    assert nqlib.nq_pages_copy(p_, A, A, -1, None) == 1
    assert nqlib.nq_pages_free(t_, None, 0, None) == 0
    assert nqlib.nq_pages_fork(t_, None, None, 0, None) == 0
    assert nqlib.nq_pages_copy(p_, None, None, 0, None) == 0


def test_llama_paged_entry_points_refuse_null(nqlib):
    c, b = cache(), batch()
    assert nqlib.nq_llama_set_prefill_chunk(None, 16) == 1
    assert nqlib.nq_llama_forward_workspace_size(None, 1, 1, 1, 16) == 0
    assert nqlib.nq_llama_forward(None, A, ctypes.byref(c), 0, ctypes.byref(b), 1, A, 1, A, A, A,
                                  1 << 30, None) == 1
    assert nqlib.nq_last_error()


def test_notes_of_cut_tiles_are_followed_only_within_the_call(nqlib, tmp_path):
    """What the merge reads from a workspace says where it reads and writes."""
    from neurons_b200 import build
    exe = str(tmp_path / "split_check")
    src = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp", "split_check.cu")
    subprocess.run([build.NVCC] + build.ARCH + ["-std=c++17", "-O1", "-I" + build.CSRC,
                                                "-I" + build.INCLUDE, src, "-o", exe], check=True)
    out = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and out.stdout.strip() == "ok", out.stdout + out.stderr
