"""Refusals of the paged-cache entry points (include/b2_kernels.h) on a host
without a GPU: every call below is refused, or has nothing to do, before any
CUDA call.  The pointers are placeholders that are never dereferenced; on GPU
hosts the module is skipped, as test_abi_validation_cpu.py is."""
from __future__ import annotations

import ctypes

import pytest

import b200_decoder as bd

try:
    import torch

    _HAS_GPU = torch.cuda.is_available()
except ImportError:  # pragma: no cover
    _HAS_GPU = False

pytestmark = pytest.mark.skipif(_HAS_GPU, reason="placeholder pointers")

P = 4096


def cache(**kw):
    a = dict(k_pages=P, v_pages=P, page_stride=8 * 64 * 128, head_stride=64 * 128, row_stride=128, n_pages=10,
             page_size=64, n_seqs=2, max_pages=4, page_table=P, kv_len=P, q_start=P)
    a.update(kw)
    return bd.B2PagedKV(*[a[f] for f, _ in bd.B2PagedKV._fields_])


def append(kv=None, q16=P, ldq=2048, qkv=P, ldqkv=4096, M=4, nq=16, nkv=8, hd=128, cos=P, sin=P, max_pos=64, style=1):
    kv = cache() if kv is None else kv
    return bd.capi().b2_qk_rope_kv_paged(q16, ldq, qkv, ldqkv, M, nq, nkv, hd, None, None, 1e-6, cos, sin, max_pos, style,
                                         None, ctypes.byref(kv), None)


def attend(kv=None, out=P, q16=P, ldq=2048, M=4, max_q=1, nq=16, nkv=8, hd=128, work=P, err=P):
    kv = cache() if kv is None else kv
    return bd.capi().b2_attention_paged(out, None, q16, ldq, M, max_q, nq, nkv, hd, ctypes.byref(kv), work, err, None)


def weigh(kv=None, w=P, ldw=256, q16=P, ldq=2048, lse=P, M=4, max_q=1, nq=16, nkv=8, hd=128, err=P):
    kv = cache() if kv is None else kv
    return bd.capi().b2_attention_paged_weights(w, None, ldw, q16, ldq, lse, M, max_q, nq, nkv, hd, ctypes.byref(kv), err,
                                                None)


def evict(kv=None, nkv=8, hd=128, w=P, ldw=256, budget=64, sink=4, recent=8, dst=P, dst_pages=1, kept=P, new_len=P):
    kv = cache() if kv is None else kv
    return bd.capi().b2_kv_evict_paged(ctypes.byref(kv), nkv, hd, w, ldw, budget, sink, recent, dst, dst_pages, kept, None,
                                       new_len, None)


BAD_CACHE = [dict(k_pages=None), dict(v_pages=None), dict(page_table=None), dict(kv_len=None), dict(page_size=48),
             dict(page_size=8), dict(page_size=256), dict(n_pages=0), dict(max_pages=0), dict(n_seqs=-1), dict(n_seqs=1025),
             dict(k_pages=P + 8), dict(v_pages=P + 2), dict(page_stride=8 * 64 * 128 + 4), dict(head_stride=12),
             dict(row_stride=132), dict(row_stride=64), dict(page_stride=0), dict(head_stride=-128),
             dict(page_stride=1 << 39), dict(max_pages=1 << 26)]


@pytest.mark.parametrize("bad", BAD_CACHE)
@pytest.mark.parametrize("call", [append, attend, weigh, evict])
def test_bad_cache(call, bad):
    assert call(kv=cache(**bad)) == -1
    assert b"paged" in bd.capi().b2_last_error()


@pytest.mark.parametrize("call", [append, attend, weigh])
def test_rows_need_q_start(call):
    assert call(kv=cache(q_start=None)) == -1


@pytest.mark.parametrize("call", [append, attend, weigh, evict])
@pytest.mark.parametrize("hd", [0, 32, 96, 256])
def test_head_dims(call, hd):
    assert call(hd=hd) == -1


@pytest.mark.parametrize("bad", [dict(q16=None), dict(qkv=None), dict(cos=None), dict(sin=None), dict(M=-1), dict(nq=0),
                                 dict(nkv=0), dict(max_pos=0), dict(style=2), dict(ldqkv=4092), dict(ldqkv=4098),
                                 dict(ldq=2040), dict(ldq=2050), dict(qkv=P + 8), dict(q16=P + 4)])
def test_append_refuses(bad):
    assert append(**bad) == -1


@pytest.mark.parametrize("bad", [dict(out=None), dict(q16=None), dict(work=None), dict(err=None), dict(M=-1), dict(max_q=-1),
                                 dict(nq=12), dict(nq=0), dict(nq=17 * 8, ldq=17 * 8 * 128), dict(ldq=2040), dict(ldq=2052),
                                 dict(q16=P + 8), dict(out=P + 8), dict(work=P + 8)])
def test_attention_refuses(bad):
    assert attend(**bad) == -1


@pytest.mark.parametrize("bad", [dict(w=None), dict(q16=None), dict(lse=None), dict(err=None), dict(M=-1), dict(max_q=-1),
                                 dict(nq=12), dict(nq=17 * 8, ldq=17 * 8 * 128), dict(ldq=2040), dict(ldq=2052),
                                 dict(q16=P + 8), dict(ldw=-1)])
def test_weights_refuses(bad):
    assert weigh(**bad) == -1


@pytest.mark.parametrize("bad", [dict(w=None), dict(dst=None), dict(kept=None), dict(new_len=None), dict(budget=-1),
                                 dict(sink=-1), dict(recent=-1), dict(sink=40, recent=25), dict(dst_pages=0), dict(ldw=-1),
                                 dict(sink=2**31 - 1, recent=2**31 - 1)])
def test_evict_refuses(bad):
    assert evict(**bad) == -1


def test_nothing_to_do():
    assert append(M=0) == 0 and attend(M=0) == 0 and attend(max_q=0) == 0
    none = cache(n_seqs=0)
    assert append(kv=none) == 0 and attend(kv=none) == 0 and weigh(kv=none) == 0 and evict(kv=none) == 0


def test_workspace_size():
    size = bd.capi().b2_attention_paged_workspace
    assert 0 < size(1, 1, 16, 8, 64) < size(64, 4096, 16, 8, 128) < 256 << 20


def test_arrays_without_entries():
    """No sequences, no rows or no budget: the arrays that would be empty may be NULL."""
    none = cache(n_seqs=0, page_table=None, kv_len=None, q_start=None)
    assert append(kv=none, M=0, q16=None, qkv=None) == 0
    assert attend(kv=none, M=0, q16=None, out=None) == 0
    assert weigh(kv=none, M=0, q16=None, lse=None, w=None) == 0
    assert evict(kv=none, w=None, new_len=None) == 0
    assert append(M=0, q16=None, qkv=None) == 0 and attend(M=0, q16=None, out=None) == 0
    assert append(M=1, q16=None) == -1 and attend(M=1, out=None) == -1 and weigh(M=1, lse=None) == -1


def arrays_of_an_eviction(**at):
    """Two sequences, 8 kv heads, rows of 256 weights, 64 slots kept; `at` moves arrays."""
    a = dict(w=1 << 20, kept=2 << 20, dw=3 << 20, new_len=4 << 20, table=5 << 20, kv_len=6 << 20, dst=7 << 20)
    a.update(at)
    return a


def evict_at(**at):
    a = arrays_of_an_eviction(**at)
    kv = cache(page_table=a["table"], kv_len=a["kv_len"])
    return bd.capi().b2_kv_evict_paged(ctypes.byref(kv), 8, 128, a["w"], 256, 64, 4, 8, a["dst"], 1, a["kept"], a["dw"],
                                       a["new_len"], None)


W, K = 2 * 8 * 256 * 4, 2 * 8 * 64 * 4  # bytes of weights; of kept and of dst_weights


@pytest.mark.parametrize("bad", [
    dict(dw=1 << 20), dict(dw=(1 << 20) + W - 4), dict(dw=(1 << 20) - K + 4),           # weights moved in place
    dict(kept=1 << 20), dict(kept=(1 << 20) + W - 4), dict(kept=3 << 20), dict(kept=(3 << 20) - K + 4),
    dict(kept=(5 << 20) + 28), dict(kept=7 << 20), dict(kept=(7 << 20) + 4), dict(kept=6 << 20),
    dict(new_len=6 << 20), dict(new_len=(6 << 20) + 4), dict(new_len=(6 << 20) - 4),     # lengths updated in place
    dict(new_len=1 << 20), dict(new_len=2 << 20), dict(new_len=(3 << 20) + K - 4), dict(new_len=5 << 20), dict(new_len=7 << 20)])
def test_evict_refuses_overlap(bad):
    assert evict_at(**bad) == -1
    assert b"overlaps" in bd.capi().b2_last_error()


def test_blocks_of_work_in_one_call():
    """Products of rows, heads and table width that the kernels' 32-bit places could not hold."""
    wide = cache(n_seqs=1024, max_pages=16384)  # tables of a million slots: 2^14 blocks of 64
    assert attend(kv=wide, M=16384, max_q=1) == -1 and b"blocks of work" in bd.capi().b2_last_error()
    assert attend(kv=cache(n_seqs=1, max_pages=1 << 24), M=1 << 20, max_q=1 << 20) == -1
    assert b"blocks of work" in bd.capi().b2_last_error()
    assert weigh(kv=cache(n_seqs=1024, max_pages=1 << 19)) == -1
    assert b"blocks of work" in bd.capi().b2_last_error()
