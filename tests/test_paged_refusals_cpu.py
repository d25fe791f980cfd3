"""Argument checks of the paged-cache and draft-check entries: refused calls
launch nothing, so they need no GPU."""
from __future__ import annotations

import ctypes as C

import pytest

from nuthatch_b200._lib import NhPagedKv, NhPagedRows, NhVerifyDrafts, lib

NH_E_ARG, NH_E_TYPE = -1, -3
A = 1 << 20  # an aligned address that nothing reads


def _kv(**k):
    f = dict(k_codes=A, v_codes=A, k_scales=A, v_scales=A, n_pages=8, page_size=16, n_head_kv=4, head_dim=64)
    f.update(k)
    return NhPagedKv(**f)


def _rows(**k):
    f = dict(n_seq=2, max_rows=4, n_rows=8, max_blocks=4, row_off=A, pos0=A, page_table=A, err=None)
    f.update(k)
    return NhPagedRows(**f)


BAD_KV = [dict(k_codes=None), dict(v_codes=None), dict(k_scales=None), dict(v_scales=None), dict(k_codes=A + 8),
          dict(v_codes=A + 1), dict(n_pages=0), dict(page_size=0), dict(page_size=8), dict(page_size=24),
          dict(page_size=48), dict(page_size=256), dict(n_head_kv=0), dict(head_dim=0), dict(head_dim=16),
          dict(head_dim=80), dict(head_dim=160), dict(head_dim=-32)]
BAD_ROWS = [dict(row_off=None), dict(pos0=None), dict(page_table=None), dict(n_seq=0), dict(n_seq=65536),
            dict(max_rows=-1), dict(n_rows=-1), dict(max_blocks=0), dict(max_blocks=1 << 28)]


def _attention(kv, rows, q=A, n_head=8, scale=0.1, window=0, sinks=0, out=A):
    return lib().nh_paged_attention(kv if kv is None else C.byref(kv), rows if rows is None else C.byref(rows), q, n_head,
                                    scale, window, sinks, out, None)


def _append(kv, rows, **k):
    f = dict(q=A, qs=512, k=A, ks=256, v=A, vs=256, qn=A, kn=A, n_head=8, rope=A, rope_len=64, qr=A)
    f.update(k)
    return lib().nh_paged_append(kv if kv is None else C.byref(kv), rows if rows is None else C.byref(rows), f["q"],
                                 f["qs"], f["k"], f["ks"], f["v"], f["vs"], f["qn"], f["kn"], 1e-5, f["n_head"],
                                 f["rope"], f["rope_len"], f["qr"], None)


def _read(kv, rows, out_type=0, k=A, v=A):
    return lib().nh_paged_read(kv if kv is None else C.byref(kv), rows if rows is None else C.byref(rows), out_type, k, v,
                               None)


@pytest.mark.parametrize("call", [_attention, _append, _read])
def test_cache_and_rows_are_checked(call):
    assert call(None, _rows()) == NH_E_ARG
    assert call(_kv(), None) == NH_E_ARG
    for bad in BAD_KV:
        assert call(_kv(**bad), _rows()) == NH_E_ARG, bad
    for bad in BAD_ROWS:
        assert call(_kv(), _rows(**bad)) == NH_E_ARG, bad


def test_attention_arguments():
    for bad in (dict(q=None), dict(out=None), dict(q=A + 4), dict(out=A + 8), dict(n_head=0), dict(n_head=6),
                dict(n_head=-4), dict(window=-1), dict(sinks=-1)):
        assert _attention(_kv(), _rows(), **bad) == NH_E_ARG, bad
    big = (1 << 31) - 1
    assert _attention(_kv(), _rows(n_rows=big, max_rows=big), n_head=8) == NH_E_ARG  # more queries than 32 bits count
    assert _attention(_kv(), _rows(n_rows=0)) == 0  # nothing to do


def test_append_arguments():
    for bad in (dict(k=None), dict(v=None), dict(rope=None), dict(rope_len=0), dict(q=None), dict(qr=None),
                dict(qn=None), dict(kn=None), dict(n_head=0), dict(n_head=7), dict(qs=508), dict(ks=252), dict(vs=252),
                dict(qs=513), dict(ks=258), dict(vs=257), dict(q=A + 4), dict(k=A + 4), dict(v=A + 8), dict(qr=A + 4),
                dict(rope=A + 8), dict(qn=A + 4), dict(kn=A + 4)):
        assert _append(_kv(), _rows(), **bad) == NH_E_ARG, bad
    for k in ("qs", "ks", "vs"):
        assert _append(_kv(), _rows(), **{k: (1 << 23) + 4}) == NH_E_ARG
    assert _append(_kv(), _rows(n_rows=0)) == 0
    assert _append(_kv(), _rows(max_rows=0)) == 0


def test_read_arguments():
    assert _read(_kv(), _rows(), out_type=12) == NH_E_TYPE
    assert _read(_kv(), _rows(), k=A + 4) == NH_E_ARG
    assert _read(_kv(), _rows(), k=None, v=None) == 0
    assert _read(_kv(), _rows(n_rows=0)) == 0


def test_verify_arguments():
    def call(**k):
        f = dict(target=A, target_stride=100, draft=A, draft_stride=100, draft_ids=A, draft_off=A, u_accept=A, u_pick=A,
                 n_seq=2, n_drafts=4, max_draft=2, n_vocab=100, n_accept=A, out_ids=A, err=None)
        f.update(k)
        return lib().nh_verify_drafts(C.byref(NhVerifyDrafts(**f)), None)

    for bad in (dict(target=None), dict(draft_off=None), dict(u_pick=None), dict(n_accept=None), dict(out_ids=None),
                dict(draft_ids=None), dict(u_accept=None), dict(n_seq=0), dict(n_seq=65536), dict(n_drafts=-1),
                dict(max_draft=-1), dict(max_draft=1025), dict(n_vocab=0), dict(n_vocab=1 << 31), dict(target_stride=99),
                dict(draft_stride=99)):
        assert call(**bad) == NH_E_ARG, bad
    assert lib().nh_verify_drafts(None, None) == NH_E_ARG
