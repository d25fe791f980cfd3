"""The launch shapes of the paged 8-bit K/V cache and of the draft check that a batch's
sizes choose: every query form under windows, long walks, wide clusters, one CTA a
sequence, several rounds of heads; and how exact the attention is, row by row."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from nuthatch_b200._lib import lib
from tests import paged_model as pm
from tests.test_gpu_paged import (EPS, P, _append, _attend_case, _cuda, _probs, _same_cache, _setup, _stream,
                                  _verify_call)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hd,page", [(32, 128), (64, 32), (96, 16), (128, 64)])
@pytest.mark.parametrize("rows_n,group", [(1, 1), (2, 1), (1, 2), (2, 2), (1, 3), (4, 2), (1, 8), (5, 3)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (21, 4), (100, 19)])
def test_decode_forms(gpu, hd, page, rows_n, group, window, sinks):
    """Batches whose sequences all bring the same few rows, so that each query form is the one that runs."""
    p0 = [0, 13, 127, 128, 500, 1]
    _attend_case([rows_n] * len(p0), p0, 3 * group, 3, hd, page, window, sinks, hd + rows_n + 7 * group + window)


def _reference(dev, cache, table, q, p0, scale, window, sinks):
    """One sequence's rows q [n][heads][hd] at p0.. by the formula in 64 bits, on the GPU; with it the spread of the scores."""
    import torch

    n, heads, hd = q.shape
    total = p0 + n
    pages = torch.from_numpy(np.ascontiguousarray(table[:(total + cache.page - 1) // cache.page].astype(np.int64))).cuda()
    k, v = ((dev.codes[w][pages].double() - 127.5) * dev.scales[w][pages].double()[:, :, None, None] for w in range(2))
    k, v = (x.transpose(1, 2).reshape(-1, cache.n_kv, hd)[:total] for x in (k, v))
    at = torch.arange(p0, total, device="cuda")[:, None]
    t = torch.arange(total, device="cuda")[None]
    hidden = t > at
    if window:
        hidden |= (t <= at - window) & (t >= sinks)
    out = torch.empty(n, heads, hd, dtype=torch.float64, device="cuda")
    spread = 0.0
    for h in range(heads):
        kh = h // (heads // cache.n_kv)
        s = (q[:, h].double() @ k[:, kh].t()) * scale
        spread = max(spread, float(s.pow(2).mean().sqrt()))
        out[:, h] = torch.softmax(s.masked_fill(hidden, -np.inf), 1) @ v[:, kh]
    return out, spread


def _precise(n, p0, n_head, n_kv, hd, page, window=0, sinks=0, positive=False, seed=3):
    """Relative root-mean-square error of each sequence's rows.

    With weights w_t and values v_t of both signs the result's size is sqrt(sum w^2) |v|, and independent relative errors
    d of the weights make an error of sqrt(sum w^2) |v| d: d is what is bounded.  The steps: hd / 8 products of 16 terms
    added by the tensor cores, each cutting the sum off by less than 2^-22 of it, so by 2^-22 sqrt(16) = 2^-20 of a score s
    as a root mean square; the score's factor, ex2.approx and the two f16 parts of query and weight, five steps of 2^-22
    and less.  2^-18 (1 + s) has a factor of four over their sum.  Planted in
    a restatement of the formula, a single f16 part of the weights is 2.6 to 9 times over it, one of the queries 9 times and
    more.
    Values of one sign (positive): errors that pull every sum one way stay.  At most three tiles of 16 products each are
    added up in tensor memory, which cuts 48 times less than 2^-22 of what is half the sum on average: 2^-17.4, and 2^-17
    is the bound.  64 tiles in one sum would cut 20 times that at most."""
    import torch

    rng, table, cache, dev = _setup(n, p0, n_head, n_kv, hd, page, seed)
    if positive:
        cache.codes[1][:] = rng.integers(160, 256, cache.codes[1].shape, dtype=np.uint8)
        dev.codes[1].copy_(_cuda(cache.codes[1]))
        cache.scales[1][:] = 2.0 ** -6
        dev.scales[1].copy_(_cuda(cache.scales[1]))
    q = _cuda(rng.standard_normal((sum(n), n_head * hd)).astype(np.float32))
    out = torch.empty_like(q)
    rows, keep = dev.rows(n, p0)
    scale = 1.0 / float(np.sqrt(hd))
    assert lib().nh_paged_attention(C.byref(dev.kv), C.byref(rows), P(q), n_head, scale, window, sinks, P(out),
                                    _stream()) == 0
    assert int(dev.err.item()) == 0
    at = 0
    for s, m in enumerate(n):
        if m:
            want, spread = _reference(dev, cache, table[s], q[at:at + m].view(m, n_head, hd), p0[s], scale, window, sinks)
            err = (out[at:at + m].double().view_as(want) - want).pow(2).mean().sqrt() / want.pow(2).mean().sqrt()
            bound = 2.0 ** -17 if positive else 2.0 ** -18 * (1 + spread)
            assert float(err) <= bound, (s, float(err), bound)
        at += m


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("positive", [False, True])
@pytest.mark.parametrize("n,p0,n_head", [([1] * 3, [900, 5000, 33], 4), ([1] * 3, [900, 5000, 33], 16), ([2, 2], [4000, 70], 16),
                                         ([4, 3], [4000, 70], 16), ([70, 1], [4000, 900], 8)])
def test_attention_precision(gpu, hd, positive, n, p0, n_head):
    """Every form: 2, 4, 8, 16 queries and tiles."""
    _precise(n, p0, n_head, 4, hd, 16, positive=positive)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("positive", [False, True])
@pytest.mark.parametrize("window", [0, 5000])
def test_attention_long_walk_tiles(gpu, hd, positive, window):
    """80 tiles of rows whose CTAs walk 68 tiles of positions alone (page ids are fetched 16 tiles at a time)."""
    _precise([640], [8000], 16, 16, hd, 16, window=window, sinks=3, positive=positive)


@pytest.mark.parametrize("hd,page", [(64, 16), (128, 32), (96, 64), (32, 128)])
@pytest.mark.parametrize("rows_n,group", [(1, 1), (1, 4), (2, 3), (3, 4)])
@pytest.mark.parametrize("window", [0, 9000])
def test_attention_long_walk_rows(gpu, hd, page, rows_n, group, window):
    """A batch with a CTA a (sequence, KV head), one sequence of which is long: more than 64 units a warp (page ids are
    fetched 32 units at a time)."""
    n_kv = 16 if hd <= 64 else 8
    p0 = [10000] + [100 + 7 * i for i in range(39)]
    _precise([rows_n] * len(p0), p0, n_kv * group, n_kv, hd, page, window=window, sinks=20)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("rows_n,group,total", [(1, 1, 33000), (2, 1, 40003), (1, 4, 33333), (2, 4, 17001), (3, 4, 20000),
                                                (4, 8, 16500)])
def test_attention_wide_clusters(gpu, hd, rows_n, group, total):
    """One long sequence of few heads: sixteen CTAs a KV head (two and four queries from 32,768 positions on, more from
    16,384)."""
    _precise([rows_n], [total - rows_n], 2 * group, 2, hd, 16)
    _precise([rows_n], [total - rows_n], 2 * group, 2, hd, 64, window=total - 100, sinks=5)


@pytest.mark.parametrize("hd", [32, 64, 96, 128])
@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("norm", [False, True])
def test_append_large_batches(gpu, hd, page, norm):
    """More than 200 pages times sequences of a call: four CTAs a page, several rounds of heads each (of q and of K and V);
    pages begun by this call and by earlier ones, bit for bit."""
    import torch

    n_head, n_kv = 32, 16
    n_seq = 12 if page <= 32 else 40
    rng0 = np.random.default_rng(page + hd)
    n = [int(x) for x in rng0.integers(1, 2 * page if page <= 32 else 40, n_seq)]
    n[0] = (200 // n_seq + 2) * page + 3 if page <= 32 else 5 * page + 1
    n[1] = 0
    p0 = [int(x) for x in rng0.integers(0, 3 * page, n_seq)]
    p0[2] = 0
    assert ((max(n) + page - 2) // page + 1) * n_seq > 200
    rng, table, cache, dev = _setup(n, p0, n_head, n_kv, hd, page, 17 + page)
    R, dq, dkv = sum(n), n_head * hd, n_kv * hd
    q, k, v = (rng.standard_normal((R, w)).astype(np.float32) for w in (dq, dkv, dkv))
    v *= np.exp(rng.standard_normal((R, 1)).astype(np.float32))
    qn, kn = (rng.uniform(0.5, 1.5, w).astype(np.float32) if norm else None for w in (dq, dkv))
    cs = pm.rope_table(hd, max(a + b for a, b in zip(n, p0)))
    pos = np.concatenate([np.arange(b, b + a) for a, b in zip(n, p0)])
    want = cache.copy()
    kr = pm.rotated_keys(k, kn, pos, cs, n_kv, EPS)
    at = 0
    for s in range(n_seq):
        for w, x in enumerate((kr, v.reshape(R, n_kv, hd))):
            want.append(w, table[s], p0[s], x[at:at + n[s]])
        at += n[s]
    qr = torch.full((R, dq), 7.0, device="cuda")
    rc, keep = _append(dev, n, p0, _cuda(q), _cuda(k), _cuda(v), None if qn is None else _cuda(qn),
                       None if kn is None else _cuda(kn), _cuda(cs), n_head, qr)
    assert rc == 0
    assert int(dev.err.item()) == 0
    _same_cache(dev.host(), want)
    assert np.array_equal(qr.cpu().numpy().reshape(R, n_head, hd), pm.rotated_rows(q, qn, pos, cs, n_head, EPS))


@pytest.mark.parametrize("n", [37, 38, 75, 76, 150, 151, 260])
@pytest.mark.parametrize("lookup", [False, True])
def test_verify_batches(gpu, n, lookup):
    """Eight, four, two CTAs a sequence and one; unequal counts of drafts, refused and accepted ones, and sequences whose
    refused row leaves nothing, so that the draw is from the target's own row."""
    v = 1777
    rng = np.random.default_rng(n)
    n_draft = rng.integers(0, 6, n)
    off = np.concatenate([[0], np.cumsum(n_draft)])
    T = int(off[-1])
    target = _probs(rng, T + n, v, 2.0)
    rows = np.concatenate([np.arange(off[s], off[s + 1]) + s for s in range(n)])
    draft = target[rows] * np.exp(0.5 * rng.standard_normal((T, v))).astype(np.float32)
    draft /= draft.sum(1, keepdims=True)
    ids = draft.argmax(1)
    ua, up = rng.random(T).astype(np.float32) * (0.3 if lookup else 1.3), rng.random(n).astype(np.float32)
    for s in range(0, n, 5):
        if n_draft[s] == 0:
            continue
        i = int(off[s])
        ua[i] = 0.99  # refused, and nothing left
        if lookup:
            ids[i] = 3
            target[rows[i]] = 0.0
            target[rows[i], 3] = 0.5
        else:
            draft[i] = np.maximum(target[rows[i]], draft[i])
            draft[i, ids[i]] = 2.0
    if lookup:
        draft = None
        for i in range(T):
            if target[rows[i], 3] != 0.5:
                ids[i] = target[rows[i]].argmax()
    acc, out, err = _verify_call(target, draft, ids, off, ua, up)
    want_acc, want = pm.verify(target, draft, ids, off, ua, up)
    assert err == 0
    assert list(acc) == want_acc
    assert 0 < sum(want_acc) < T
    for s in range(n):
        assert list(out[s, :acc[s] + 1]) == want[s], s
        assert (out[s, acc[s] + 1:] == -7).all()
