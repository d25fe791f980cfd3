"""The paged 8-bit K/V cache and the draft check where a call's data decide: what
hidden positions hold, values at the ends of f32, entries that are not finite."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from nuthatch_b200._lib import lib
from tests import paged_model as pm
from tests.test_gpu_paged import NH_E_ARG, P, _append, _cuda, _probs, _same_cache, _setup, _stream, _verify_call

pytestmark = pytest.mark.gpu


def _attend(dev, q, n, p0, n_head, scale, window, sinks, rows=None):
    import torch

    rows, keep = dev.rows(n, p0) if rows is None else rows
    qd = _cuda(q.reshape(q.shape[0], -1))
    out = torch.full_like(qd, 7.0)
    assert lib().nh_paged_attention(C.byref(dev.kv), C.byref(rows), P(qd), n_head, scale, window, sinks, P(out),
                                    _stream()) == 0
    return out.cpu().numpy().reshape(q.shape)


def _seen(pos, total, window, sinks):
    t = np.arange(total)
    return (t <= pos) & ((window == 0) | (t > pos - window) | (t < sinks))


# Rows and heads a KV head that take each form: 2, 4, 8 and 16 queries a CTA, tiles.
FORMS = [(2, 1), (2, 2), (5, 1), (8, 2), (80, 2), (200, 1)]


@pytest.mark.parametrize("rows_n,group", FORMS)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("case", ["later pages", "earlier pages", "no numbers"])
def test_hidden_scales_do_not_count(gpu, rows_n, group, hd, case):
    """V's scale grows by many powers of two from page to page where causality hides the later pages from a row, or falls where the
    window hides the earlier ones, or is not a number there: each row is held to the largest value that it sees itself."""
    n_kv, page = 2, 16
    p0 = {"later pages": page - 1, "earlier pages": 60, "no numbers": page - 1}[case]
    window = 20 if case == "earlier pages" else 0
    total = p0 + rows_n
    rng, table, cache, dev = _setup([rows_n], [p0], group * n_kv, n_kv, hd, page, rows_n + hd)
    blocks = (total + page - 1) // page
    for b in range(blocks):
        pg = table[0, b]
        step = 200 // blocks
        e = -100 + step * b if case != "earlier pages" else 100 - step * b
        cache.scales[1][pg] = 1.0 if case == "no numbers" else 2.0 ** e
        if case == "no numbers" and b > 0:
            cache.scales[0][pg], cache.scales[1][pg] = [np.nan, np.inf], [np.inf, np.nan]
    for w in range(2):
        dev.scales[w].copy_(_cuda(cache.scales[w]))
    q = rng.standard_normal((rows_n, group * n_kv, hd)).astype(np.float32)
    got = _attend(dev, q, [rows_n], [p0], group * n_kv, 0.125, window, 0)
    clean = cache.copy()
    for w in range(2):
        clean.scales[w][~np.isfinite(clean.scales[w])] = 1.0
    k, v = clean.values(0, table[0], total), clean.values(1, table[0], total)
    want, size = pm.attention(q, k, v, p0, 0.125, window, 0)
    for i in range(rows_n):
        sel = _seen(p0 + i, total, window, 0)
        if case == "no numbers" and p0 + i >= page:
            break
        bound = pm.attention_bound(size, hd, total, np.abs(v[sel]).max())
        assert np.abs(got[i] - want[i]).max() <= bound, i


@pytest.mark.parametrize("n_head", [2, 4])
def test_pages_behind_the_window_may_be_gone(gpu, n_head):
    """A sequence that gives up its pages between the sinks and the window: nothing is reported, nothing missed."""
    n_kv, hd, page, window, sinks = 2, 64, 16, 50, 4
    for rows_n in (1, 3, 9, 120):
        p0 = 307
        total = p0 + rows_n
        rng, table, cache, dev = _setup([rows_n], [p0], n_head, n_kv, hd, page, rows_n)
        first = (p0 - window + 1) // page  # the page of the first position that the first row's window holds
        for b in range(1, first):
            dev.table[0, b] = -1 if b % 2 else 1 << 29
        q = rng.standard_normal((rows_n, n_head, hd)).astype(np.float32)
        got = _attend(dev, q, [rows_n], [p0], n_head, 0.125, window, sinks)
        assert int(dev.err.item()) == 0, rows_n
        k, v = cache.values(0, table[0], total), cache.values(1, table[0], total)
        want, size = pm.attention(q, k, v, p0, 0.125, window, sinks)
        assert np.abs(got - want).max() <= pm.attention_bound(size, hd, total, np.abs(v).max())
        # one page more is missed
        dev.table[0, first] = -1
        _attend(dev, q, [rows_n], [p0], n_head, 0.125, window, sinks)
        assert int(dev.err.item()) == NH_E_ARG, rows_n


@pytest.mark.parametrize("rows_n,group", FORMS)
def test_largest_values(gpu, rows_n, group):
    """Values up to f32's range: the sum of the weighted values passes it, their mean does not."""
    n_kv, hd, page = 2, 64, 16
    for p0 in (100, 3000):
        total = p0 + rows_n
        rng, table, cache, dev = _setup([rows_n], [p0], group * n_kv, n_kv, hd, page, rows_n)
        cache.scales[1][:] = 2.0 ** 121
        cache.codes[1][:] = np.where(rng.random(cache.codes[1].shape) < 0.9, 255, 0)
        dev.scales[1].copy_(_cuda(cache.scales[1]))
        dev.codes[1].copy_(_cuda(cache.codes[1]))
        q = rng.standard_normal((rows_n, group * n_kv, hd)).astype(np.float32)
        got = _attend(dev, q, [rows_n], [p0], group * n_kv, 0.125, 0, 0).astype(np.float64)
        k, v = cache.values(0, table[0], total), cache.values(1, table[0], total)
        want, size = pm.attention(q, k, v, p0, 0.125, 0, 0)
        assert np.abs(got - want).max() <= pm.attention_bound(size, hd, total, np.abs(v).max()), p0


@pytest.mark.parametrize("hd,page", [(32, 16), (64, 32), (96, 128), (128, 64)])
def test_codes_of_tiny_values_under_large_scales(gpu, hd, page):
    """floor(x / scale) of a negative x is -1 however small x is, in one call or over several."""
    n_kv, n = 2, 9
    rng, table, cache, dev = _setup([n], [0], n_kv, n_kv, hd, page, 4)
    _, _, _, dev2 = _setup([n], [0], n_kv, n_kv, hd, page, 4)
    v = (-np.exp2(rng.uniform(-148, 60, (n, n_kv, hd)))).astype(np.float32)
    v[:, :, ::3] *= -1
    v[:, :, ::5] = 0.0
    v[n - 1, 0, 1], v[n - 2, 1, 2] = 3.3e38, -2.0 ** 100
    k = v[::-1].copy()
    cs = np.zeros((n + 1, hd // 2, 2), np.float32)
    cs[:, :, 0] = 1.0  # no rotation: K's rows are coded as they are
    want = cache.copy()
    for w, x in enumerate((k, v)):
        want.append(w, table[0], 0, x)
    kd, vd, cs = _cuda(k.reshape(n, -1)), _cuda(v.reshape(n, -1)), _cuda(cs)
    rc, keep = _append(dev, [n], [0], None, kd, vd, None, None, cs, n_kv, None)
    assert rc == 0 and int(dev.err.item()) == 0
    _same_cache(dev.host(), want)
    for at in range(n):
        rc, keep = _append(dev2, [1], [at], None, kd[at:], vd[at:], None, None, cs, n_kv, None)
        assert rc == 0
    _same_cache(dev2.host(), want)


def test_verify_infinite_entries(gpu):
    """An infinite draft entry takes its own id's mass alone; a target row with an infinite one has no distribution."""
    v, n = 700, 4
    rng = np.random.default_rng(2)
    off = np.arange(0, n + 1)
    target, draft = _probs(rng, 2 * n, v, 1.0), _probs(rng, n, v, 1.0)
    ids = np.array([3, 4, 5, 6])
    for s in range(n):
        draft[s, ids[s]] = 1.0
    draft[0, [3, 9, 300]] = np.inf
    draft[1, 4] = np.inf
    draft[1, 650] = -np.inf      # not above 0: no mass
    draft[2, :] = np.inf         # nothing is left: the target's own mass
    target[2 * 3, 8] = np.inf    # the row that sequence 3's draw is from
    ua, up = np.full(n, 0.9, np.float32), np.array([0.2, 0.7, 0.5, 0.5], np.float32)
    acc, out, err = _verify_call(target, draft, ids, off, ua, up)
    want_acc, want = pm.verify(target, draft, ids, off, ua, up)
    assert list(acc) == [0, 0, 0, 0] == want_acc
    assert [int(out[s, 0]) for s in range(3)] == [want[s][0] for s in range(3)]
    assert int(out[3, 0]) == -1 and err == NH_E_ARG
    acc, out, err = _verify_call(target[:6], draft[:3], ids[:3], off[:4], ua[:3], up[:3])
    assert err == 0 and [int(out[s, 0]) for s in range(3)] == [want[s][0] for s in range(3)]


@pytest.mark.parametrize("n,p0", [([1, 1, 1], [20, 0, 333]), ([4, 2, 0], [20, 0, 333]), ([90, 1, 40], [0, 500, 30])])
def test_rows_amid_larger_buffers(gpu, n, p0):
    """Offsets that do not begin at 0, and bounds (rows, rows of a sequence, pages of the table) far above what the call
    holds, as a captured step's are: the same rows and cache, the rest of the buffers left as it was."""
    import torch

    n_head, n_kv, hd, page, lead, behind = 8, 4, 64, 16, 3, 2000
    R, dq, dkv = sum(n), n_head * hd, n_kv * hd
    cs = _cuda(pm.rope_table(hd, 700))
    got = []
    for wide in (False, True):
        rng, table, cache, dev = _setup(n, p0, n_head, n_kv, hd, page, 6)
        if wide:
            dev = pm.Device(cache, np.concatenate([table, np.full((len(n), 900), -1)], 1))
        a, b = (lead, lead + R + behind) if wide else (0, R)
        bufs = [torch.full((b, w), 7.0, device="cuda") for w in (dq, dkv, dkv, dq, dq, dkv, dkv)]
        q, k, v, qr, out, ko, vo = bufs
        for x in (q, k, v):
            x[a:a + R] = _cuda(rng.standard_normal((R, x.shape[1])).astype(np.float32))
        more = dict(max_rows=4000, n_rows=b, offset=lead) if wide else {}
        rc, keep = _append(dev, n, p0, q, k, v, None, None, cs, n_head, qr, **more)
        assert rc == 0
        rows, keep2 = dev.rows(n, p0, **more)
        assert lib().nh_paged_attention(C.byref(dev.kv), C.byref(rows), P(qr), n_head, 0.125, 0, 0, P(out), _stream()) == 0
        assert lib().nh_paged_read(C.byref(dev.kv), C.byref(rows), 0, P(ko), P(vo), _stream()) == 0
        assert int(dev.err.item()) == 0
        for x in bufs[3:]:
            assert (x[:a] == 7.0).all() and (x[a + R:] == 7.0).all()
        h = dev.host()
        got.append((qr[a:a + R], ko[a:a + R], vo[a:a + R], out[a:a + R], h))
    for x, y in zip(got[0][:3], got[1][:3]):
        assert torch.equal(x, y)
    _same_cache(got[1][4], got[0][4])
    at = 0
    for s, m in enumerate(n):
        if m:
            total = m + p0[s]
            k, v = got[0][4].values(0, table[s], total), got[0][4].values(1, table[s], total)
            qs = got[0][0][at:at + m].cpu().numpy().reshape(m, n_head, hd)
            want, size = pm.attention(qs, k, v, p0[s], 0.125, 0, 0)
            for g in got:  # how the positions are shared out depends on the bounds, so the bits may differ
                err = np.abs(g[3][at:at + m].cpu().numpy().reshape(want.shape) - want).max()
                assert err <= pm.attention_bound(size, hd, total, np.abs(v).max())
        at += m
