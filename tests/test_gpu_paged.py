"""The paged 8-bit K/V cache (nh_paged_append, nh_paged_attention,
nh_paged_read) and the check of drafted tokens (nh_verify_drafts) against
numpy restatements in 64 bits."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from nuthatch_b200._lib import NhVerifyDrafts, lib
from tests import paged_model as pm

pytestmark = pytest.mark.gpu

EPS = 1e-5
NH_OK, NH_E_ARG = 0, -1
F32, BF16 = 0, 30
P = lambda t: None if t is None else C.c_void_p(t.data_ptr())  # noqa: E731


def _stream():
    import torch

    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


def _cuda(x):
    import torch

    return torch.from_numpy(np.ascontiguousarray(x)).cuda()


def _table(total, page, rng, spare=2):
    """Pages of each sequence, shuffled over the pool; unused places hold a page out of range."""
    need = [(t + page - 1) // page for t in total]
    order = rng.permutation(sum(need) + spare)
    table = np.full((len(total), max(max(need), 1)), 1 << 30, dtype=np.int64)
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = order[at:at + n]
        at += n
    return table, sum(need) + spare


def _setup(n, p0, n_head, n_kv, hd, page, seed):
    rng = np.random.default_rng(seed)
    table, n_pages = _table([a + b for a, b in zip(n, p0)], page, rng)
    cache = pm.Cache(n_pages, n_kv, page, hd, rng)
    return rng, table, cache, pm.Device(cache, table)


def _append(dev, n, p0, q, k, v, qn, kn, cs, n_head, qr, **more):
    rows, keep = dev.rows(n, p0, **more)
    rc = lib().nh_paged_append(C.byref(dev.kv), C.byref(rows), P(q), q.stride(0) if q is not None else 0, P(k),
                               k.stride(0), P(v), v.stride(0), P(qn), P(kn), EPS, n_head, P(cs), cs.shape[0], P(qr),
                               _stream())
    return rc, keep


def _same_cache(got, want):
    for w in range(2):
        assert np.array_equal(got.scales[w], want.scales[w])
        assert np.array_equal(got.codes[w], want.codes[w])


HEADS = [(16, 16, 128, 16), (6, 2, 64, 32), (3, 1, 96, 64), (10, 5, 32, 128), (24, 12, 32, 16)]


@pytest.mark.parametrize("n_head,n_kv,hd,page", HEADS)
@pytest.mark.parametrize("norm", [True, False])
def test_append_codes(gpu, n_head, n_kv, hd, page, norm):
    """One position, several inside a page, over pages, none, and a page that is begun here; old codes kept, or moved
    to a larger scale.  Codes, scales and rotated q bit for bit."""
    n = [1, 5, 2 * page + 3, 0, page, 1]
    p0 = [0, page - 2, 7, 4, page, 3 * page - 1]
    rng, table, cache, dev = _setup(n, p0, n_head, n_kv, hd, page, 11 * n_head + page)
    R, dq, dkv = sum(n), n_head * hd, n_kv * hd
    q, k, v = (rng.standard_normal((R, w)).astype(np.float32) for w in (dq, dkv, dkv))
    v *= np.exp(rng.standard_normal((R, 1)).astype(np.float32))
    qn, kn = (rng.uniform(0.5, 1.5, w).astype(np.float32) if norm else None for w in (dq, dkv))
    cs = pm.rope_table(hd, 6 * page)
    want = cache.copy()
    pos = np.concatenate([np.arange(b, b + a) for a, b in zip(n, p0)])
    kr = pm.rotated_keys(k, kn, pos, cs, n_kv, EPS)
    at = 0
    for s in range(len(n)):
        for w, x in enumerate((kr, v.reshape(R, n_kv, hd))):
            want.append(w, table[s], p0[s], x[at:at + n[s]])
        at += n[s]
    import torch

    # rows inside wider ones (a fused q, k, v product), two rows of the buffers behind the last
    fused = torch.zeros(R + 2, dq + 2 * dkv + 8, device="cuda")
    fused[:R, :dq], fused[:R, dq:dq + dkv], fused[:R, dq + dkv:dq + 2 * dkv] = _cuda(q), _cuda(k), _cuda(v)
    qr = torch.full((R + 2, dq), 7.0, device="cuda")
    rc, keep = _append(dev, n, p0, fused[:, :dq], fused[:, dq:], fused[:, dq + dkv:], None if qn is None else _cuda(qn),
                       None if kn is None else _cuda(kn), _cuda(cs), n_head, qr, n_rows=R + 2)
    assert rc == NH_OK
    torch.cuda.synchronize()
    assert int(dev.err.item()) == 0
    _same_cache(dev.host(), want)
    got = qr.cpu().numpy()
    assert np.array_equal(got[:R].reshape(R, n_head, hd), pm.rotated_rows(q, qn, pos, cs, n_head, EPS))
    assert (got[R:] == 7.0).all()


def test_append_matches_the_f32_cache_rows(gpu):
    """The coded rows are nh_prefill_qk's K and V rows: a value is off by half a scale at most (of K by its f32 roundings
    more: the factor, two products with it, two of the rotation and their sum, half a step of 2^-23 each of a magnitude of
    at most 64 scales' worth twice over), q bit for bit."""
    import torch

    n_head, n_kv, hd, page, n = 16, 8, 64, 32, 75
    rng, table, cache, dev = _setup([n], [0], n_head, n_kv, hd, page, 5)
    q, k, v = (_cuda(rng.standard_normal((n, w)).astype(np.float32)) for w in (n_head * hd, n_kv * hd, n_kv * hd))
    qn, kn = (_cuda(rng.uniform(0.5, 1.5, w).astype(np.float32)) for w in (n_head * hd, n_kv * hd))
    cs = _cuda(pm.rope_table(hd, n))
    kc, vc = (torch.zeros(n, n_kv * hd, device="cuda") for _ in range(2))
    a, b = (torch.zeros(n, n_head * hd, device="cuda") for _ in range(2))
    assert lib().nh_prefill_qk(P(q), P(k), P(v), P(qn), P(kn), EPS, n, 0, n_head, n_kv, hd, P(cs), P(kc), P(vc), n, P(a),
                               _stream()) == 0
    rc, keep = _append(dev, [n], [0], q, k, v, qn, kn, cs, n_head, b)
    assert rc == 0
    rows, keep2 = dev.rows([n], [0])
    for out_type, dt in ((F32, torch.float32), (BF16, torch.bfloat16)):
        ko, vo = (torch.empty(n, n_kv * hd, dtype=dt, device="cuda") for _ in range(2))
        assert lib().nh_paged_read(C.byref(dev.kv), C.byref(rows), out_type, P(ko), P(vo), _stream()) == 0
        torch.cuda.synchronize()
        for w, (got, want) in enumerate(((ko, kc), (vo, vc))):
            vals = dev.host().values(w, table[0], n).reshape(n, -1)
            assert np.array_equal(got.double().cpu().numpy(), vals)  # exact in both types
            sc = np.repeat(dev.host().scales[w][table[0]], page, 0)[:n].repeat(hd, 1)
            more = 0 if w else 128 * sc * 6 * 2.0 ** -24 * 2
            assert (np.abs(vals - want.double().cpu().numpy()) <= sc / 2 + more).all()
    assert torch.equal(a, b)


@pytest.mark.parametrize("page", [16, 128])
def test_append_split_over_calls(gpu, page):
    """One call, one position at a time, and uneven pieces leave the same cache."""
    n_head, n_kv, hd, total = 4, 4, 128, 2 * page + 9
    states = []
    for pieces in ([total], [1] * total, [3, page - 1, total - page - 2]):
        rng, table, cache, dev = _setup([total], [0], n_head, n_kv, hd, page, 3)
        k, v = (rng.standard_normal((total, n_kv * hd)).astype(np.float32) for _ in range(2))
        grow = np.exp(0.5 * rng.standard_normal((total, 1))).astype(np.float32)
        kd, vd, cs = _cuda(k * grow), _cuda(v * grow), _cuda(pm.rope_table(hd, total))
        at = 0
        for m in pieces:
            rc, keep = _append(dev, [m], [at], None, kd[at:], vd[at:], None, None, cs, n_head, None)
            assert rc == 0
            at += m
        states.append(dev.host())
    used = table[0][:(total + page - 1) // page]
    last = total % page
    for other in states[1:]:
        for w in range(2):
            a, b = states[0], other
            assert np.array_equal(a.scales[w][used], b.scales[w][used])
            assert np.array_equal(a.codes[w][used[:-1]], b.codes[w][used[:-1]])
            assert np.array_equal(a.codes[w][used[-1], :, :last], b.codes[w][used[-1], :, :last])


def test_append_extreme_values(gpu):
    """Zeros, subnormals, the largest floats, powers of two at a scale's border, and values that are not finite."""
    import torch

    n_kv, hd, page, n = 2, 32, 16, 12
    rng, table, cache, dev = _setup([n], [0], 2, n_kv, hd, page, 9)
    v = np.zeros((n, n_kv, hd), np.float32)
    v[1, 0, 3] = 1e-42
    v[2, 1, :4] = [1.0, -1.0, 0.9999999, -0.9999999]
    v[3, 1, :2] = [2.0 ** -5, -2.0 ** -5]
    cs = _cuda(pm.rope_table(hd, n + 4))
    k = _cuda(np.zeros((n, n_kv * hd), np.float32))
    rc, keep = _append(dev, [n], [0], None, k, _cuda(v.reshape(n, -1)), None, None, cs, 2, None)
    assert rc == 0
    torch.cuda.synchronize()
    assert int(dev.err.item()) == 0
    want = cache.copy()
    want.append(0, table[0], 0, np.zeros((n, n_kv, hd), np.float32))
    want.append(1, table[0], 0, v)
    _same_cache(dev.host(), want)
    # the largest floats grow every scale; then values that are not finite
    big = np.full((1, n_kv, hd), 3.4e38, np.float32)
    big[0, :, ::2] *= -1
    rc, keep = _append(dev, [1], [n], None, k, _cuda(big.reshape(1, -1)), None, None, cs, 2, None)
    want.append(1, table[0], n, big)
    want.append(0, table[0], n, np.zeros((1, n_kv, hd), np.float32))
    assert rc == 0
    torch.cuda.synchronize()
    assert int(dev.err.item()) == 0
    _same_cache(dev.host(), want)
    odd = np.ones((1, n_kv, hd), np.float32)
    odd[0, 0, :3] = [np.nan, np.inf, -np.inf]
    rc, keep = _append(dev, [1], [0], None, k, _cuda(odd.reshape(1, -1)), None, None, cs, 2, None)
    assert rc == 0
    torch.cuda.synchronize()
    assert int(dev.err.item()) == NH_E_ARG
    got = dev.host()
    pg = table[0][0]
    assert list(got.codes[1][pg, 0, 0, :4]) == [128, 255, 0, 128 + 64]
    assert got.scales[1][pg, 0] == 2.0 ** -6


def _attend_case(n, p0, n_head, n_kv, hd, page, window, sinks, seed, sharp=1.0):
    import torch

    rng, table, cache, dev = _setup(n, p0, n_head, n_kv, hd, page, seed)
    R = sum(n)
    q = (rng.standard_normal((R, n_head, hd)) * sharp).astype(np.float32)
    out = torch.full((R + 1, n_head * hd), 7.0, device="cuda")
    rows, keep = dev.rows(n, p0, n_rows=R + 1)
    qd = torch.zeros(R + 1, n_head * hd, device="cuda")
    qd[:R] = _cuda(q.reshape(R, -1))
    scale = 1.0 / float(np.sqrt(hd))
    call = lambda o: lib().nh_paged_attention(C.byref(dev.kv), C.byref(rows), P(qd), n_head, scale, window, sinks,  # noqa: E731
                                              P(o), _stream())
    assert call(out) == NH_OK
    again = torch.full((R + 1, n_head * hd), 7.0, device="cuda")
    assert call(again) == NH_OK
    torch.cuda.synchronize()
    assert int(dev.err.item()) == 0
    assert torch.equal(out, again)
    got = out.cpu().numpy()
    assert (got[R:] == 7.0).all()  # rows behind the last stay
    at = 0
    for s in range(len(n)):
        if n[s] == 0:
            continue
        total = p0[s] + n[s]
        k, v = cache.values(0, table[s], total), cache.values(1, table[s], total)
        want, size = pm.attention(q[at:at + n[s]], k, v, p0[s], scale, window, sinks)
        bound = pm.attention_bound(size, hd, total, np.abs(v).max())
        err = np.abs(got[at:at + n[s]].reshape(n[s], n_head, hd) - want).max()
        assert err <= bound, (s, err, bound)
        at += n[s]


@pytest.mark.parametrize("n_head,n_kv,hd,page", HEADS + [(32, 8, 128, 16), (16, 2, 64, 64), (17, 1, 128, 32)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (21, 4), (70, 17)])
def test_attention_decode_rows(gpu, n_head, n_kv, hd, page, window, sinks):
    """One row a sequence and a few drafted ones, from the first position of a sequence to ones that end inside a page,
    a tile and a split; a sequence without rows."""
    n = [1, 1, 0, 3, 1, 8, 1]
    p0 = [0, 15, 9, 126, 255, 300, 1100]
    _attend_case(n, p0, n_head, n_kv, hd, page, window, sinks, 7 * n_head + page + window)


@pytest.mark.parametrize("n_head,n_kv,hd,page", HEADS + [(8, 1, 128, 16), (40, 8, 64, 32)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (37, 3), (128, 0), (200, 150)])
def test_attention_prompt_rows(gpu, n_head, n_kv, hd, page, window, sinks):
    """Chunks from the first position on and behind cached ones, beside sequences with one row and none."""
    n = [130, 1, 300, 0, 64, 17]
    p0 = [0, 200, 77, 5, 600, 1]
    _attend_case(n, p0, n_head, n_kv, hd, page, window, sinks, 13 * n_head + page + window)


@pytest.mark.parametrize("n,p0", [([1], [5000]), ([9], [9000]), ([700], [1500]), ([40], [5000])])
def test_attention_long_and_sharp(gpu, n, p0):
    """Long caches with scores far apart (the running maximum moves often)."""
    _attend_case(n, p0, 8, 4, 64, 32, 0, 0, 21, sharp=40.0)


def test_attention_zero_queries_and_factors(gpu):
    """A factor of zero, a negative one and queries of zeros: weights by the formula (equal ones, or turned round), hidden
    positions hidden."""
    import torch

    n_head, n_kv, hd, page, total = 4, 2, 64, 16, 200
    for rows_n, window in ((1, 0), (3, 50), (60, 50), (130, 0)):
        rng, table, cache, dev = _setup([rows_n], [total - rows_n], n_head, n_kv, hd, page, 8)
        rows, keep = dev.rows([rows_n], [total - rows_n])
        k, v = cache.values(0, table[0], total), cache.values(1, table[0], total)
        for scale, size_q in ((0.0, 1.0), (-0.2, 1.0), (0.1, 0.0), (0.125, 1e-36), (1e-3, 1e3), (2.0**-126, 8e37)):
            q = np.clip(rng.standard_normal((rows_n, n_head, hd)) * size_q, -3.2e38, 3.2e38).astype(np.float32)
            out = torch.full((rows_n, n_head * hd), 7.0, device="cuda")
            qd = _cuda(q.reshape(rows_n, -1))
            assert lib().nh_paged_attention(C.byref(dev.kv), C.byref(rows), P(qd), n_head, scale, window, 2, P(out),
                                            _stream()) == 0
            want, size = pm.attention(q, k, v, total - rows_n, scale, window, 2)
            bound = pm.attention_bound(size, hd, total, np.abs(v).max())
            err = np.abs(out.cpu().numpy().reshape(want.shape) - want).max()
            assert err <= bound, (rows_n, window, scale, size_q, err, bound)


def test_attention_not_finite_queries_stay_apart(gpu):
    """A query that holds a NaN or an infinity gives no number in its own row and leaves the others as they are."""
    import torch

    n_head, n_kv, hd, page = 4, 2, 64, 16
    for rows_n in (2, 5, 100):
        total = rows_n + 150
        rng, table, cache, dev = _setup([rows_n], [150], n_head, n_kv, hd, page, 18)
        rows, keep = dev.rows([rows_n], [150])
        q = rng.standard_normal((rows_n, n_head * hd)).astype(np.float32)
        outs = []
        for bad in (False, True):
            if bad:
                q[1, hd + 5] = np.nan   # row 1, head 1
                q[0, 3 * hd + 1] = np.inf  # row 0, head 3
            out = torch.full((rows_n, n_head * hd), 7.0, device="cuda")
            qd = _cuda(q)
            assert lib().nh_paged_attention(C.byref(dev.kv), C.byref(rows), P(qd), n_head, 0.125, 0, 0, P(out),
                                            _stream()) == 0
            outs.append(out.cpu().numpy().reshape(rows_n, n_head, hd))
        same = np.ones((rows_n, n_head), bool)
        same[1, 1] = same[0, 3] = False
        assert np.array_equal(outs[0][same], outs[1][same])
        assert np.isnan(outs[1][1, 1]).all() and np.isnan(outs[1][0, 3]).all()


def test_attention_far_pages(gpu):
    """Pages beyond 2^31 bytes of the pool, for every form."""
    import torch

    n_head, n_kv, hd, page = 16, 16, 128, 128
    total = 300
    pages = 10000  # 2.6 GB of codes, keys and values apart
    codes = [torch.empty(pages, n_kv, page, hd, dtype=torch.uint8, device="cuda") for _ in range(2)]
    scales = [torch.empty(pages, n_kv, device="cuda") for _ in range(2)]
    rng = np.random.default_rng(6)
    small = pm.Cache(3, n_kv, page, hd, rng)
    order = [9999, 8700, 9100]
    for w in range(2):
        codes[w][order] = _cuda(small.codes[w])
        scales[w][order] = _cuda(small.scales[w])
    dev = pm.Device(small, np.array([order]))
    dev.kv = pm.NhPagedKv(codes[0].data_ptr(), codes[1].data_ptr(), scales[0].data_ptr(), scales[1].data_ptr(), pages, page,
                          n_kv, hd)
    k, v = small.values(0, [0, 1, 2], total), small.values(1, [0, 1, 2], total)
    for n in (1, 3, 6, 9, 50):
        q = rng.standard_normal((n, n_head, hd)).astype(np.float32)
        rows, keep = dev.rows([n], [total - n])
        out = torch.empty(n, n_head * hd, device="cuda")
        qd = _cuda(q.reshape(n, -1))
        assert lib().nh_paged_attention(C.byref(dev.kv), C.byref(rows), P(qd), n_head, 0.088, 0, 0, P(out), _stream()) == 0
        want, size = pm.attention(q, k, v, total - n, 0.088, 0, 0)
        bound = pm.attention_bound(size, hd, total, np.abs(v).max())
        assert np.abs(out.cpu().numpy().reshape(want.shape) - want).max() <= bound
    # an append and a read there
    x = [_cuda(rng.standard_normal((2, n_kv * hd)).astype(np.float32)) for _ in range(2)]
    cs = _cuda(pm.rope_table(hd, 400))
    rows, keep = dev.rows([2], [total])
    assert lib().nh_paged_append(C.byref(dev.kv), C.byref(rows), None, 0, P(x[0]), n_kv * hd, P(x[1]), n_kv * hd, None, None,
                                 EPS, n_head, P(cs), 400, None, _stream()) == 0
    ko, vo = (torch.empty(2, n_kv * hd, device="cuda") for _ in range(2))
    assert lib().nh_paged_read(C.byref(dev.kv), C.byref(rows), F32, P(ko), P(vo), _stream()) == 0
    sc = scales[1][order[2]].repeat_interleave(hd)
    assert (vo - x[1]).abs().le(sc / 2).all()
    assert int(dev.err.item()) == 0


@pytest.mark.parametrize("hd", [64, 128])
def test_attention_equal_calls_give_equal_bits(gpu, hd):
    """The warps and CTAs that share a row join what they have in an order that does not depend on which comes first."""
    import torch

    for n, p0 in (([1] * 3, [2000, 40, 777]), ([6, 3], [900, 31]), ([300, 7, 129], [500, 1200, 0]), ([64], [3000])):
        rng, table, cache, dev = _setup(n, p0, 16, 4, hd, 16, 31)
        q = _cuda(rng.standard_normal((sum(n), 16 * hd)).astype(np.float32) * 4)
        rows, keep = dev.rows(n, p0)
        outs = []
        for _ in range(12):
            out = torch.empty_like(q)
            assert lib().nh_paged_attention(C.byref(dev.kv), C.byref(rows), P(q), 16, 0.1, 600, 3, P(out), _stream()) == 0
            outs.append(out)
        torch.cuda.synchronize()
        assert all(torch.equal(outs[0], o) for o in outs[1:]), n


def test_two_streams_at_once(gpu):
    """Calls on two streams over caches of their own, with nothing shared, give what they give alone."""
    import torch

    cases = []
    for seed, n, p0 in ((1, [1] * 6, [700, 20, 300, 5, 90, 411]), (2, [200, 1, 90], [60, 500, 0])):
        rng, table, cache, dev = _setup(n, p0, 8, 4, 128, 32, seed)
        q = _cuda(rng.standard_normal((sum(n), 8 * 128)).astype(np.float32))
        rows, keep = dev.rows(n, p0)
        cases.append((dev, rows, keep, q))
    streams = [torch.cuda.Stream() for _ in cases]

    def call(c, s):
        dev, rows, keep, q = c
        with torch.cuda.stream(s):
            out = torch.empty_like(q)
            assert lib().nh_paged_attention(C.byref(dev.kv), C.byref(rows), P(q), 8, 0.09, 0, 0, P(out), _stream()) == 0
        return out

    alone = []
    for c, s in zip(cases, streams):
        s.wait_stream(torch.cuda.default_stream())
        alone.append(call(c, s))
        torch.cuda.synchronize()
    for _ in range(5):
        got = [call(c, s) for c, s in zip(cases, streams)]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, alone))


def test_attention_scales_far_apart(gpu):
    """Pages whose scales differ by many powers of two: the small ones' values must not disturb the large ones', nor
    overflow."""
    import torch

    n_head, n_kv, hd, page, total = 4, 2, 64, 16, 333
    for rows_n in (1, 150):
        rng, table, cache, dev = _setup([rows_n], [total - rows_n], n_head, n_kv, hd, page, 31)
        for w, (lo, hi) in enumerate(((-12, -6), (-60, 30))):
            s = np.exp2(rng.integers(lo, hi, cache.scales[w].shape).astype(np.float64)).astype(np.float32)
            cache.scales[w][:] = s
            dev.scales[w].copy_(_cuda(s))
        q = rng.standard_normal((rows_n, n_head, hd)).astype(np.float32)
        out = torch.empty(rows_n, n_head * hd, device="cuda")
        rows, keep = dev.rows([rows_n], [total - rows_n])
        qd = _cuda(q.reshape(rows_n, -1))
        assert lib().nh_paged_attention(C.byref(dev.kv), C.byref(rows), P(qd), n_head, 0.125, 0, 0, P(out),
                                        _stream()) == 0
        k, v = cache.values(0, table[0], total), cache.values(1, table[0], total)
        want, size = pm.attention(q, k, v, total - rows_n, 0.125, 0, 0)
        bound = pm.attention_bound(size, hd, total, np.abs(v).max())
        assert np.abs(out.cpu().numpy().reshape(want.shape) - want).max() <= bound


def test_bad_pages_and_sequences(gpu):
    """A page out of range is neither written nor seen; a sequence out of bounds is left alone; both are recorded."""
    import torch

    n_head, n_kv, hd, page = 4, 2, 64, 16
    n, p0 = [2, 3, 40], [30, 20, 50]
    rng, table, cache, dev = _setup(n, p0, n_head, n_kv, hd, page, 41)
    dev.table[0, 1] = -1                        # the rows' own page
    dev.table[2, 2] = cache.codes[0].shape[0]   # a page in the middle of the written ones and of the seen ones
    R, dkv = sum(n), n_kv * hd
    q, k, v = (_cuda(rng.standard_normal((R, w)).astype(np.float32)) for w in (n_head * hd, dkv, dkv))
    cs = _cuda(pm.rope_table(hd, 100))
    qr = torch.zeros(R, n_head * hd, device="cuda")
    before = dev.host()
    rc, keep = _append(dev, n, [30, 1 << 20, 30], q, k, v, None, None, cs, n_head, qr)
    assert rc == 0
    torch.cuda.synchronize()
    assert int(dev.err.item()) == NH_E_ARG
    after = dev.host()
    touched = {int(table[2][b]) for b in (1, 3, 4)}  # positions 30..69 without the missing page's 32..47
    for pg in range(before.codes[0].shape[0]):
        same = all(np.array_equal(after.codes[w][pg], before.codes[w][pg]) for w in range(2))
        assert same == (pg not in touched), pg
    assert torch.count_nonzero(qr[2:5]) == 0 and torch.count_nonzero(qr[:2]) > 0 and torch.count_nonzero(qr[5:]) > 0
    for rows_pos in ([30, 1 << 20, 50], [30, -1, 50]):
        dev.err.zero_()
        out = torch.full((R, n_head * hd), 7.0, device="cuda")
        rows, keep = dev.rows(n, rows_pos)
        assert lib().nh_paged_attention(C.byref(dev.kv), C.byref(rows), P(q), n_head, 0.125, 0, 0, P(out), _stream()) == 0
        torch.cuda.synchronize()
        assert int(dev.err.item()) == NH_E_ARG
        got = out.cpu().numpy()
        assert (got[2:5] == 7.0).all()
        c = dev.host()
        at = {0: 0, 2: 5}
        for s in (0, 2):
            total = n[s] + p0[s]
            pages = [int(x) for x in dev.table[s].cpu()]
            gone = [b for b in range((total + page - 1) // page) if not 0 <= pages[b] < c.codes[0].shape[0]]
            ok = [x if b not in gone else 0 for b, x in enumerate(pages)]
            kk, vv = c.values(0, ok, total), c.values(1, ok, total)
            keep_t = np.array([t // page not in gone for t in range(total)])
            qs = q.cpu().numpy()[at[s]:at[s] + n[s]].reshape(n[s], n_head, hd)
            for i in range(n[s]):
                sel = keep_t[:p0[s] + i + 1]
                w, size = pm.attention(qs[i:i + 1], kk[:p0[s] + i + 1][sel], vv[:p0[s] + i + 1][sel], sel.sum() - 1, 0.125,
                                       0, 0)
                err = np.abs(got[at[s] + i].reshape(n_head, hd) - w[0]).max()
                assert err <= pm.attention_bound(size, hd, total, np.abs(vv).max())
    # every page gone: zeros, and zeros read back
    dev.table.fill_(-5)
    for m in ([2, 3, 40], [2, 3, 4]):
        out = torch.full((sum(m), n_head * hd), 7.0, device="cuda")
        rows, keep = dev.rows(m, p0)
        assert lib().nh_paged_attention(C.byref(dev.kv), C.byref(rows), P(q), n_head, 0.125, 0, 0, P(out), _stream()) == 0
        assert torch.count_nonzero(out) == 0
        ko = torch.full((sum(m), dkv), 7.0, device="cuda")
        assert lib().nh_paged_read(C.byref(dev.kv), C.byref(rows), F32, P(ko), None, _stream()) == 0
        assert torch.count_nonzero(ko) == 0
    # one sequence alone, of many rows, past its pages
    dev.err.zero_()
    out = torch.full((R, n_head * hd), 7.0, device="cuda")
    rows, keep = dev.rows([R], [1 << 20])
    assert lib().nh_paged_attention(C.byref(dev.kv), C.byref(rows), P(q), n_head, 0.125, 0, 0, P(out), _stream()) == 0
    torch.cuda.synchronize()
    assert int(dev.err.item()) == NH_E_ARG and (out == 7.0).all()
    # more rows than the call's bounds say: left alone
    dev.err.zero_()
    out = torch.full((R, n_head * hd), 7.0, device="cuda")
    rows, keep = dev.rows(n, p0, max_rows=2)
    assert lib().nh_paged_attention(C.byref(dev.kv), C.byref(rows), P(q), n_head, 0.125, 0, 0, P(out), _stream()) == 0
    torch.cuda.synchronize()
    assert int(dev.err.item()) == NH_E_ARG and (out[2:] == 7.0).all() and torch.count_nonzero(out[:2]) == 0


def _verify_call(target, draft, ids, off, ua, up, max_draft=None):
    import torch

    n = len(off) - 1
    md = max_draft if max_draft is not None else int(max(np.diff(off)))
    t = [_cuda(target), None if draft is None else _cuda(draft), _cuda(ids.astype(np.int32)), _cuda(off.astype(np.int32)),
         _cuda(ua.astype(np.float32)), _cuda(up.astype(np.float32))]
    acc = torch.full((n,), -9, dtype=torch.int32, device="cuda")
    out = torch.full((n, md + 1), -7, dtype=torch.int32, device="cuda")
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    v = target.shape[1]
    d = NhVerifyDrafts(t[0].data_ptr(), v, None if draft is None else t[1].data_ptr(), v,
                       t[2].data_ptr() if len(ids) else None, t[3].data_ptr(), t[4].data_ptr() if len(ids) else None,
                       t[5].data_ptr(), n, len(ids), md, v, acc.data_ptr(), out.data_ptr(), err.data_ptr())
    assert lib().nh_verify_drafts(C.byref(d), _stream()) == NH_OK
    torch.cuda.synchronize()
    return acc.cpu().numpy(), out.cpu().numpy(), int(err.item())


def _probs(rng, rows, v, sharp):
    x = np.exp(sharp * rng.standard_normal((rows, v)))
    return (x / x.sum(1, keepdims=True)).astype(np.float32)


@pytest.mark.parametrize("v", [1, 2, 127, 1000, 4099, 50304, 131072])
@pytest.mark.parametrize("lookup", [False, True])
def test_verify_drafts(gpu, v, lookup):
    rng = np.random.default_rng(v)
    n_draft = np.array([3, 0, 1, 8, 4, 4, 5])
    off = np.concatenate([[0], np.cumsum(n_draft)])
    T, n = int(off[-1]), len(n_draft)
    target = _probs(rng, T + n, v, 2.0)
    rows = np.concatenate([np.arange(off[s], off[s + 1]) + s for s in range(n)])
    draft = target[rows] * np.exp(0.5 * rng.standard_normal((T, v))).astype(np.float32)
    draft /= draft.sum(1, keepdims=True)
    ids = np.array([rng.choice(v, p=r.astype(np.float64) / r.astype(np.float64).sum()) for r in draft])
    if lookup:
        draft, ids = None, target[rows].argmax(1)
    for seed in range(3):
        r2 = np.random.default_rng(seed)
        ua, up = r2.random(T).astype(np.float32) * (0.3 if lookup else 1.0), r2.random(n).astype(np.float32)
        if seed == 2:
            ua[:], up[:] = 0.0, [0.0, np.float32(1) - np.float32(2) ** -24, 1.0, 0.5, 0.0, 0.25, 0.75]
        acc, out, err = _verify_call(target, draft, ids, off, ua, up)
        want_acc, want = pm.verify(target, draft, ids, off, ua, up)
        assert list(acc) == want_acc
        assert err == 0
        for s in range(n):
            assert list(out[s, :acc[s] + 1]) == want[s], s
            assert (out[s, acc[s] + 1:] == -7).all()


def test_verify_edges(gpu):
    """A draft equal to the target that is refused, rows without mass, values that are no probabilities, ids and
    offsets out of range."""
    v = 300
    rng = np.random.default_rng(0)
    off = np.arange(0, 7)
    target = _probs(rng, 12, v, 1.0)
    draft = target[0::2].copy()
    ids = np.array([5, 6, 7, 8, v, -1])
    target[2 * 1 + 0, 6] = 0.0          # sequence 1: the drafted id has no mass
    target[2 * 2] = 0.0                 # sequence 2: a row without any
    target[2 * 3, :10] = [np.nan, -1, 0.1, 0, 0, 0, 0, 0, -0.5, 0]
    target[2 * 3, 10:] = np.nan
    draft[3, 2] = np.nan
    draft[0] = target[0]
    draft[0, 5] = 1.0                   # refused by u; nothing else left of the target
    ua, up = np.full(6, 0.999, np.float32), np.linspace(0.1, 0.9, 6).astype(np.float32)
    acc, out, err = _verify_call(target, draft, ids, off, ua, up)
    assert err == NH_E_ARG
    assert list(acc) == [0] * 6
    safe = np.where((ids < 0) | (ids >= v), 0, ids)
    want_acc, want = pm.verify(target, draft, safe, off, ua, up)
    for s in (0, 1, 3):
        assert out[s, 0] == want[s][0], s
    assert out[2, 0] == -1 and out[3, 0] == 2
    assert (out[:, 1] == -7).all()
    # offsets out of range: that sequence is left alone
    off = np.array([0, 3, 2, 50, 6, 6, 6])
    acc, out, err = _verify_call(target, draft, np.zeros(6), off, ua, up, max_draft=4)
    assert err == NH_E_ARG
    assert acc[0] >= 0 and list(acc[1:4]) == [-9, -9, -9] and (out[1:4] == -7).all() and acc[4] == 0 and acc[5] == 0


def _step_buffers(rng, n_head, n_kv, hd, R):
    return [_cuda(rng.standard_normal((R, w)).astype(np.float32)) for w in (n_head * hd, n_kv * hd, n_kv * hd)]


@pytest.mark.parametrize("captured", [False, True])
def test_serving_steps(gpu, captured):
    """A prompt chunk for each of three sequences, then steps of drafted rows whose positions move on by what the
    check accepts, on a stream of its own, as calls or as one captured graph that is replayed."""
    import torch

    n_head, n_kv, hd, page, V, K = 8, 4, 64, 16, 997, 3
    prompt = [70, 5, 33]
    steps = 6
    rng, table, cache, dev = _setup([p + steps * (K + 1) for p in prompt], [0] * 3, n_head, n_kv, hd, page, 77)
    qn, kn = (_cuda(rng.uniform(0.5, 1.5, w).astype(np.float32)) for w in (n_head * hd, n_kv * hd))
    cs_h = pm.rope_table(hd, 200)
    cs = _cuda(cs_h)
    model = cache.copy()
    stream = torch.cuda.Stream()
    L = lib()
    with torch.cuda.stream(stream):
        q, k, v = _step_buffers(rng, n_head, n_kv, hd, sum(prompt))
        qr, out = torch.empty_like(q), torch.empty_like(q)
        stream.wait_stream(torch.cuda.default_stream())
        rc, keep = _append(dev, prompt, [0] * 3, q, k, v, qn, kn, cs, n_head, qr)
        assert rc == 0
        rows, keep2 = dev.rows(prompt, [0] * 3)
        assert L.nh_paged_attention(C.byref(dev.kv), C.byref(rows), P(qr), n_head, 0.125, 40, 4, P(out), _stream()) == 0
    stream.synchronize()

    def model_append(n, p0, k, v):
        pos = np.concatenate([np.arange(b, b + a) for a, b in zip(n, p0)])
        kr = pm.rotated_keys(k, kn.cpu().numpy(), pos, cs_h, n_kv, EPS)
        at = 0
        for s in range(3):
            for w, x in enumerate((kr, v.reshape(-1, n_kv, hd))):
                model.append(w, table[s], p0[s], x[at:at + n[s]])
            at += n[s]

    def check(n, p0, qr, out):
        at = 0
        for s in range(3):
            total = n[s] + p0[s]
            kk, vv = model.values(0, table[s], total), model.values(1, table[s], total)
            want, size = pm.attention(qr[at:at + n[s]].reshape(n[s], n_head, hd), kk, vv, p0[s], 0.125, 40, 4)
            err = np.abs(out[at:at + n[s]].reshape(want.shape) - want).max()
            assert err <= pm.attention_bound(size, hd, total, np.abs(vv).max())
            at += n[s]

    model_append(prompt, [0] * 3, k.cpu().numpy(), v.cpu().numpy())
    check(prompt, [0] * 3, qr.cpu().numpy(), out.cpu().numpy())

    # steps of K + 1 rows
    n = [K + 1] * 3
    R = sum(n)
    with torch.cuda.stream(stream):
        q, k, v = (torch.zeros(R, w, device="cuda") for w in (n_head * hd, n_kv * hd, n_kv * hd))
        qr, out = torch.empty_like(q), torch.empty_like(q)
        rows, (off_d, pos_d) = dev.rows(n, prompt)
        probs = torch.zeros(R, V, device="cuda")
        doff = torch.tensor([0, K, 2 * K, 3 * K], dtype=torch.int32, device="cuda")
        ids = torch.zeros(3 * K, dtype=torch.int32, device="cuda")
        ua, up = torch.zeros(3 * K, device="cuda"), torch.zeros(3, device="cuda")
        acc = torch.zeros(3, dtype=torch.int32, device="cuda")
        got = torch.zeros(3, K + 1, dtype=torch.int32, device="cuda")
    stream.synchronize()
    vd = NhVerifyDrafts(probs.data_ptr(), V, None, V, ids.data_ptr(), doff.data_ptr(), ua.data_ptr(), up.data_ptr(), 3,
                        3 * K, K, V, acc.data_ptr(), got.data_ptr(), dev.err.data_ptr())

    def step():
        s = _stream()
        assert L.nh_paged_append(C.byref(dev.kv), C.byref(rows), P(q), n_head * hd, P(k), n_kv * hd, P(v), n_kv * hd,
                                 P(qn), P(kn), EPS, n_head, P(cs), 200, P(qr), s) == 0
        assert L.nh_paged_attention(C.byref(dev.kv), C.byref(rows), P(qr), n_head, 0.125, 40, 4, P(out), s) == 0
        assert L.nh_verify_drafts(C.byref(vd), s) == 0

    graph = None
    pos = list(prompt)
    for i in range(steps):
        with torch.cuda.stream(stream):
            for t, x in zip((q, k, v), _step_buffers(rng, n_head, n_kv, hd, R)):
                t.copy_(x)
            tp = _probs(rng, R, V, 1.0)
            d = rng.integers(0, V, 3 * K)
            for s in range(3):
                for j in range(K):
                    tp[s * (K + 1) + j, d[s * K + j]] += 1.0  # likely
            probs.copy_(_cuda(tp))
            ids.copy_(_cuda(d.astype(np.int32)))
            ua.copy_(_cuda(rng.random(3 * K).astype(np.float32) * 1.6))
            up.copy_(_cuda(rng.random(3).astype(np.float32)))
            pos_d.copy_(_cuda(np.array(pos, np.int32)))
        stream.synchronize()
        with torch.cuda.stream(stream):
            if not captured:
                step()
            else:
                if i == 0:
                    step()  # the first call outside the capture; the replay repeats it
                    stream.synchronize()
                    graph = torch.cuda.CUDAGraph()
                    with torch.cuda.graph(graph, stream=stream):
                        step()
                graph.replay()
        stream.synchronize()
        assert int(dev.err.item()) == 0
        model_append(n, pos, k.cpu().numpy(), v.cpu().numpy())
        h = dev.host()
        for s in range(3):
            total = pos[s] + n[s]
            for w in range(2):
                assert np.array_equal(h.values(w, table[s], total), model.values(w, table[s], total))
        check(n, pos, qr.cpu().numpy(), out.cpu().numpy())
        want_acc, want = pm.verify(tp, None, d, np.arange(0, 3 * K + 1, K), ua.cpu().numpy(), up.cpu().numpy())
        assert acc.cpu().tolist() == want_acc
        for s in range(3):
            assert got[s, :want_acc[s] + 1].cpu().tolist() == want[s]
            pos[s] += want_acc[s] + 1  # the refused drafts' positions are written again
    del graph
