"""The paged 8-bit K/V cache and the draft check in numpy, for the tests: the
formulas of nh_kernels.h in 64 bits (the rotated q in the kernels' f32 steps,
each a correctly rounded IEEE operation; K's rows rounded to f32 once, so that
codes can be compared bit for bit)."""
from __future__ import annotations

import ctypes as C

import numpy as np

from nuthatch_b200._lib import NhPagedKv, NhPagedRows, lib

F = np.float32


def rope_table(hd: int, n: int) -> np.ndarray:
    cs = np.zeros(n * hd, dtype=F)
    lib().nh_rope_table(10000.0, hd, n, cs.ctypes.data_as(C.POINTER(C.c_float)))
    return cs.reshape(n, hd // 2, 2)


def rotated_rows(x: np.ndarray, w, pos: np.ndarray, cs: np.ndarray, heads: int, eps: float) -> np.ndarray:
    """RMSNorm over the full width (w None: none) and NEOX rotation, in f32 steps with the sum of squares in f64."""
    n, hd = x.shape[0], x.shape[1] // heads
    x = x.astype(F)
    if w is not None:
        mean = ((x * x).astype(np.float64).sum(1) / x.shape[1]).astype(F)
        inv = F(1) / np.sqrt(mean + F(eps))
        x = (x * inv[:, None]) * w.astype(F)
    x = x.reshape(n, heads, 2, hd // 2)
    c, s = cs[pos][:, None, :, 0], cs[pos][:, None, :, 1]
    lo = x[:, :, 0] * c - x[:, :, 1] * s
    hi = x[:, :, 0] * s + x[:, :, 1] * c
    return np.concatenate([lo, hi], -1)  # [n][heads][hd]


def rotated_keys(x: np.ndarray, w, pos: np.ndarray, cs: np.ndarray, heads: int, eps: float) -> np.ndarray:
    """The same in f64, rounded to f32 at the end."""
    n, hd = x.shape[0], x.shape[1] // heads
    x = x.astype(np.float64)
    if w is not None:
        x = x / np.sqrt((x * x).mean(1, keepdims=True) + np.float64(F(eps))) * w.astype(np.float64)
    x = x.reshape(n, heads, 2, hd // 2)
    c, s = (cs[pos][:, None, :, i].astype(np.float64) for i in range(2))
    return np.concatenate([x[:, :, 0] * c - x[:, :, 1] * s, x[:, :, 0] * s + x[:, :, 1] * c], -1).astype(F)


def scale_for(m: float) -> float:
    e = np.frexp(np.float64(m))[1] - 1 if m > 0 else -1000
    return 2.0 ** (max(int(e), -100) - 6)


class Cache:
    """Codes [n_pages][n_kv][page][hd] and scales [n_pages][n_kv], for K (0) and V (1)."""

    def __init__(self, n_pages, n_kv, page, hd, rng):
        self.n_kv, self.page, self.hd = n_kv, page, hd
        self.codes = [rng.integers(0, 256, (n_pages, n_kv, page, hd), dtype=np.uint8) for _ in range(2)]
        self.scales = [np.exp2(rng.integers(-8, -3, (n_pages, n_kv)).astype(np.float64)).astype(F) for _ in range(2)]

    def copy(self):
        c = object.__new__(Cache)
        c.n_kv, c.page, c.hd = self.n_kv, self.page, self.hd
        c.codes, c.scales = [x.copy() for x in self.codes], [x.copy() for x in self.scales]
        return c

    def append(self, which, pages, p0, rows):
        """rows [n][n_kv][hd] at positions p0.. of the sequence with these pages, one position after the other."""
        codes, scales = self.codes[which], self.scales[which]
        for i, row in enumerate(rows):
            b, t = divmod(p0 + i, self.page)
            pg = pages[b]
            for h in range(self.n_kv):
                need = scale_for(float(np.abs(row[h]).max()))
                old = float(scales[pg, h])
                if t == 0:
                    sc = need
                else:
                    sc = max(old, need)
                    if sc > old:
                        held = codes[pg, h, :t].astype(np.int64) - 128
                        codes[pg, h, :t] = np.floor(held * (old / sc)) + 128
                scales[pg, h] = sc
                codes[pg, h, t] = np.clip(np.floor(row[h].astype(np.float64) / sc) + 128, 0, 255)

    def values(self, which, pages, n):
        """[n][n_kv][hd] in f64: positions 0..n-1 of the sequence."""
        nb = (n + self.page - 1) // self.page
        pg = np.asarray(pages[:nb], dtype=np.int64)
        v = (self.codes[which][pg].astype(np.float64) - 127.5) * self.scales[which][pg].astype(np.float64)[..., None, None]
        return v.transpose(0, 2, 1, 3).reshape(nb * self.page, self.n_kv, self.hd)[:n]


def attention(q, k, v, p0, scale, window, sinks):
    """q [n][heads][hd] at positions p0.. over k, v [p0+n][n_kv][hd], in f64; with it, for the error bounds, the
    largest sum of the magnitudes of a row's products, scaled."""
    n, heads, hd = q.shape
    group = heads // k.shape[1]
    q = q.astype(np.float64)
    kk, vv = np.repeat(k, group, 1), np.repeat(v, group, 1)
    s = np.einsum("nhd,thd->hnt", q, kk) * scale
    size = np.einsum("nhd,thd->hnt", np.abs(q), np.abs(kk)).max() * abs(scale) if k.shape[0] else 0.0
    at, t = np.arange(p0, p0 + n)[:, None], np.arange(k.shape[0])[None]
    seen = t <= at
    if window > 0:
        seen &= (t > at - window) | (t < sinks)
    s = np.where(seen[None], s, -np.inf)
    w = np.exp(s - s.max(-1, keepdims=True))
    w /= w.sum(-1, keepdims=True)
    return np.einsum("hnt,thd->nhd", w, vv), float(size)


def attention_bound(size, hd, n_keys, v_max):
    """Worst case for f32 arithmetic with e = 2^-24: a score is a sum of hd products whose factors carry 22 bits at
    least, so it is off by (hd + 16) e size; a weight by twice that (its own score and the maximum) and 8 e (1 + size)
    for the scaled argument and the exponential; the two sums over the keys by n_keys e each."""
    e = 2.0 ** -24
    return v_max * (2 * (hd + 16) * e * size + 16 * e * (1 + size) + 2 * (n_keys + 16) * e)


class Device:
    """A cache, its page table and the rows of a call in device memory."""

    def __init__(self, cache: Cache, table: np.ndarray):
        import torch

        self.torch, self.cache = torch, cache
        self.codes = [torch.from_numpy(x.copy()).cuda() for x in cache.codes]
        self.scales = [torch.from_numpy(x.copy()).cuda() for x in cache.scales]
        self.table = torch.from_numpy(table.astype(np.int32)).cuda()
        self.err = torch.zeros(1, dtype=torch.int32, device="cuda")
        self.kv = NhPagedKv(self.codes[0].data_ptr(), self.codes[1].data_ptr(), self.scales[0].data_ptr(),
                            self.scales[1].data_ptr(), cache.codes[0].shape[0], cache.page, cache.n_kv, cache.hd)

    def rows(self, n, p0, max_rows=None, n_rows=None, offset=0):
        off = np.concatenate([[0], np.cumsum(n)]).astype(np.int32) + offset
        off_d = self.torch.from_numpy(off.astype(np.int32)).cuda()
        pos_d = self.torch.from_numpy(np.asarray(p0, dtype=np.int32)).cuda()
        r = NhPagedRows(len(n), max(n) if max_rows is None else max_rows, int(off[-1]) if n_rows is None else n_rows,
                        self.table.shape[1], off_d.data_ptr(), pos_d.data_ptr(), self.table.data_ptr(),
                        self.err.data_ptr())
        return r, (off_d, pos_d)

    def host(self) -> Cache:
        c = self.cache.copy()
        c.codes = [x.cpu().numpy() for x in self.codes]
        c.scales = [x.cpu().numpy() for x in self.scales]
        return c


def verify(target, draft, ids, off, u_accept, u_pick):
    """(n_accept, list of id lists) by the definition in f64."""
    n_accept, out = [], []
    mass = lambda x: np.where(x > 0, x, 0).astype(np.float64)  # noqa: E731
    for s in range(len(off) - 1):
        o, n = int(off[s]), int(off[s + 1] - off[s])
        a = 0
        while a < n:
            i = int(ids[o + a])
            q = 1.0 if draft is None else float(mass(draft[o + a, i]))
            if not float(u_accept[o + a]) * q < float(mass(target[o + s + a, i])):
                break
            a += 1
        p = mass(target[o + s + a])
        r = p.copy()
        if a < n:
            if draft is None:
                r[int(ids[o + a])] = 0.0
            else:
                r = np.maximum(p - mass(draft[o + a]), 0)
        if not r.sum() > 0:
            r = p
        c = np.cumsum(r)
        hit = np.nonzero((c > float(u_pick[s]) * c[-1]) & (r > 0))[0]
        have = np.nonzero(r > 0)[0]
        pick = int(hit[0]) if hit.size else (int(have[-1]) if have.size else -1)
        n_accept.append(a)
        out.append([int(x) for x in ids[o:o + a]] + [pick])
    return n_accept, out
