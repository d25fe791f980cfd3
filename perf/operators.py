"""Cases of the paged 8-bit KV cache and of draft verification: appending
rotated keys and values to the cache, attention over it, and checking drafted
tokens against the target's probabilities.

The cache holds a sequence's positions in pages of `page` tokens.  A page keeps
unsigned 8-bit codes [n_kv][page][hd] and one scale, a power of two, for each
KV head (keys and values apart); code u stands for (u - 127.5) * scale.
"""
import ctypes
import math
import random

import torch

own = False

EPS = 1e-5
ROPE_BASE = 10000.0
NH_TYPE_BF16 = 30


# ------------------------------------------------------------------ the cases
def _append(name, n_seq, rows, pos, heads, page):
    n_head, n_kv, hd = heads
    return {"name": name, "op": "append", "n_seq": n_seq, "rows": rows, "len": pos, "n_head": n_head, "n_kv": n_kv,
            "hd": hd, "page": page, "mix": 1}


def _attend(name, n_seq, rows, length, heads, page, window=0, sinks=0):
    n_head, n_kv, hd = heads
    return {"name": name, "op": "attend", "n_seq": n_seq, "rows": rows, "len": length, "n_head": n_head,
            "n_kv": n_kv, "hd": hd, "page": page, "window": window, "sinks": sinks, "mix": 2}


def _verify(name, n_seq, drafts, n_vocab, lookup):
    return {"name": name, "op": "verify", "n_seq": n_seq, "drafts": drafts, "n_vocab": n_vocab, "lookup": lookup,
            "mix": 3}


def listed():
    full, grouped, small = (16, 16, 128), (32, 8, 128), (16, 8, 64)
    return [
        # the append of one decode step of one sequence: latency
        _append("append one token", 1, 1, 1000, full, 16),
        # the append of one decode step of a serving batch
        _append("append decode batch", 64, 1, 4000, full, 16),
        # a chunk of several prompts of unequal lengths, some of them continued inside a page
        _append("append prompt chunks", 16, 600, 777, full, 32),
        # one decode step of one short conversation: latency
        _attend("attend short", 1, 1, 300, full, 16),
        # one decode step of a serving batch of unequal lengths up to the model's context
        _attend("attend decode batch", 64, 1, 4096, full, 16),
        # one decode step over one very long document
        _attend("attend one long", 1, 1, 131001, full, 64),
        # a step that verifies up to four drafted tokens a sequence, grouped heads
        _attend("attend drafted rows", 16, 5, 6001, grouped, 32),
        # the second chunk of a long prompt
        _attend("attend prompt chunk", 1, 2048, 4096, full, 64),
        # whole prompts of unequal lengths under a sliding window with four sinks, grouped narrow heads
        _attend("attend windowed prompts", 4, 4000, 4000, small, 16, 1024, 4),
        # one sequence's four drafts: latency
        _verify("verify one", 1, 4, 50304, False),
        # a serving batch's drafts from a draft model
        _verify("verify batch", 64, 5, 50304, False),
        # a larger batch whose drafts come from looking up the prompt (no draft probabilities)
        _verify("verify lookup batch", 256, 7, 50304, True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "append", "decode", "decode", "drafted", "prompt", "prompt", "verify", "verify"])
    mix = rng.randrange(1 << 20)
    if kind == "verify":
        drafts = rng.randint(1, 8)
        vocab = _log(rng, 1000, 131072)
        n_seq = _log(rng, 1, max(1, min(256, 100_000_000 // (vocab * (drafts + 1)))))
        return {"op": "verify", "n_seq": n_seq, "drafts": drafts, "n_vocab": vocab, "lookup": rng.random() < 0.3,
                "mix": mix}
    n_kv = rng.choice([1, 2, 4, 8, 16])
    group = rng.choice([1, 1, 2, 3, 4, 8])
    while n_kv * group > 64:
        group = rng.choice([1, 2, 4])
    c = {"n_head": n_kv * group, "n_kv": n_kv, "hd": rng.choice([32, 64, 96, 128, 128]),
         "page": rng.choice([16, 32, 64, 128]), "mix": mix}
    wide = n_kv * c["hd"]
    if kind == "append":
        if rng.random() < 0.5:
            return dict(c, op="append", n_seq=_log(rng, 1, 128), rows=rng.randint(1, 6), len=_log(rng, 8, 8000))
        rows = _log(rng, 17, 2000)
        return dict(c, op="append", n_seq=_log(rng, 1, max(1, min(16, 9000 // rows))), rows=rows,
                    len=_log(rng, rows, rows + 1500))
    if kind == "prompt":
        rows = _log(rng, 20, 2048)
        length = _log(rng, rows, 2 * rows + 1000)
        most = 16 * 2048 * 3100 // (rows * length * c["n_head"])
        n_seq = _log(rng, 1, max(1, min(8, most)))
        while n_seq * rows * length * c["n_head"] > 16 * 2048 * 3100:
            rows, length = rows // 2 + 1, length // 2 + 1
    else:
        rows = 1 if kind == "decode" else rng.randint(2, 8)
        n_seq = _log(rng, 1, 64)
        most = max(64, min(131072, 260_000_000 // (wide * n_seq), 400_000_000 // (wide * n_seq)))
        length = _log(rng, 40, most)
    window, sinks = 0, 0
    if rng.random() < 0.35:
        window = _log(rng, 16, max(17, length))
        sinks = rng.choice([0, 1, 4, 19])
    return dict(c, op="attend", n_seq=n_seq, rows=rows, len=max(length, rows), window=window, sinks=sinks)


def _shape(case):
    """Rows of each sequence in this call, and its positions in the cache before them (the same for every seed)."""
    rng = random.Random(case["mix"])
    rows, first = [], []
    for s in range(case["n_seq"]):
        n = case["rows"] if s == 0 else rng.randint((case["rows"] + 1) // 2, case["rows"])
        total = case["len"] if s == 0 else rng.randint(max(n, case["len"] // 4), max(n, case["len"]))
        if case["op"] == "append":  # `len` positions at most are there before the rows
            total += n
        rows.append(n)
        first.append(max(0, total - n))
    return rows, first


def _drafts(case):
    rng = random.Random(case["mix"])
    return [case["drafts"] if s == 0 else rng.randint((case["drafts"] + 1) // 2, case["drafts"])
            for s in range(case["n_seq"])]


def work(case):
    if case["op"] == "verify":
        # What every sequence needs whole: the target's row that the last token is drawn from and, for the part that
        # ends in a rejection (taken as half), the draft's row beside it.
        n, v = case["n_seq"], case["n_vocab"]
        rows = n * (1.0 if case["lookup"] else 1.5)
        return {"bytes": rows * v * 4 + sum(_drafts(case)) * 16, "flops": 3.0 * n * v}
    rows, first = _shape(case)
    dq, dkv = case["n_head"] * case["hd"], case["n_kv"] * case["hd"]
    if case["op"] == "append":
        n = sum(rows)
        back = sum(p + r - p // case["page"] * case["page"] for r, p in zip(rows, first))  # positions read back
        return {"bytes": n * (2 * dq * 4 + 2 * dkv * 4 + 2 * dkv) + back * 2 * dkv * 3, "flops": 8.0 * n * (dq + dkv)}
    w, k = case["window"], case["sinks"]
    pairs, keys = 0, 0
    for n, p in zip(rows, first):
        for i in range(p, p + n):
            low = max(0, i - w + 1) if w else 0
            pairs += i + 1 - low + min(k if w else 0, low)
        low = max(0, p - w + 1) if w else 0
        keys += p + n - low + min(k if w else 0, low)
    n = sum(rows)
    return {"bytes": keys * 2 * dkv + n * 2 * dq * 4, "flops": 4.0 * pairs * case["n_head"] * case["hd"]}


# ------------------------------------------------------------------ inputs
def _blocks(total, page):
    return [(t + page - 1) // page for t in total]


def _code(x, page_dim=-2):
    """Codes and scale of whole pages x [..., page, hd]."""
    _, e = torch.frexp(x.abs().amax(dim=(-2, -1)))
    scale = torch.ldexp(torch.ones_like(x[..., 0, 0]), e - 7)
    u = torch.floor(x / scale[..., None, None]) + 128
    return u.clamp(0, 255).to(torch.uint8), scale


def _cache(case, total, gen, dev):
    """Pages of every sequence at shuffled places of the pool, filled with keys and values of a trained model's kind:
    channels of unequal size, tokens of unequal size."""
    page, n_kv, hd = case["page"], case["n_kv"], case["hd"]
    blocks = _blocks(total, page)
    n_pages, most = sum(blocks) + 3, max(blocks)
    codes, scales = [], []
    for _ in range(2):
        c = torch.empty(n_pages, n_kv, page, hd, dtype=torch.uint8, device=dev)
        s = torch.empty(n_pages, n_kv, dtype=torch.float32, device=dev)
        chan = torch.exp(0.5 * torch.randn(n_kv, 1, hd, generator=gen, device=dev))
        for a in range(0, n_pages, 1024):
            b = min(n_pages, a + 1024)
            x = torch.randn(b - a, n_kv, page, hd, generator=gen, device=dev) * chan
            x *= torch.exp(0.2 * torch.randn(b - a, n_kv, page, 1, generator=gen, device=dev))
            c[a:b], s[a:b] = _code(x)
        codes.append(c)
        scales.append(s)
    order = torch.randperm(n_pages, generator=gen, device=dev).to(torch.int32)
    table = torch.zeros(len(total), most, dtype=torch.int32, device=dev)
    at = 0
    for s, n in enumerate(blocks):
        table[s, :n] = order[at:at + n]
        at += n
    return {"k_codes": codes[0], "v_codes": codes[1], "k_scales": scales[0], "v_scales": scales[1], "table": table}


def _ints(v, dev):
    return torch.tensor(v, dtype=torch.int32, device=dev)


def _offsets(v):
    out = [0]
    for x in v:
        out.append(out[-1] + x)
    return out


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed * 7919 + 11)
    st = {"case": dict(case)}
    if case["op"] == "verify":
        n_draft = _drafts(case)
        off, v, total = _offsets(n_draft), case["n_vocab"], sum(n_draft)
        n = case["n_seq"]
        rows = total + n
        target = torch.randn(rows, v, generator=gen, device=dev).mul_(3.0)
        # each draft row is its target row with noise; row i of sequence s is target row off[s] + s + i
        pick = torch.tensor([off[s] + s + i for s in range(n) for i in range(n_draft[s])], device=dev)
        noise = torch.rand(total, v, generator=gen, device=dev).clamp_(1e-20, 1.0)
        noise = -torch.log(-torch.log(noise))  # Gumbel: its argmax on top of the logits is a draw from them
        draft = target[pick] + torch.randn(total, v, generator=gen, device=dev).mul_(0.7)
        st["ids"] = (draft + noise).argmax(dim=-1).to(torch.int32)
        del noise
        if case["lookup"]:  # text that repeats: the drafted token is likely, most of the time
            target[pick, st["ids"].long()] += 12.0 * (torch.rand(total, generator=gen, device=dev) < 0.7)
        st["draft"] = None if case["lookup"] else torch.softmax(draft, dim=-1)
        st["target"] = torch.softmax(target, dim=-1)
        st["u_accept"] = torch.rand(total, generator=gen, device=dev)
        st["u_pick"] = torch.rand(n, generator=gen, device=dev)
        st["off"] = _ints(off, dev)
        st["n_accept"] = torch.zeros(n, dtype=torch.int32, device=dev)
        st["out_ids"] = torch.full((n, max(n_draft) + 1), -1, dtype=torch.int32, device=dev)
        st["most"] = max(n_draft)
    else:
        rows, first = _shape(case)
        page, hd = case["page"], case["hd"]
        dq, dkv = case["n_head"] * hd, case["n_kv"] * hd
        total = [r + p for r, p in zip(rows, first)]
        st["kv"] = _cache(case, total, gen, dev)
        st["off"], st["pos0"] = _ints(_offsets(rows), dev), _ints(first, dev)
        st["n"], st["most"] = sum(rows), max(rows)
        n = st["n"]
        if case["op"] == "append":
            st["q"] = torch.randn(n, dq, generator=gen, device=dev)
            st["k"] = torch.randn(n, dkv, generator=gen, device=dev) * 1.5
            st["v"] = torch.randn(n, dkv, generator=gen, device=dev) * 0.6
            st["q_norm"] = torch.rand(dq, generator=gen, device=dev) + 0.5
            st["k_norm"] = torch.rand(dkv, generator=gen, device=dev) + 0.5
            i = torch.arange(hd // 2, dtype=torch.float64, device=dev)
            angle = torch.arange(max(total), dtype=torch.float64, device=dev)[:, None] * ROPE_BASE ** (-2 * i / hd)
            st["rope"] = torch.stack([angle.cos(), angle.sin()], dim=-1).float().contiguous()
            st["qr"] = torch.empty(n, dq, device=dev)
            # the positions read back: from the start of the first page that is written
            start = [p // page * page for p in first]
            back = [t - s for t, s in zip(total, start)]
            st["back_off"], st["back_pos"] = _ints(_offsets(back), dev), _ints(start, dev)
            st["back_n"], st["back_most"] = sum(back), max(back)
            st["k_back"] = torch.empty(sum(back), dkv, dtype=torch.bfloat16, device=dev)
            st["v_back"] = torch.empty(sum(back), dkv, dtype=torch.bfloat16, device=dev)
        else:
            st["q"] = torch.randn(n, dq, generator=gen, device=dev)
            st["out"] = torch.empty(n, dq, device=dev)
    if own:
        st["own"] = _handles(st)
    return st


# ------------------------------------------------------------------ the framework's calls
def _handles(st):
    """The argument blocks that a program keeps: pointers and sizes of the buffers above."""
    from nuthatch_b200 import _lib

    p = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    c, lib = st["case"], _lib.lib()
    if c["op"] == "verify":
        d = _lib.NhVerifyDrafts(
            target=p(st["target"]), target_stride=c["n_vocab"], draft=p(st["draft"]), draft_stride=c["n_vocab"],
            draft_ids=p(st["ids"]), draft_off=p(st["off"]), u_accept=p(st["u_accept"]), u_pick=p(st["u_pick"]),
            n_seq=c["n_seq"], n_drafts=st["ids"].numel(), max_draft=st["most"], n_vocab=c["n_vocab"], n_accept=p(st["n_accept"]),
            out_ids=p(st["out_ids"]), err=None)
        return lib, ctypes.byref(d), d
    kv = st["kv"]
    cache = _lib.NhPagedKv(
        k_codes=p(kv["k_codes"]), v_codes=p(kv["v_codes"]), k_scales=p(kv["k_scales"]), v_scales=p(kv["v_scales"]),
        n_pages=kv["k_codes"].shape[0], page_size=c["page"], n_head_kv=c["n_kv"], head_dim=c["hd"])

    def rows(off, pos, n, most):
        return _lib.NhPagedRows(n_seq=c["n_seq"], max_rows=most, n_rows=n, max_blocks=kv["table"].shape[1],
                                row_off=p(off), pos0=p(pos), page_table=p(kv["table"]), err=None)

    r = rows(st["off"], st["pos0"], st["n"], st["most"])
    back = rows(st["back_off"], st["back_pos"], st["back_n"], st["back_most"]) if c["op"] == "append" else r
    return lib, ctypes.byref(cache), ctypes.byref(r), ctypes.byref(back), cache, r, back


def _checked(rc):
    if rc != 0:
        raise RuntimeError("the call returned %d" % rc)


def _run_own(st):
    c, h = st["case"], st["own"]
    lib, stream = h[0], torch.cuda.current_stream().cuda_stream
    if c["op"] == "verify":
        _checked(lib.nh_verify_drafts(h[1], stream))
        return {"n_accept": st["n_accept"], "ids": st["out_ids"]}
    if c["op"] == "append":
        dq, dkv = c["n_head"] * c["hd"], c["n_kv"] * c["hd"]
        _checked(lib.nh_paged_append(
            h[1], h[2], st["q"].data_ptr(), dq, st["k"].data_ptr(), dkv, st["v"].data_ptr(), dkv,
            st["q_norm"].data_ptr(), st["k_norm"].data_ptr(), EPS, c["n_head"], st["rope"].data_ptr(),
            st["rope"].shape[0], st["qr"].data_ptr(), stream))
        _checked(lib.nh_paged_read(h[1], h[3], NH_TYPE_BF16, st["k_back"].data_ptr(), st["v_back"].data_ptr(), stream))
        return {"qr": st["qr"], "k": st["k_back"], "v": st["v_back"]}
    _checked(lib.nh_paged_attention(h[1], h[2], st["q"].data_ptr(), c["n_head"], 1.0 / math.sqrt(c["hd"]), c["window"],
                                    c["sinks"], st["out"].data_ptr(), stream))
    return {"out": st["out"]}


# ------------------------------------------------------------------ the plain forms
def _row_index(off, n):
    """Sequence of each row, and the row's place among its sequence's."""
    per = (off[1:] - off[:-1]).long()
    seq = torch.repeat_interleave(torch.arange(per.numel(), device=off.device), per, output_size=n)
    return seq, torch.arange(n, device=off.device) - off.long()[seq]


def _values(kv, which, pages):
    """What the codes of `pages` stand for, in float32 [..., n_kv, page, hd]."""
    return (kv[which + "_codes"][pages].float() - 127.5) * kv[which + "_scales"][pages][..., None, None]


def _plain_append(st):
    c, kv = st["case"], st["kv"]
    n, page, hd, h, g = st["n"], c["page"], c["hd"], c["n_kv"], c["n_head"]
    seq, i = _row_index(st["off"], n)
    pos = st["pos0"].long()[seq] + i
    cos, sin = st["rope"].double()[pos].unbind(-1)

    # In 64 bits: what stands next to a code's border must not cross it.
    def turn(x, w, heads):
        x = x.double()
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.double()
        a, b = x.view(n, heads, 2, hd // 2).unbind(2)
        return torch.cat([a * cos[:, None] - b * sin[:, None], a * sin[:, None] + b * cos[:, None]], -1).float()

    qr = turn(st["q"], st["q_norm"], g).view(n, g * hd)
    first = st["pos0"].long()
    block, slot = torch.div(pos, page, rounding_mode="floor"), pos % page
    where = kv["table"].long()[seq, block]  # each row's page
    held = first % page  # positions of a sequence's first written page that are there already
    head_page = kv["table"].long()[torch.arange(first.numel(), device=first.device), torch.div(first, page, rounding_mode="floor")]
    for name, x in (("k", turn(st["k"], st["k_norm"], h)), ("v", st["v"].view(n, h, hd))):
        codes, scales = kv[name + "_codes"], kv[name + "_scales"]
        big = torch.zeros_like(scales).scatter_reduce_(0, where[:, None].expand(-1, h), x.abs().amax(-1), "amax")
        need = torch.ldexp(torch.ones_like(big), torch.frexp(big)[1] - 7)
        old = scales[head_page]
        # a first page keeps its scale unless the new rows need a larger one; a page begun here starts afresh
        now = torch.where((held > 0)[:, None], torch.maximum(need[head_page], old), need[head_page])
        fell = (torch.log2(now) - torch.log2(old)).clamp(0, 31).to(torch.int32)
        kept = torch.arange(page, device=held.device) < held[:, None]
        moved = ((codes[head_page].to(torch.int32) - 128) >> fell[:, :, None, None]) + 128
        codes[head_page] = torch.where(kept[:, None, :, None], moved.to(torch.uint8), codes[head_page])
        scales[where] = need[where]
        scales[head_page] = now
        u = torch.floor(x / scales[where][:, :, None]) + 128
        codes[where, :, slot] = u.clamp(0, 255).to(torch.uint8)
    seq, i = _row_index(st["back_off"], st["back_n"])
    pos = st["back_pos"].long()[seq] + i
    where = kv["table"].long()[seq, torch.div(pos, page, rounding_mode="floor")]
    out = {"qr": qr}
    for name in ("k", "v"):
        x = (kv[name + "_codes"][where, :, pos % page].float() - 127.5) * kv[name + "_scales"][where][:, :, None]
        out[name] = x.to(torch.bfloat16).view(st["back_n"], h * hd)
    return out


def _plain_attend(st):
    c, kv = st["case"], st["kv"]
    n, s, most, hd, h = st["n"], c["n_seq"], st["most"], c["hd"], c["n_kv"]
    g = c["n_head"] // h
    seq, i = _row_index(st["off"], n)
    q = torch.zeros(s, most, h * g, hd, device=st["q"].device)
    q[seq, i] = st["q"].view(n, h * g, hd)
    q = q.view(s, most, h, g, hd).permute(0, 2, 3, 1, 4).reshape(s, h, g * most, hd)
    pages = kv["table"].long()
    k, v = (_values(kv, w, pages).transpose(1, 2).reshape(s, h, -1, hd) for w in ("k", "v"))
    length = k.shape[2]
    score = torch.matmul(q, k.transpose(-1, -2)).mul_(1.0 / math.sqrt(hd)).view(s, h, g, most, length)
    at = st["pos0"].long()[:, None] + torch.arange(most, device=q.device)
    key = torch.arange(length, device=q.device)
    seen = key <= at[..., None]
    if c["window"]:
        seen &= (key > at[..., None] - c["window"]) | (key < c["sinks"])
    score.masked_fill_(~seen[:, None, None], -math.inf)
    score = score.sub_(score.amax(-1, keepdim=True)).exp_()
    score = score.div_(score.sum(-1, keepdim=True))
    out = torch.matmul(score.view(s, h, g * most, length), v).view(s, h, g, most, hd)
    return {"out": out.permute(0, 3, 1, 2, 4)[seq, i].reshape(n, h * g * hd)}


def _plain_verify(st):
    c = st["case"]
    n, most, v = c["n_seq"], st["most"], c["n_vocab"]
    off = st["off"].long()
    count = off[1:] - off[:-1]
    step = torch.arange(most, device=off.device)
    real = step < count[:, None]
    d = (off[:-1, None] + step).clamp(max=st["ids"].numel() - 1)  # each draft's row
    s = torch.arange(n, device=off.device)
    ids = st["ids"].long()[d]
    p = st["target"][(d + s[:, None]), ids].double()
    q = torch.ones_like(p) if c["lookup"] else st["draft"][d, ids].double()
    took = (st["u_accept"].double()[d] * q < p) & real
    n_accept = took.int().cumprod(-1).sum(-1)
    stop = torch.minimum(n_accept, count - 1)
    refused = n_accept < count
    row = st["target"][off[:-1] + s + n_accept].double()
    at = off[:-1] + stop
    if c["lookup"]:
        less = torch.zeros_like(row).scatter_(1, ids[s, stop][:, None], math.inf)
    else:
        less = st["draft"][at].double()
    rest = torch.where(refused[:, None], (row - less).clamp(min=0), row)
    rest = torch.where(rest.sum(-1, keepdim=True) > 0, rest, row)
    total = rest.cumsum(-1)
    pick = torch.searchsorted(total, (st["u_pick"].double() * total[:, -1])[:, None], right=True)[:, 0]
    last = torch.where(rest > 0, torch.arange(v, device=off.device), 0).amax(-1)
    pick = torch.minimum(pick, last)
    place = torch.arange(most + 1, device=off.device)
    out = torch.full((n, most + 1), -1, dtype=torch.int32, device=off.device)
    padded = torch.cat([ids, ids[:, :1]], 1)
    out = torch.where(place < n_accept[:, None], padded.int(), out)
    out = torch.where(place == n_accept[:, None], pick[:, None].int(), out)
    return {"n_accept": n_accept.int(), "ids": out}


def run(state):
    if own:
        return _run_own(state)
    return {"append": _plain_append, "attend": _plain_attend, "verify": _plain_verify}[state["case"]["op"]](state)


# ------------------------------------------------------------------ from the definitions, in 64 bits
def _exact_append(st):
    c, kv = st["case"], st["kv"]
    page, hd, h = c["page"], c["hd"], c["n_kv"]
    rows, first = _shape(c)
    out = {"qr": [], "k": [], "v": []}
    at = 0
    for s, (n, p0) in enumerate(zip(rows, first)):
        cs = st["rope"][p0:p0 + n].double()

        def rotated(x, w, heads):
            x = x[at:at + n].double()
            rms = ((x ** 2).sum(1) / x.shape[1] + EPS).sqrt()
            x = (x / rms[:, None] * w.double()).view(n, heads, hd)
            y = torch.empty_like(x)
            for m, (one, two) in enumerate(((cs[..., 0], -cs[..., 1]), (cs[..., 1], cs[..., 0]))):
                lo, hi = x[..., :hd // 2], x[..., hd // 2:]
                y[..., m * hd // 2:(m + 1) * hd // 2] = lo * one[:, None] + hi * two[:, None]
            return y

        out["qr"].append(rotated(st["q"], st["q_norm"], c["n_head"]).reshape(n, -1))
        start = p0 // page * page
        pages = kv["table"][s, start // page:(p0 + n - 1) // page + 1].long()
        for name, x in (("k", rotated(st["k"], st["k_norm"], h)), ("v", st["v"][at:at + n].double().view(n, h, hd))):
            scale = kv[name + "_scales"][pages].double()  # [blocks][h]
            code = kv[name + "_codes"][pages].double() - 128  # [blocks][h][page][hd]
            code = code.transpose(1, 2).reshape(-1, h, hd)[:p0 + n - start]
            new = torch.cat([torch.zeros(p0 - start, h, hd, dtype=torch.float64, device=x.device), x])
            vals = torch.empty_like(new)
            for b in range(pages.numel()):
                i = slice(b * page, min((b + 1) * page, new.shape[0]))
                big = new[i].abs().amax((0, 2))
                sc = 2.0 ** (torch.floor(torch.log2(big)) - 6)
                # the logarithm's own rounding at a power of two
                sc = torch.where(big >= 128 * sc, sc * 2, torch.where(big < 64 * sc, sc / 2, sc))
                u = torch.floor(new[i] / sc[:, None])
                if b == 0 and p0 > start:
                    sc = torch.maximum(sc, scale[0])
                    u = torch.floor(new[i] / sc[:, None])
                    u[:p0 - start] = torch.floor(code[:p0 - start] * (scale[0] / sc)[:, None])
                vals[i] = (u.clamp(-128, 127) + 0.5) * sc[:, None]
            out[name].append(vals.reshape(-1, h * hd))
        at += n
    return {k: torch.cat(x) for k, x in out.items()}


def _exact_attend(st):
    c, kv = st["case"], st["kv"]
    hd, h = c["hd"], c["n_kv"]
    g = c["n_head"] // h
    rows, first = _shape(c)
    out = torch.empty(st["n"], h, g, hd, dtype=torch.float64, device=st["q"].device)
    at = 0
    for s, (n, p0) in enumerate(zip(rows, first)):
        total = p0 + n
        pages = kv["table"][s, :(total + c["page"] - 1) // c["page"]].long()
        q = st["q"][at:at + n].double().view(n, h, g, hd) / math.sqrt(hd)
        where = torch.arange(p0, total, device=q.device)[:, None]
        key = torch.arange(total, device=q.device)[None]
        hidden = key > where
        if c["window"]:
            hidden |= (key <= where - c["window"]) & (key >= c["sinks"])
        for j in range(h):
            k, v = ((kv[w + "_codes"][pages, j].double() - 127.5).mul_(kv[w + "_scales"][pages, j].double()[:, None, None])
                    .view(-1, hd)[:total] for w in ("k", "v"))
            for m in range(g):
                a = (q[:, j, m] @ k.t()).masked_fill_(hidden, -math.inf)
                a = torch.exp(a - torch.logsumexp(a, 1, keepdim=True))
                out[at:at + n, j, m] = a @ v
        at += n
    return {"out": out.view(st["n"], -1)}


def exact(case, seed):
    if case["op"] == "verify":
        return None  # whole numbers alone
    st = prepare(case, seed)
    return _exact_append(st) if case["op"] == "append" else _exact_attend(st)
