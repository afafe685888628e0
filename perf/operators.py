"""The paged key/value cache: what its three operators are measured on, with the same steps in plain torch.

A serving process keeps the keys and values of all its sequences in pages of a few rows, in the framework's cache format (int32 at
2^16, keys rotated): ``kpages`` / ``vpages`` [pages, KV heads, rows of a page, head dimension], a table of physical pages per
sequence, and for every page the largest and the smallest value of each key dimension (``bounds``).

* ``append``: the new keys and values of every sequence, rotated at their positions, into their pages; the bounds follow;
* ``attend``: the new token of every sequence attends to all its keys (or the last ``window`` of them);
* ``sparse``: pages are ranked by an upper bound of their scores, the token attends to the rows of the best ones only.

Everything is defined in integers (products and sums modulo 2^64, shifts that floor), so outputs are equal or wrong.
Head layouts are those of this repository's models: 32 query heads over 4 or 8 KV heads of 128, 8 over 2 of 64 in its tests.
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

FA = 16
ONE = 1 << FA
LOG2E, C0, C1, C2, C3 = 94548, 65536, 45426, 15743, 3638       # of the fixed-point exponential at 2^16
CLIP = ((FA + 2) << (2 * FA)) // LOG2E
ROPE_BASE = 50000.0


def listed():
    moe = {"heads": 32, "kv": 4, "hd": 128}                     # the mixture-of-experts decoder
    one_bit = {"heads": 32, "kv": 8, "hd": 128}                 # the 1-bit decoder
    return [
        # one step of a full server: a new row for every running sequence
        {"name": "append_step_64", "kind": "append", "sequences": 64, "length": 1000, "rows": 1, "page": 16, "rope": 1, **moe},
        # prompts of four requests in one packed batch, some of them later chunks
        {"name": "append_prompts_2048", "kind": "append", "sequences": 4, "length": 2500, "rows": 700, "page": 16, "rope": 2, **one_bit},
        # the smallest call: a single conversation's token
        {"name": "append_one", "kind": "append", "sequences": 1, "length": 300, "rows": 1, "page": 16, "rope": 1, **moe},
        # interactive generation, one sequence: young and long conversation
        {"name": "attend_1x300", "kind": "attend", "sequences": 1, "length": 300, "page": 16, "rope": 1, "window": 0, **moe},
        {"name": "attend_1x4096", "kind": "attend", "sequences": 1, "length": 4096, "page": 16, "rope": 1, "window": 0, **moe},
        # a nearly idle server with the other model, ragged lengths, larger pages
        {"name": "attend_7x1500", "kind": "attend", "sequences": 7, "length": 1500, "page": 32, "rope": 2, "window": 0, **one_bit},
        # sliding-window blocks: most of each conversation is out of sight
        {"name": "attend_window_12x6000", "kind": "attend", "sequences": 12, "length": 6000, "page": 16, "rope": 1, "window": 2048, **moe},
        # few long documents
        {"name": "attend_3x30000", "kind": "attend", "sequences": 3, "length": 30000, "page": 64, "rope": 0, "window": 0, **moe},
        # a full server
        {"name": "attend_64x4096", "kind": "attend", "sequences": 64, "length": 4096, "page": 16, "rope": 1, "window": 0, **moe},
        # long contexts where a token reads a fraction of the pages: one conversation, a few, many at moderate length
        {"name": "sparse_1x8000", "kind": "sparse", "sequences": 1, "length": 8000, "page": 16, "rope": 1, "window": 0, "select": 64, **moe},
        {"name": "sparse_32x2000", "kind": "sparse", "sequences": 32, "length": 2000, "page": 32, "rope": 2, "window": 0, "select": 13, **one_bit},
        {"name": "sparse_8x32000", "kind": "sparse", "sequences": 8, "length": 32000, "page": 16, "rope": 1, "window": 0, "select": 128, **moe},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "attend", "attend", "sparse"])
    heads, kv, hd = rng.choice([(32, 4, 128), (32, 8, 128), (8, 2, 64), (16, 4, 64), (12, 2, 128), (5, 5, 128)])
    case = {"kind": kind, "heads": heads, "kv": kv, "hd": hd, "page": rng.choice([16, 16, 32, 64, 128]), "rope": rng.choice([0, 1, 2])}
    keys = 160000 * 4 * 128 // (kv * hd)                        # keys of all sequences: at most as the full server's
    if kind == "append":
        rows = rng.choice([1, 1, _log(rng, 2, 700)])
        sequences = _log(rng, 1, 64 if rows == 1 else 4)
        length = max(rows, _log(rng, 1, 2500))
        return {**case, "sequences": sequences, "length": length if rows > 1 else min(length, 1000), "rows": rows}
    sequences = _log(rng, 1, 64)
    length = _log(rng, 1 if kind == "attend" else 200, min(30000, keys // sequences))
    case.update(sequences=sequences, length=length, window=rng.choice([0, 0, _log(rng, 1, 4096)]))
    if kind == "sparse":
        case["select"] = _log(rng, 2, 128)
    return case


def lengths(case):
    """Keys of every sequence, the new token's own among them: the longest first, in a batch of eight and more one slot without a sequence."""
    rng = random.Random(case["sequences"] * 1000003 + case["length"])
    out = [case["length"]] + [rng.randint(max(1, case["length"] // 4), case["length"]) for _ in range(case["sequences"] - 1)]
    if len(out) >= 8:
        out[rng.randrange(1, len(out))] = 0
    return out


def new_rows(case):
    """Rows that an append brings for every sequence (they end at its length)."""
    if case["rows"] == 1:
        return [min(1, n) for n in lengths(case)]
    rng = random.Random(case["sequences"] + case["rows"] * 7919)
    return [min(n, rng.randint(max(1, case["rows"] // 2), case["rows"])) for n in lengths(case)]


def visible(case):
    """First visible key and keys behind the last, of every sequence."""
    w = case["window"]
    return [(max(0, n - w) if w else 0, n) for n in lengths(case)]


def work(case):
    H, kv, hd, P = case["heads"], case["kv"], case["hd"], case["page"]
    if case["kind"] == "append":
        rows, pages, behind = 0, 0, 0
        for n, m in zip(lengths(case), new_rows(case)):
            if m:
                rows += m
                pages += (n - 1) // P - (n - m) // P + 1
                behind += (n - m) % P                           # rows of the first page that the bounds take in
        return {"bytes": kv * hd * (rows * 24 + behind * 4 + pages * 8), "flops": rows * kv * hd * 3}
    keys = extra = flops = 0
    for lo, n in visible(case):
        if n == 0:
            continue
        if case["kind"] == "sparse":
            pages = (n - 1) // P - lo // P + 1
            picked = min(pages, case["select"])
            extra += pages * kv * hd * 8 + picked * kv * 4
            flops += pages * H * hd * 4
            keys += min(n - lo, picked * P)
        else:
            keys += n - lo
    rows = case["sequences"] * H * hd * 16
    return {"bytes": keys * kv * hd * 8 + extra + rows, "flops": flops + keys * H * hd * 4}


# ------------------------------------------------------------------------------------------------------------- inputs ---
def _tables(rows, hd):
    inv = ROPE_BASE ** (-np.arange(hd // 2, dtype=np.float64) * 2 / hd)
    ang = np.arange(rows, dtype=np.float64)[:, None] * inv[None]
    return (torch.from_numpy(np.rint(f(ang) * ONE).astype(np.int64)).cuda() for f in (np.cos, np.sin))


def _bounds_of(kpages, table, lens):
    """[pages, kv, 2, hd]: largest and smallest written value of every dimension (pages of no sequence: zero)."""
    P = kpages.shape[2]
    out = torch.zeros((kpages.shape[0], kpages.shape[1], 2, kpages.shape[3]), dtype=torch.int32, device=kpages.device)
    for b, n in enumerate(lens):
        for first in range(0, (n + P - 1) // P, 512):           # (in parts: a long sequence's rows are gathered)
            ids = table[b, first:min(first + 512, (n + P - 1) // P)].long()
            rows = kpages[ids]
            written = (torch.arange(first * P, first * P + len(ids) * P, device=rows.device) < n).view(-1, 1, P, 1)
            lim = torch.iinfo(torch.int32)
            out[ids, :, 0] = rows.masked_fill(~written, lim.min).amax(2)
            out[ids, :, 1] = rows.masked_fill(~written, lim.max).amin(2)
    return out


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    H, kv, hd, P, lens = case["heads"], case["kv"], case["hd"], case["page"], lengths(case)
    per_seq = max(1, (max(lens) + P - 1) // P)
    need = sum((n + P - 1) // P for n in lens)
    n_pages = need + 3                                          # the pool has a few free pages
    order = torch.randperm(n_pages, generator=gen, device="cuda").to(torch.int32)
    table = torch.zeros((len(lens), per_seq), dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(lens):
        m = (n + P - 1) // P
        table[b, :m] = order[at:at + m]
        at += m
    # keys drift from page to page (a text has topics), values do not; pages hold old rows behind a sequence's last
    kpages = torch.empty((n_pages, kv, P, hd), dtype=torch.int32, device="cuda")
    vpages = torch.empty_like(kpages)
    for first in range(0, n_pages, 4096):
        part = slice(first, min(first + 4096, n_pages))
        shape = kpages[part].shape
        topic = 0.6 * torch.randn((shape[0], kv, 1, hd), generator=gen, device="cuda")
        kpages[part] = ((torch.randn(shape, generator=gen, device="cuda") * 0.8 + topic) * ONE).round().to(torch.int32)
        vpages[part] = (torch.randn(shape, generator=gen, device="cuda") * ONE).round().to(torch.int32)
    cos, sin = _tables(max(1, max(lens)), hd)
    state = {"case": case, "table": table, "kpages": kpages, "vpages": vpages, "cos": cos, "sin": sin}
    if case["kind"] == "append":
        rows = new_rows(case)
        total = sum(rows)
        # keys and values are columns of the fused product's rows
        qkv = (torch.randn((max(total, len(lens)) if case["rows"] == 1 else total, (H + 2 * kv) * hd), generator=gen, device="cuda") * ONE).round().to(torch.int64)
        state.update(k=qkv[:, H * hd:(H + kv) * hd], v=qkv[:, (H + kv) * hd:], bounds=_bounds_of(kpages, table, [n - m for n, m in zip(lens, rows)]))
        state["start"] = torch.tensor([n - m if m else -1 for n, m in zip(lens, rows)], dtype=torch.int32, device="cuda")
        if case["rows"] > 1:
            state["rows"] = torch.tensor(np.concatenate([[0], np.cumsum(rows)]), dtype=torch.int32, device="cuda")
    else:
        state["q"] = (torch.randn((len(lens), H * hd), generator=gen, device="cuda") * (1.5 * ONE)).round().to(torch.int64)
        state["lengths"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        if case["kind"] == "sparse":
            state["bounds"] = _bounds_of(kpages, table, lens)
    return state


# --------------------------------------------------------------------------------------------------------- plain form ---
def _rotate(x, cos, sin, rope):
    """x [rows, heads, hd] int64, one table row per row."""
    if rope == 0:
        return x
    half = x.shape[-1] // 2
    c, s = cos[:, None], sin[:, None]
    out = torch.empty_like(x)
    a, b = (x[..., 0::2], x[..., 1::2]) if rope == 1 else (x[..., :half], x[..., half:])
    y0, y1 = (a * c - b * s) >> FA, (a * s + b * c) >> FA
    if rope == 1:
        out[..., 0::2], out[..., 1::2] = y0, y1
    else:
        out[..., :half], out[..., half:] = y0, y1
    return out


def _product(a, b):
    """a @ b of whole numbers in int32's range, exactly: in pieces of sixteen bits whose products and sums doubles hold without rounding."""
    a, b = a.to(torch.int64), b.to(torch.int64)
    a1, b1 = a >> 16, b >> 16
    a0, b0 = a - (a1 << 16), b - (b1 << 16)
    a0, a1, b0, b1 = a0.double(), a1.double(), b0.double(), b1.double()
    low, mid, high = a0 @ b0, a0 @ b1 + a1 @ b0, a1 @ b1
    return low.to(torch.int64) + (mid.to(torch.int64) << 16) + (high.to(torch.int64) << 32)


def _exponential(below):
    u = (below.clamp(max=CLIP) * LOG2E) >> FA
    f = u & (ONE - 1)
    f2 = (f * f) >> FA
    f3 = (f2 * f) >> FA
    p = C0 - ((C1 * f) >> FA) + ((C2 * f2) >> FA) - ((C3 * f3) >> FA)
    return p.clamp(min=0) >> (u >> FA).clamp(max=63)


def _attend(q, k, v, seen, hd):
    """q [B, kv, rep, hd] rotated, k / v [B, kv, L, hd], seen [B, kv, L] -> [B, kv, rep, hd]."""
    inv_sqrt = round(ONE / math.sqrt(hd))
    s = ((_product(q, k.transpose(-1, -2)) >> FA) * inv_sqrt) >> FA
    seen = seen[:, :, None]
    top = s.masked_fill(~seen, -(1 << 62)).amax(-1, keepdim=True)
    e = _exponential((top - s).clamp(min=0)).masked_fill(~seen, 0)
    z = e.sum(-1, keepdim=True)
    p = (e << FA) // z.clamp(min=1)
    return _product(p, v) >> FA


def _queries(st):
    c = st["case"]
    n = st["lengths"].long()
    at = (n - 1).clamp(min=0)
    q = st["q"].view(-1, c["heads"], c["hd"])
    return _rotate(q, st["cos"][at], st["sin"][at], c["rope"]).view(-1, c["kv"], c["heads"] // c["kv"], c["hd"])


def _plain_append(st):
    c = st["case"]
    kv, hd, P = c["kv"], c["hd"], c["page"]
    start = st["start"].long()
    B = len(start)
    if "rows" in st:
        edge = st["rows"].long()
        seq = torch.repeat_interleave(torch.arange(B, device="cuda"), edge[1:] - edge[:-1])
        row = torch.arange(len(seq), device="cuda")
        pos = start[seq] + row - edge[seq]
    else:
        seq = row = torch.nonzero(start >= 0).view(-1)
        pos = start[seq]
    k = _rotate(st["k"][row].view(-1, kv, hd), st["cos"][pos], st["sin"][pos], c["rope"])
    page = st["table"][seq, pos // P].long()
    st["kpages"][page, :, pos % P] = k.to(torch.int32)
    st["vpages"][page, :, pos % P] = st["v"][row].view(-1, kv, hd).to(torch.int32)
    # the written rows of every page that was met: up to the last position in it
    last = torch.zeros(st["kpages"].shape[0], dtype=torch.int64, device="cuda").scatter_reduce(0, page, pos % P, "amax")
    rows = st["kpages"][page]
    written = (torch.arange(P, device="cuda")[None] <= last[page][:, None]).view(-1, 1, P, 1)
    lim = torch.iinfo(torch.int32)
    st["bounds"][page, :, 0] = rows.masked_fill(~written, lim.min).amax(2)
    st["bounds"][page, :, 1] = rows.masked_fill(~written, lim.max).amin(2)
    return {"kpages": st["kpages"], "vpages": st["vpages"], "bounds": st["bounds"]}


def _parts(st):
    """Sequences a few at a time: what the plain form lays out stays within some gigabytes."""
    c = st["case"]
    step = max(1, (1 << 27) // (c["kv"] * c["hd"] * max(1, c["length"])))
    return [slice(b, min(b + step, c["sequences"])) for b in range(0, c["sequences"], step)]


def _plain_attend(st):
    c = st["case"]
    P, hd = c["page"], c["hd"]
    q, outs = _queries(st), []
    for part in _parts(st):
        n, table = st["lengths"][part].long(), st["table"][part].long()
        lay = lambda pages: pages[table].transpose(1, 2).reshape(len(n), c["kv"], -1, hd)
        key = torch.arange(table.shape[1] * P, device="cuda")[None]
        seen = key < n[:, None]
        if c["window"]:
            seen &= key >= (n - c["window"])[:, None]
        outs.append(_attend(q[part], lay(st["kpages"]), lay(st["vpages"]), seen[:, None].expand(-1, c["kv"], -1), hd).reshape(len(n), -1))
    return torch.cat(outs)


def _plain_select(st, q, part):
    c = st["case"]
    P = c["page"]
    n, table = st["lengths"][part].long(), st["table"][part].long()
    bounds = st["bounds"][table].transpose(1, 2)                # [B, kv, pages, 2, hd]
    score = (_product(q.clamp(min=0), bounds[:, :, :, 0].transpose(-1, -2)) + _product(q.clamp(max=0), bounds[:, :, :, 1].transpose(-1, -2))).amax(2)
    page = torch.arange(table.shape[1], device="cuda")[None, None]
    first = ((n - c["window"]).clamp(min=0) // P if c["window"] else torch.zeros_like(n))[:, None, None]
    last = ((n - 1) // P)[:, None, None]                        # -1: no key
    lim = torch.iinfo(torch.int64)
    score = score.masked_fill((page == first) | (page == last), lim.max)
    shown = (page >= first) & (page <= last)
    score = score.masked_fill(~shown, lim.min)
    order = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :c["select"]]
    took = shown.expand_as(score).gather(-1, order)
    picked = torch.where(took, order, table.shape[1]).sort(-1).values
    if picked.shape[-1] < c["select"]:
        picked = torch.nn.functional.pad(picked, (0, c["select"] - picked.shape[-1]), value=table.shape[1])
    return torch.where(picked < table.shape[1], picked, -1)


def _plain_sparse(st):
    c = st["case"]
    P, hd, kv = c["page"], c["hd"], c["kv"]
    q, pages, outs = _queries(st), [], []
    for part in _parts(st):
        n, table = st["lengths"][part].long(), st["table"][part].long()
        picked = _plain_select(st, q[part], part)
        at = picked.clamp(min=0)
        physical = table[:, None].expand(-1, kv, -1).gather(-1, at)
        head = torch.arange(kv, device="cuda")[None, :, None]
        lay = lambda pool: pool[physical, head].reshape(len(n), kv, -1, hd)
        key = (at[..., None] * P + torch.arange(P, device="cuda")).view(len(n), kv, -1)
        seen = (picked >= 0).repeat_interleave(P, -1) & (key < n[:, None, None])
        if c["window"]:
            seen &= key >= (n - c["window"])[:, None, None]
        outs.append(_attend(q[part], lay(st["kpages"]), lay(st["vpages"]), seen, hd).reshape(len(n), -1))
        pages.append(picked.to(torch.int32))
    return {"pages": torch.cat(pages), "out": torch.cat(outs)}


# ------------------------------------------------------------------------------------------------------------ one pass ---
def run(st):
    c = st["case"]
    if not own:
        return {"append": _plain_append, "attend": _plain_attend, "sparse": _plain_sparse}[c["kind"]](st)
    from integer_inference_engine_b200 import device
    turn = dict(fa=FA, cos=st["cos"], sin=st["sin"], rope=c["rope"])
    if c["kind"] == "append":
        device.paged_append(st["k"], st["v"], st["kpages"], st["vpages"], st["table"], st["start"], rows=st.get("rows"), bounds=st["bounds"], **turn)
        return {"kpages": st["kpages"], "vpages": st["vpages"], "bounds": st["bounds"]}
    if c["kind"] == "attend":
        return device.paged_attention(st["q"], st["kpages"], st["vpages"], st["table"], st["lengths"], window=c["window"], **turn)
    pages = device.paged_select(st["q"], st["bounds"], st["table"], st["lengths"], c["page"], c["select"], window=c["window"], **turn)
    out = device.paged_attention(st["q"], st["kpages"], st["vpages"], st["table"], st["lengths"], window=c["window"], pages=pages, **turn)
    return {"pages": pages, "out": out}


# ------------------------------------------------------------------------------------- the definition, in NumPy's int64 ---
def _np_turn(x, c, s, rope):
    if rope == 0:
        return x
    y = np.empty_like(x)
    i = np.arange(x.shape[-1] // 2)
    a, b = (2 * i, 2 * i + 1) if rope == 1 else (i, i + len(i))
    y[..., a] = (x[..., a] * c - x[..., b] * s) >> FA
    y[..., b] = (x[..., a] * s + x[..., b] * c) >> FA
    return y


def _np_head(q, k, v):
    """One query head [hd] over its visible rows [n, hd]."""
    if len(k) == 0:
        return np.zeros_like(q)
    s = (((k @ q) >> FA) * round(ONE / math.sqrt(len(q)))) >> FA
    u = (np.minimum(s.max() - s, CLIP) * LOG2E) >> FA
    whole, f = u >> FA, u & (ONE - 1)
    sq = (f * f) >> FA
    poly = C0 - ((C1 * f) >> FA) + ((C2 * sq) >> FA) - ((C3 * ((sq * f) >> FA)) >> FA)
    e = np.maximum(poly, 0) >> np.minimum(whole, 63)
    return (((e << FA) // e.sum()) @ v) >> FA


def exact(case, seed):
    if work(case)["flops"] > 9e9:
        return None
    st = {k: v.cpu().numpy() if isinstance(v, torch.Tensor) else v for k, v in prepare(case, seed).items()}
    H, kv, hd, P = case["heads"], case["kv"], case["hd"], case["page"]
    table, cos, sin, rep = st["table"], st["cos"], st["sin"], H // kv
    if case["kind"] == "append":
        kp, vp, bounds, row = st["kpages"].copy(), st["vpages"].copy(), st["bounds"].copy(), 0
        for b, (n, m) in enumerate(zip(lengths(case), new_rows(case))):
            if case["rows"] == 1:
                row = b
            for pos in range(n - m, n):
                page = table[b, pos // P]
                kp[page, :, pos % P] = _np_turn(st["k"][row].reshape(kv, hd), cos[pos], sin[pos], case["rope"])
                vp[page, :, pos % P] = st["v"][row].reshape(kv, hd)
                row += 1
            for logical in range((n - m) // P, (n + P - 1) // P if m else 0):
                rows = kp[table[b, logical], :, :min(P, n - logical * P)]
                bounds[table[b, logical], :, 0], bounds[table[b, logical], :, 1] = rows.max(1), rows.min(1)
        return {"kpages": kp, "vpages": vp, "bounds": bounds}
    out = np.zeros((case["sequences"], H, hd), np.int64)
    pages = np.full((case["sequences"], kv, case.get("select", 0)), -1, np.int32)
    for b, (lo, n) in enumerate(visible(case)):
        if n == 0:
            continue
        q = _np_turn(st["q"][b].reshape(H, hd), cos[n - 1], sin[n - 1], case["rope"])
        shown = np.arange(lo // P, (n - 1) // P + 1)
        for g in range(kv):
            mine = shown
            if case["kind"] == "sparse":
                mx, mn = (st["bounds"][table[b, shown], g, i].astype(np.int64) for i in (0, 1))
                best = np.max([np.maximum(mx * q[h], mn * q[h]).sum(1) for h in range(g * rep, g * rep + rep)], axis=0)
                best[[0, -1]] = np.iinfo(np.int64).max
                mine = np.sort(shown[np.lexsort((shown, -best))[:case["select"]]])
                pages[b, g, :len(mine)] = mine
            key = (mine[:, None] * P + np.arange(P)).reshape(-1)
            inside = (key >= lo) & (key < n)
            k, v = (st[pool][table[b, mine], g].reshape(-1, hd)[inside].astype(np.int64) for pool in ("kpages", "vpages"))
            for h in range(g * rep, g * rep + rep):
                out[b, h] = _np_head(q[h], k, v)
    out = out.reshape(case["sequences"], -1)
    return out if case["kind"] == "attend" else {"pages": pages, "out": out}
