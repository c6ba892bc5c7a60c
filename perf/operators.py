"""The serving operators around a paged K/V cache, as they are measured: attention of whole prompts (packed) and of new
tokens over a paged cache, the write of new tokens into pages, and the page bookkeeping (resize, fork, compact) with its
page copies.

Each case is one call as a serving loop makes it.  `own` false computes it from elementary torch operations in 32 bits;
`own` true calls the framework's operators.
"""

from __future__ import annotations

import math
import os
import random
import sys

import numpy as np
import torch

own = False

BF16 = torch.bfloat16
DEVICE = "cuda"


# --------------------------------------------------------------------- cases
def listed():
    return [
        # A short interactive prompt beside two tiny ones: the latency of a first token.  A fixed-size batch, so rows
        # behind the last sequence are padding.
        dict(name="prefill short ragged d64", op="prefill", hq=32, hkv=32, d=64, batch=3, longest=129, pad=3, mix=1),
        # One long document, the head layout of an 8B GQA model: bound by the tensor cores.
        dict(name="prefill 8192 d128", op="prefill", hq=32, hkv=8, d=128, batch=1, longest=8192, pad=0, mix=2),
        # Verification of a few drafted tokens per sequence over long caches: few rows, bound by reading the cache.
        dict(name="chunk verify hnd16", op="chunk", hq=32, hkv=8, d=128, batch=8, longest=16384, new=5, page=16, nhd=False, mix=3),
        # A mixed step: a chunk of a long prompt together with single-token rows.
        dict(name="chunk mixed nhd64", op="chunk", hq=64, hkv=8, d=128, batch=4, longest=8192, new=1021, page=64, nhd=True, mix=4),
        # One decode step's new tokens into their pages.
        dict(name="write step hnd16", op="write", hkv=8, d=128, batch=32, longest=4096, new=1, page=16, nhd=False, mix=5),
        # The prompts of an admitted batch into their pages.
        dict(name="write prompts nhd16", op="write", hkv=8, d=128, batch=8, longest=8192, new=4097, page=16, nhd=True, mix=6),
        # A decode step's bookkeeping: every row grows by a token, a few finish.
        dict(name="resize step", op="resize", batch=32, longest=4096, grow=1, page=16, spare=64, mix=7),
        # Admission: finished rows leave, new prompts take their pages; a pool as large as a GPU's memory holds.
        dict(name="resize admission", op="resize", batch=256, longest=16384, grow=8192, page=16, spare=40000, mix=8),
        # Beams of a few sequences.
        dict(name="fork beams hnd16", op="fork", hkv=8, d=128, rows=4, forks=12, longest=1024, page=16, nhd=False, spare=32, mix=9),
        # Many samples of long shared prompts.
        dict(name="fork samples nhd64", op="fork", hkv=8, d=128, rows=8, forks=248, longest=16384, page=64, nhd=True, spare=300, mix=10),
        # A small pool after a few sequences ended.
        dict(name="compact small hnd16", op="compact", hkv=8, d=128, rows=8, longest=512, page=16, nhd=False, spare=150, mix=11),
        # A fragmented pool of 64K tokens of live cache.
        dict(name="compact pool hnd16", op="compact", hkv=8, d=128, rows=64, longest=4096, page=16, nhd=False, spare=4000, mix=12),
    ]


HEADS = ((8, 8), (32, 8), (32, 32), (64, 8), (24, 8), (28, 4))
PAGES = (8, 16, 32, 64, 128, 256)


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(("prefill", "prefill", "chunk", "chunk", "write", "resize", "fork", "compact"))
    hq, hkv = rng.choice(HEADS)
    d = rng.choice((64, 128))
    page = rng.choice(PAGES)
    common = dict(op=op, mix=rng.randrange(1 << 30))
    pages = dict(common, page=page, longest=max(page, log(32, 16384)))
    layout = dict(nhd=rng.random() < 0.5, hkv=hkv, d=d)
    if op == "prefill":
        batch = log(1, 48)
        longest = log(1, int(min(8192, math.sqrt(2.1e9 / (batch * hq)))))
        return dict(common, hq=hq, hkv=hkv, d=d, batch=batch, longest=longest, pad=rng.choice((0, 0, 1, 77)))
    if op == "chunk":
        batch = log(1, 32)
        new = log(1, int(min(2048, max(1, 2.1e9 / (batch * hq * pages["longest"])))))
        return dict(pages, **layout, hq=hq, batch=batch, new=min(new, pages["longest"]))
    if op == "write":
        batch = log(1, 64)
        new = log(1, min(pages["longest"], max(1, 32768 // batch)))
        return dict(pages, **layout, batch=batch, new=new, longest=min(pages["longest"], max(page, new, 262144 // batch)))
    if op == "resize":
        return dict(pages, batch=log(1, 256), grow=log(1, pages["longest"]), spare=log(1, 40000))
    if op == "fork":
        rows = log(1, 8)
        forks = log(1, 248)
        return dict(pages, **layout, rows=rows, forks=forks, spare=rng.choice((forks + 5, forks + 50, forks // 2 + 1)))
    rows = log(1, 64)
    longest = max(page, min(pages["longest"], 262144 // rows))
    live = rows * longest // page
    return dict(pages, **layout, rows=rows, longest=longest, spare=max(1, int(live * rng.uniform(0.05, 1.0))))


def _lengths(case, count, longest, salt=0, zero=True):
    """`count` lengths spread over the logarithm up to `longest`, which one of them has; a row in eight or so is empty."""
    rng = random.Random(case["mix"] * 7919 + salt)
    lens = [int(round(math.exp(rng.uniform(0.0, math.log(longest))))) if longest > 1 else 1 for _ in range(count)]
    if zero and count >= 3:
        for i in range(count):
            if rng.random() < 0.12:
                lens[i] = 0
    lens[rng.randrange(count)] = longest
    return lens


def _chunk_lengths(case):
    """(new tokens, all tokens) of each row of a chunk or write case."""
    new = _lengths(case, case["batch"], case["new"], 1)
    held = _lengths(case, case["batch"], case["longest"], 2)
    total = [min(case["longest"], max(n, h)) for n, h in zip(new, held)]
    return new, total


def _ceil(a, b):
    return -(-a // b)


def _resize_lengths(case):
    """(lengths before, lengths wanted): rows that end, rows that start, rows cut back a little, the others grow."""
    rng = random.Random(case["mix"] * 7919 + 3)
    old = _lengths(case, case["batch"], case["longest"], 4)
    want = []
    for n in old:
        u = rng.random()
        if n and u < 0.15:
            want.append(0)
        elif n > 2 and u < 0.22:
            want.append(n - rng.randrange(1, min(n - 1, 6) + 1))
        else:
            want.append(min(case["longest"], n + rng.randrange(1, case["grow"] + 1)))
    return old, want


def _shared(case, lens):
    """How many leading full pages each row shares with the row before it."""
    rng = random.Random(case["mix"] * 7919 + 5)
    share = [0]
    for a, b in zip(lens, lens[1:]):
        full = min(a, b) // case["page"]
        share.append(rng.randrange(full + 1) if rng.random() < 0.25 else 0)
    return share


# -------------------------------------------------------------------- inputs
def _generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(seed)


def _randn(gen, *shape):
    return torch.randn(shape, generator=gen, device=DEVICE, dtype=BF16)


def _cu(lens):
    return torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device=DEVICE)


def _int(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def _tables(case, lens, width, spare, seed, share=None, rows=None):
    """A table whose rows hold randomly placed pages for `lens` tokens, and the count of rows that hold each page."""
    page = case["page"]
    share = share or [0] * len(lens)
    held = [_ceil(n, page) for n in lens]
    blocks = sum(h - s for h, s in zip(held, share)) + spare
    order = np.random.default_rng(seed).permutation(blocks).astype(np.int32)
    table = np.full((rows or len(lens), width), -1, dtype=np.int32)
    at = 0
    for b, (h, s) in enumerate(zip(held, share)):
        if s:
            table[b, :s] = table[b - 1, :s]
        table[b, s:h] = order[at : at + h - s]
        at += h - s
    refs = np.bincount(table[table >= 0], minlength=blocks).astype(np.int32)
    return torch.from_numpy(table).to(DEVICE), torch.from_numpy(refs).to(DEVICE)


def _pools(gen, case, blocks):
    shape = (blocks, case["page"], case["hkv"], case["d"]) if case["nhd"] else (blocks, case["hkv"], case["page"], case["d"])
    return _randn(gen, *shape), _randn(gen, *shape)


def _width(case):
    return _ceil(case["longest"], case["page"]) + 1


def prepare(case, seed):
    gen = _generator(seed)
    op = case["op"]
    s = dict(op=op, case=case)
    if op == "prefill":
        hq, hkv, d = case["hq"], case["hkv"], case["d"]
        lens = _lengths(case, case["batch"], case["longest"])
        rows = sum(lens) + case["pad"]
        # the views that a fused projection gives
        qkv = _randn(gen, rows, (hq + 2 * hkv) * d)
        s["q"] = qkv[:, : hq * d].view(rows, hq, d)
        s["k"] = qkv[:, hq * d : (hq + hkv) * d].view(rows, hkv, d)
        s["v"] = qkv[:, (hq + hkv) * d :].view(rows, hkv, d)
        s["cu"], s["longest"] = _cu(lens), max(lens)
        return s
    if op in ("chunk", "write"):
        new, total = _chunk_lengths(case)
        s["table"], refs = _tables(case, total, _width(case), 8, seed)
        s["k_cache"], s["v_cache"] = _pools(gen, case, refs.numel())
        s["cu"], s["new"], s["longest"] = _cu(new), max(new), max(total)
        if op == "chunk":
            s["q"] = _randn(gen, sum(new), case["hq"], case["d"])
            s["lens"] = _int(total)
        else:
            s["k"] = _randn(gen, sum(new), case["hkv"], case["d"])
            s["v"] = _randn(gen, sum(new), case["hkv"], case["d"])
            s["starts"] = _int([t - n for n, t in zip(new, total)])
        return s
    if op == "resize":
        old, want = _resize_lengths(case)
        s["table"], s["refs"] = _tables(case, old, _width(case), case["spare"], seed, _shared(case, old))
        s["lens"], s["want"] = _int(old), _int(want)
        return s
    if op == "fork":
        rows, forks = case["rows"], case["forks"]
        lens = _lengths(case, rows, case["longest"], 6, zero=False)
        s["table"], s["refs"] = _tables(case, lens, _width(case), case["spare"], seed, rows=rows + forks)
        s["lens"] = _int(lens + [0] * forks)
        rng = random.Random(seed)
        s["parents"] = _int([rng.randrange(rows) for _ in range(forks)])
        s["children"] = _int(rng.sample(range(rows, rows + forks), forks))
    else:
        lens = _lengths(case, case["rows"], case["longest"], 7)
        s["table"], s["refs"] = _tables(case, lens, _width(case), case["spare"], seed, _shared(case, lens))
        s["lens"] = _int(lens)
    s["k_cache"], s["v_cache"] = _pools(gen, case, s["refs"].numel())
    return s


# ----------------------------------------------------------------------- run
def _framework():
    path = os.path.join(os.getcwd(), "hpc-ops-sm120_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import attention_decode

    return attention_decode


def run(s):
    return (_run_own if own else _run_plain)(s)


def _run_own(s):
    ad, op, case = _framework(), s["op"], s["case"]
    if op == "prefill":
        return ad.attention_prefill(s["q"], s["k"], s["v"], s["cu"])
    if op == "chunk":
        return ad.attention_prefill_paged(
            s["q"], s["k_cache"], s["v_cache"], s["table"], s["cu"], s["lens"], layout="NHD" if case["nhd"] else "HND"
        )
    if op == "write":
        ad.cache_write(
            s["k"], s["v"], s["k_cache"], s["v_cache"], s["table"], s["cu"], s["starts"], layout="NHD" if case["nhd"] else "HND"
        )
        return {"k": s["k_cache"], "v": s["v_cache"]}
    # The tables are changed in place: a pass works on a copy, so that the next finds the state as it was.
    table, refs = s["table"].clone(), s["refs"].clone()
    if op == "resize":
        lens = ad.cache_resize(table, s["lens"], s["want"], refs, page_size=case["page"])
        return {"table": table, "refs": refs, "lens": lens}
    if op == "fork":
        lens, src, dst = ad.cache_fork(table, s["lens"], refs, s["parents"], s["children"], page_size=case["page"])
    else:
        lens = s["lens"]
        src, dst = ad.cache_compact(table, lens, refs, page_size=case["page"])
    ad.cache_copy_pages(s["k_cache"], s["v_cache"], src, dst)
    return {"table": table, "refs": refs, "lens": lens, "src": src, "dst": dst, "k": s["k_cache"], "v": s["v_cache"]}


# --------------------------------------------------------------- plain forms
def _run_plain(s):
    op = s["op"]
    if op == "prefill":
        return _plain_prefill(s)
    if op == "chunk":
        return _plain_chunk(s)
    if op == "write":
        return _plain_write(s)
    table, refs = s["table"].clone(), s["refs"].clone()
    if op == "resize":
        lens = _plain_resize(table, s["lens"], s["want"], refs, s["case"]["page"])
        return {"table": table, "refs": refs, "lens": lens}
    if op == "fork":
        lens, src, dst = _plain_fork(table, s["lens"], refs, s["parents"], s["children"], s["case"]["page"])
    else:
        lens = s["lens"]
        src, dst = _plain_compact(table, lens, refs, s["case"]["page"])
    keep = dst >= 0
    to, at = dst[keep].long(), src[keep].long()
    s["k_cache"][to] = s["k_cache"][at]
    s["v_cache"][to] = s["v_cache"][at]
    return {"table": table, "refs": refs, "lens": lens, "src": src, "dst": dst, "k": s["k_cache"], "v": s["v_cache"]}


def _attend(q, k, v, limit, group):
    """q [B, n, Hq, D]; k, v [B, m, Hkv, D]; row (b, i) sees its first limit[b, i] keys.  32 bits throughout."""
    b, n, hq, d = q.shape
    hkv = k.shape[2]
    q = q.float().view(b, n, hkv, group, d).permute(0, 2, 3, 1, 4).reshape(b, hkv, group * n, d)
    k = k.float().permute(0, 2, 3, 1)
    v = v.float().permute(0, 2, 1, 3)
    scores = torch.matmul(q * (1.0 / math.sqrt(d)), k).view(b, hkv, group, n, -1)
    hidden = torch.arange(scores.shape[-1], device=q.device) >= limit[:, None, None, :, None]
    scores.masked_fill_(hidden, float("-inf"))
    top = scores.amax(-1, keepdim=True)
    scores.sub_(torch.where(top == float("-inf"), 0.0, top)).exp_()
    total = scores.sum(-1, keepdim=True)
    out = torch.matmul(scores.view(b, hkv, group * n, -1), v).view(b, hkv, group, n, d)
    out = torch.where(total > 0, out / total, 0.0)
    return out.permute(0, 3, 1, 2, 4).reshape(b, n, hq, d)


def _plain_prefill(s):
    q, k, v, cu = s["q"], s["k"], s["v"], s["cu"].long()
    lens = cu[1:] - cu[:-1]
    i = torch.arange(s["longest"], device=q.device)
    rows = (cu[:-1, None] + i).clamp_(max=q.shape[0] - 1)
    valid = i < lens[:, None]
    limit = (i + 1).expand_as(rows)
    out = _attend(q[rows], k[rows], v[rows], limit, q.shape[1] // k.shape[1])
    full = torch.zeros(q.shape, dtype=BF16, device=q.device)
    full[rows[valid]] = out[valid].to(BF16)
    return full


def _gather(cache, table, longest, page, nhd):
    j = torch.arange(longest, device=cache.device)
    blocks = table[:, j // page].clamp(min=0).long()
    return cache[blocks, j % page] if nhd else cache[blocks, :, j % page]


def _plain_chunk(s):
    q, table, cu, lens, case = s["q"], s["table"], s["cu"].long(), s["lens"].long(), s["case"]
    k = _gather(s["k_cache"], table, s["longest"], case["page"], case["nhd"])
    v = _gather(s["v_cache"], table, s["longest"], case["page"], case["nhd"])
    new = cu[1:] - cu[:-1]
    i = torch.arange(s["new"], device=q.device)
    rows = (cu[:-1, None] + i).clamp_(max=q.shape[0] - 1)
    valid = i < new[:, None]
    limit = (lens - new)[:, None] + i + 1
    out = _attend(q[rows], k, v, limit, q.shape[1] // k.shape[2])
    full = torch.zeros(q.shape, dtype=BF16, device=q.device)
    full[rows[valid]] = out[valid].to(BF16)
    return full


def _plain_write(s):
    cu, case = s["cu"].long(), s["case"]
    t = torch.arange(s["k"].shape[0], device=cu.device)
    b = torch.searchsorted(cu, t, right=True) - 1
    pos = s["starts"].long()[b] + t - cu[b]
    blocks = s["table"][b, pos // case["page"]].long()
    at = (blocks, pos % case["page"]) if case["nhd"] else (blocks, slice(None), pos % case["page"])
    s["k_cache"][at] = s["k"]
    s["v_cache"][at] = s["v"]
    return {"k": s["k_cache"], "v": s["v_cache"]}


def _let_go(table, refs, drop):
    """Takes the entries where `drop` is true out of the table and the counts."""
    refs.index_add_(0, table.clamp(min=0).flatten().long(), -drop.flatten().to(torch.int32))
    table.masked_fill_(drop, -1)


def _free_pages(refs):
    """(free pages, lowest first, then the others; how many are free)."""
    free = refs == 0
    return torch.argsort(free.to(torch.int32), descending=True, stable=True).to(torch.int32), free.sum()


def _plain_resize(table, lens, want, refs, page):
    width = table.shape[1]
    j = torch.arange(width, device=table.device)
    old = lens.clamp(0, width * page)
    held = (old + page - 1) // page
    ok = (want >= 0) & (want <= width * page)
    _let_go(table, refs, (ok & (want == 0))[:, None] & (j < held[:, None]))
    keep = (want.clamp(0, width * page) + page - 1) // page
    cut = ok & (want > 0) & (want < old)
    tail = table.gather(1, (keep - 1).clamp(0, width - 1)[:, None].long())[:, 0]
    cut &= (want % page == 0) | (refs[tail.clamp(min=0).long()] <= 1)
    _let_go(table, refs, cut[:, None] & (j >= keep[:, None]) & (j < held[:, None]))
    grows = ok & (want > old)
    need = torch.where(grows, keep - held, 0)
    upto = need.cumsum(0)
    pages, count = _free_pages(refs)
    grows &= (need == 0) | (upto <= count)
    take = grows[:, None] & (j >= held[:, None]) & (j < keep[:, None])
    rank = ((upto - need)[:, None] + j - held[:, None]).clamp(0, refs.numel() - 1)
    given = pages[rank.long()]
    table.copy_(torch.where(take, given, table))
    refs.index_add_(0, given.flatten().long(), take.flatten().to(torch.int32))
    return torch.where(grows | cut | (ok & (want == 0)), want, old)


def _plain_fork(table, lens, refs, parents, children, page):
    width = table.shape[1]
    parents, children = parents.long(), children.long()
    length = lens[parents]
    full, part = length // page, length % page
    need = (part > 0).to(torch.int32)
    upto = need.cumsum(0)
    pages, count = _free_pages(refs)
    ok = (need == 0) | (upto <= count)
    j = torch.arange(width, device=table.device)
    share = ok[:, None] & (j < full[:, None])
    rows = table[parents]
    refs.index_add_(0, rows.clamp(min=0).flatten().long(), share.flatten().to(torch.int32))
    given = pages[(upto - need).clamp(max=refs.numel() - 1).long()]
    own_page = ok & (need > 0)
    refs.index_add_(0, given.long(), own_page.to(torch.int32))
    tail = rows.gather(1, full.clamp(max=width - 1)[:, None].long())[:, 0]
    src = torch.where(own_page, tail, -1)
    dst = torch.where(own_page, given, -1)
    mine = torch.where(share, rows, -1)
    mine = torch.where(own_page[:, None] & (j == full[:, None]), given[:, None], mine)
    table[children] = mine
    after = lens.clone()
    after[children] = torch.where(ok, length, 0)
    return after, src, dst


def _plain_compact(table, lens, refs, page):
    blocks = refs.numel()
    p = torch.arange(blocks, device=table.device)
    live = refs > 0
    count = live.sum()
    hole, high = ~live & (p < count), live & (p >= count)
    limit = blocks // 2
    holes = torch.argsort(hole.to(torch.int32), descending=True, stable=True)
    highs = torch.argsort(high.to(torch.int32), descending=True, stable=True)
    moved = p < hole.sum()
    target = p.clone()
    target[highs] = torch.where(moved, holes, highs)
    src = torch.where(moved, highs, -1)[:limit].to(torch.int32)
    dst = torch.where(moved, holes, -1)[:limit].to(torch.int32)
    held = torch.arange(table.shape[1], device=table.device) < ((lens + page - 1) // page)[:, None]
    table.copy_(torch.where(held, target[table.clamp(min=0).long()].to(torch.int32), table))
    old = refs.clone()
    refs.copy_(torch.where(high | hole, 0, old))
    refs.index_add_(0, target, torch.where(high, old, 0))
    return src, dst


# ---------------------------------------------------------------------- work
def work(case):
    op = case["op"]
    if op == "prefill":
        lens = _lengths(case, case["batch"], case["longest"])
        rows = sum(lens)
        pairs = sum(n * (n + 1) // 2 for n in lens)
        return {"bytes": 4 * case["d"] * (case["hq"] + case["hkv"]) * rows, "flops": 4 * case["d"] * case["hq"] * pairs}
    if op in ("chunk", "write"):
        new, total = _chunk_lengths(case)
        if op == "write":
            return {"bytes": 8 * case["d"] * case["hkv"] * sum(new), "flops": 0}
        pairs = sum(n * (t - n) + n * (n + 1) // 2 for n, t in zip(new, total))
        read = sum(t for n, t in zip(new, total) if n)
        size = 4 * case["d"] * (case["hq"] * sum(new) + case["hkv"] * read)
        return {"bytes": size, "flops": 4 * case["d"] * case["hq"] * pairs}
    page = case["page"]
    if op == "resize":
        old, want = _resize_lengths(case)
        share = _shared(case, old)
        held = [_ceil(n, page) for n in old]
        blocks = sum(h - s for h, s in zip(held, share)) + case["spare"]
        changed = sum(abs(_ceil(w, page) - h) for w, h in zip(want, held))
        # the copies of the table and the counts, the counts once, each changed entry and its count
        copies = 8 * (blocks + len(old) * _width(case))
        return {"bytes": copies + 4 * blocks + 16 * changed + 12 * len(old), "flops": 0}
    one = 2 * 2 * page * case["hkv"] * case["d"]  # a page of K and of V
    if op == "fork":
        lens = _lengths(case, case["rows"], case["longest"], 6, zero=False)
        blocks = sum(_ceil(n, page) for n in lens) + case["spare"]
        rows = case["rows"] + case["forks"]
        tails = min(case["spare"], case["forks"] * sum(n % page > 0 for n in lens) / len(lens))
        entries = case["forks"] * sum(_ceil(n, page) for n in lens) / len(lens)
        copies = 8 * (blocks + rows * _width(case))
        return {"bytes": int(copies + 4 * blocks + 16 * entries + 8 * rows + 2 * one * tails), "flops": 0}
    lens = _lengths(case, case["rows"], case["longest"], 7)
    share = _shared(case, lens)
    held = [_ceil(n, page) for n in lens]
    live = sum(h - s for h, s in zip(held, share))
    blocks = live + case["spare"]
    moved = live * case["spare"] / blocks
    copies = 8 * (blocks + case["rows"] * _width(case))
    return {"bytes": int(copies + 12 * blocks + 8 * sum(held) + 2 * one * moved), "flops": 0}


# --------------------------------------------------------------------- exact
def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op in ("prefill", "chunk"):
        return _exact_attention(s, case)
    page = case["page"]
    host = {name: x.cpu().numpy() for name, x in s.items() if isinstance(x, torch.Tensor) and not x.is_floating_point()}
    if op == "write":
        pools = {"k": s["k_cache"].clone(), "v": s["v_cache"].clone()}
        cu = host["cu"]
        for b in range(len(cu) - 1):
            for i in range(cu[b], cu[b + 1], 1):
                pos = int(host["starts"][b]) + i - int(cu[b])
                block, slot = int(host["table"][b, pos // page]), pos % page
                for name in ("k", "v"):
                    place = pools[name][block, slot] if case["nhd"] else pools[name][block, :, slot]
                    place.copy_(s[name][i])
        return {name: x.double() for name, x in pools.items()}
    table, refs, lens = (host[n].tolist() for n in ("table", "refs", "lens"))
    if op == "resize":
        after = _exact_resize(table, lens, host["want"].tolist(), refs, page)
        return {"table": _int(table), "refs": _int(refs), "lens": _int(after)}
    if op == "fork":
        lens, src, dst = _exact_fork(table, lens, host["parents"].tolist(), host["children"].tolist(), refs, page)
    else:
        src, dst = _exact_compact(table, lens, refs, page)
    pools = {"k": s["k_cache"].clone(), "v": s["v_cache"].clone()}
    for a, b in zip(src, dst):
        if b >= 0:
            for name in ("k", "v"):
                pools[name][b] = s[name + "_cache"][a]
    return {"table": _int(table), "refs": _int(refs), "lens": _int(lens), "src": _int(src), "dst": _int(dst),
            "k": pools["k"].double(), "v": pools["v"].double()}


def _exact_attention(s, case):
    q = s["q"].double()
    out = torch.zeros_like(q)
    cu = s["cu"].tolist()
    group = case["hq"] // case["hkv"]
    for b in range(len(cu) - 1):
        n = cu[b + 1] - cu[b]
        if not n:
            continue
        if case["op"] == "prefill":
            total = n
            k, v = s["k"][cu[b] : cu[b + 1]].double(), s["v"][cu[b] : cu[b + 1]].double()
        else:
            total = int(s["lens"][b])
            ids = s["table"][b, : _ceil(total, case["page"])].long()
            k, v = (c[ids].double() for c in (s["k_cache"], s["v_cache"]))
            if not case["nhd"]:
                k, v = k.transpose(1, 2), v.transpose(1, 2)
            k, v = (x.reshape(-1, case["hkv"], case["d"])[:total] for x in (k, v))
        sees = torch.ones(n, total, dtype=torch.bool, device=q.device).tril(total - n)
        for h in range(case["hq"]):
            x = q[cu[b] : cu[b + 1], h] @ k[:, h // group].T / math.sqrt(case["d"])
            weights = torch.softmax(x.masked_fill(~sees, -math.inf), -1)
            out[cu[b] : cu[b + 1], h] = weights @ v[:, h // group]
    return out


def _exact_resize(table, lens, want, refs, page):
    after = list(lens)
    for b, (n, w) in enumerate(zip(lens, want)):
        if w == 0:
            for j in range(_ceil(n, page)):
                refs[table[b][j]] -= 1
                table[b][j] = -1
            after[b] = 0
    cuts = [b for b, (n, w) in enumerate(zip(lens, want)) if 0 < w < n and (w % page == 0 or refs[table[b][w // page]] == 1)]
    for b in cuts:
        for j in range(_ceil(want[b], page), _ceil(lens[b], page)):
            refs[table[b][j]] -= 1
            table[b][j] = -1
        after[b] = want[b]
    free = [p for p, r in enumerate(refs) if r == 0]
    at = 0
    for b, (n, w) in enumerate(zip(lens, want)):
        if w <= n:
            continue
        first, last = _ceil(n, page), _ceil(w, page)
        at += last - first
        if last > first and at > len(free):
            continue
        for j in range(first, last):
            table[b][j] = free[at - last + j]
            refs[table[b][j]] = 1
        after[b] = w
    return after


def _exact_fork(table, lens, parents, children, refs, page):
    after, src, dst, at = list(lens), [], [], 0
    free = [p for p, r in enumerate(refs) if r == 0]
    for a, b in zip(parents, children):
        n = lens[a]
        src.append(-1)
        dst.append(-1)
        if n % page:
            at += 1
            if at > len(free):
                continue
            src[-1], dst[-1] = table[a][n // page], free[at - 1]
            refs[dst[-1]] = 1
            table[b][n // page] = dst[-1]
        for j in range(n // page):
            table[b][j] = table[a][j]
            refs[table[a][j]] += 1
        after[b] = n
    return after, src, dst


def _exact_compact(table, lens, refs, page):
    live = [p for p, r in enumerate(refs) if r > 0]
    holes = [p for p in range(len(live)) if refs[p] == 0]
    highs = [p for p in live if p >= len(live)]
    place = dict(zip(highs, holes))
    for a, b in place.items():
        refs[b], refs[a] = refs[a], 0
    for b, n in enumerate(lens):
        for j in range(_ceil(n, page)):
            table[b][j] = place.get(table[b][j], table[b][j])
    none = [-1] * (len(refs) // 2 - len(highs))
    return highs + none, holes + none
