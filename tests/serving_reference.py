"""Plain implementations of the operators around a paged cache: attention in 64
bits with the error that the BF16 kernel may make, and the page bookkeeping on
Python lists."""

from __future__ import annotations

import math

import torch


def attend(q, k, v, before):
    """Attention of q [n, Hq, D] over k, v [m, Hkv, D], token i seeing the first
    before + i + 1 keys; (result, bound), both float64.

    The bound per element, from the roundings that the operator makes, with
    w_j the exact weights, A = sum_j w_j |v_j|:
      * the weights are rounded to BF16 before the product with V (half a step
        is 2^-8 of the value): 2^-8 A;
      * the output is rounded to BF16: 2^-8 |o|;
      * FP32 sums that round each step by at most 2^-23: D of them in a score,
        which move its exponent by (D + 4) 2^-23 sum_d |q_d k_d| / sqrt(D), twice
        because the total moves as well; m of them in the product and m in the
        total: 2 m 2^-23 A;
      * 2^-16 A for the exponential (approximated to 2^-17 or better) in
        numerator and total.
    """
    n, hq, d = q.shape
    m, hkv = k.shape[0], k.shape[1]
    q, k, v = q.double(), k.double(), v.double()
    out = torch.zeros_like(q)
    bound = torch.zeros_like(q)
    limit = (before + 1 + torch.arange(n, device=q.device)).clamp(0, m)
    hidden = torch.arange(m, device=q.device)[None, :] >= limit[:, None]
    for h in range(hq):
        keys, values = k[:, h // (hq // hkv)], v[:, h // (hq // hkv)]
        scores = (q[:, h] @ keys.T / math.sqrt(d)).masked_fill(hidden, -math.inf)
        top = scores.amax(-1, keepdim=True) if m else scores.new_zeros(n, 1)
        weights = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
        total = weights.sum(-1, keepdim=True)
        weights = torch.where(total > 0, weights / total, 0.0)
        out[:, h] = weights @ values
        spread = (q[:, h].abs() @ keys.abs().T / math.sqrt(d)).masked_fill(hidden, 0.0)
        moved = torch.expm1(2 * (d + 4) * 2.0**-23 * spread)
        size = weights @ values.abs()
        bound[:, h] = (
            2.0**-8 * (size + out[:, h].abs()) * (1 + 2.0**-7)
            + (weights * moved) @ values.abs()
            + moved.mul(weights).sum(-1, keepdim=True) * size
            + (2 * m * 2.0**-23 + 2.0**-16) * size
        )
    return out, bound


def check_close(got, want, bound):
    assert got.dtype == torch.bfloat16
    assert torch.isfinite(got).all(), "output contains NaN or Inf"
    error = (got.double() - want).abs()
    worst = (error - bound).max().item() if error.numel() else 0.0
    assert worst <= 0, f"error exceeds its bound by {worst}; largest error {error.max().item()}"


def pages_of(n, page):
    return -(-n // page)


def resize(table, lens, want, refs, page):
    """(lengths after, error bits); table and refs are changed."""
    width, after, bits = len(table[0]), list(lens), 0
    for b, w in enumerate(want):
        if w == 0:
            for j in range(pages_of(lens[b], page)):
                refs[table[b][j]] -= 1
                table[b][j] = -1
            after[b] = 0
        elif w < 0 or w > width * page:
            bits |= 64
    cuts = []
    for b, w in enumerate(want):
        if 0 < w < lens[b]:
            if w % page and refs[table[b][w // page]] > 1:
                bits |= 64
            else:
                cuts.append(b)
    for b in cuts:
        for j in range(pages_of(want[b], page), pages_of(lens[b], page)):
            refs[table[b][j]] -= 1
            table[b][j] = -1
        after[b] = want[b]
    free = [p for p, r in enumerate(refs) if r == 0]
    taken = 0
    for b, w in enumerate(want):
        if not lens[b] < w <= width * page:
            continue
        first, last = pages_of(lens[b], page), pages_of(w, page)
        taken += last - first
        if last > first and taken > len(free):
            bits |= 32
            continue
        for j in range(first, last):
            table[b][j] = free[taken - last + j]
            refs[table[b][j]] = 1
        after[b] = w
    return after, bits


def fork(table, lens, refs, parents, children, page):
    """(lengths after, copies from, copies to, error bits)."""
    after, src, dst, bits = list(lens), [], [], 0
    free = [p for p, r in enumerate(refs) if r == 0]
    named, taken = set(), 0
    for a, c in zip(parents, children):
        src.append(-1)
        dst.append(-1)
        seen = c in named
        named.add(c)
        if not (0 <= a < len(lens) and 0 <= c < len(lens)) or seen or lens[c]:
            bits |= 64
            continue
        n = lens[a]
        if n % page:
            taken += 1
            if taken > len(free):
                bits |= 32
                continue
            src[-1], dst[-1] = table[a][n // page], free[taken - 1]
            table[c][n // page] = dst[-1]
            refs[dst[-1]] = 1
        for j in range(n // page):
            table[c][j] = table[a][j]
            refs[table[a][j]] += 1
        after[c] = n
    return after, src, dst, bits


def compact(table, lens, refs, page):
    """(copies from, copies to)."""
    live = [p for p, r in enumerate(refs) if r > 0]
    holes = [p for p in range(len(live)) if refs[p] == 0]
    highs = [p for p in live if p >= len(live)]
    for a, b in zip(highs, holes):
        refs[b], refs[a] = refs[a], 0
    to = dict(zip(highs, holes))
    for b, n in enumerate(lens):
        for j in range(pages_of(n, page)):
            table[b][j] = to.get(table[b][j], table[b][j])
    none = [-1] * (len(refs) // 2 - len(highs))
    return highs + none, holes + none


def random_rows(gen, lens, width, spare, page, share=True):
    """A table of randomly placed pages for `lens` (a row may share leading full
    pages with the one before it) and its counts, as lists."""
    draw = lambda n: int(torch.randint(n, (1,), generator=gen))  # noqa: E731
    shared = [0] * len(lens)
    for b in range(1, len(lens)):
        if share and draw(3) == 0:
            shared[b] = draw(min(lens[b - 1], lens[b]) // page + 1)
    count = sum(pages_of(n, page) - s for n, s in zip(lens, shared)) + spare
    order = torch.randperm(count, generator=gen).tolist()
    table = [[-1] * width for _ in lens]
    refs = [0] * count
    for b, n in enumerate(lens):
        for j in range(pages_of(n, page)):
            table[b][j] = table[b - 1][j] if j < shared[b] else order.pop()
            refs[table[b][j]] += 1
    return table, refs
