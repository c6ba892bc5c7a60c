"""Prompt attention, packed and over pages, against 64 bits with the error bound
that the operator's roundings give (serving_reference.attend)."""

from __future__ import annotations

import math

import pytest
import torch

import attention_decode as ad
import serving_reference as ref

gpu = pytest.mark.gpu
HEADS = ((8, 8), (32, 8), (64, 8), (24, 8), (28, 4), (10, 2), (16, 1), (64, 1))


def ints(values, device):
    return torch.tensor(values, dtype=torch.int32, device=device)


def offsets(lens):
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return cu


def randn(gen, *shape):
    return torch.randn(shape, generator=gen, device=gen.device).bfloat16()


def check_packed(out, q, k, v, lens):
    cu = offsets(lens)
    for a, b in zip(cu, cu[1:]):
        want, bound = ref.attend(q[a:b], k[a:b], v[a:b], 0)
        ref.check_close(out[a:b], want, bound)
    assert (out[cu[-1] :] == 0).all()


@gpu
@pytest.mark.parametrize("dim", (64, 128))
@pytest.mark.parametrize("hq,hkv", HEADS)
@pytest.mark.parametrize("lens", ([1], [129], [0, 5, 0, 127, 1, 300, 0], [128, 256, 64]))
def test_packed(lens, hq, hkv, dim, device):
    gen = torch.Generator(device).manual_seed(sum(lens) + hq)
    rows = sum(lens) + 3
    q, k, v = randn(gen, rows, hq, dim), randn(gen, rows, hkv, dim), randn(gen, rows, hkv, dim)
    for t in (q, k, v):
        t[sum(lens) :] = float("nan")  # padding behind the last sequence
    out = ad.attention_prefill(q, k, v, ints(offsets(lens), device))
    check_packed(out, q, k, v, lens)
    assert torch.equal(out, ad.attention_prefill(q, k, v, ints(offsets(lens), device)))


@gpu
@pytest.mark.parametrize("hq,hkv,dim,lens", (
    (8, 2, 128, [5000]), (4, 4, 64, [2500, 3, 1111]), (2, 2, 128, [9001]), (32, 8, 128, [700] * 9 + [1]),
    (8, 8, 128, [17] * 200), (7, 1, 64, [3, 2] * 700), (8, 2, 64, [0, 70] * 128), (8, 2, 64, [40] * 256 + [300]),
    (8, 1, 128, [4000, 1, 1700]), (4, 1, 64, [2100]),
))
def test_packed_long_or_many(hq, hkv, dim, lens, device):
    gen = torch.Generator(device).manual_seed(len(lens))
    rows = sum(lens)
    q, k, v = randn(gen, rows, hq, dim), randn(gen, rows, hkv, dim), randn(gen, rows, hkv, dim)
    check_packed(ad.attention_prefill(q, k, v, ints(offsets(lens), device)), q, k, v, lens)


@gpu
@pytest.mark.parametrize("kind", ("fused", "head-major", "offset"))
def test_packed_strides(kind, device):
    gen = torch.Generator(device).manual_seed(3)
    lens, hq, hkv, dim = [70, 200], 12, 4, 128
    rows = sum(lens)
    if kind == "fused":
        qkv = randn(gen, rows, hq + 2 * hkv, dim)
        q, k, v = qkv[:, :hq], qkv[:, hq : hq + hkv], qkv[:, hq + hkv :]
    elif kind == "head-major":
        q, k, v = (randn(gen, h, rows, dim).transpose(0, 1) for h in (hq, hkv, hkv))
    else:
        q, k, v = (randn(gen, rows + 1, h + 1, dim + 8)[1:, 1:, 8:] for h in (hq, hkv, hkv))
    check_packed(ad.attention_prefill(q, k, v, ints(offsets(lens), device)), q, k, v, lens)


@gpu
@pytest.mark.parametrize("what", ("k scaled", "one key", "low scores", "equal", "large v"))
def test_packed_values(what, device):
    gen = torch.Generator(device).manual_seed(11)
    lens, hq, hkv, dim = [300, 140], 8, 2, 128
    rows = sum(lens)
    q, k, v = randn(gen, rows, hq, dim), randn(gen, rows, hkv, dim), randn(gen, rows, hkv, dim)
    if what == "k scaled":
        k = (k.float() * 8).bfloat16()
        k[150] *= 50
    elif what == "one key":  # weights of all other keys vanish
        k[40] = q[60:61, ::4] * 4
    elif what == "low scores":  # all scores far below zero
        q = q.abs() * 16
        k = -k.abs() * 16
    elif what == "equal":
        k.fill_(0)
    else:
        v = (v.float() * 2.0**100).bfloat16()
    out = ad.attention_prefill(q, k, v, ints(offsets(lens), device))
    check_packed(out, q, k, v, lens)


@gpu
@pytest.mark.parametrize("bad", (float("nan"), float("inf"), -float("inf")))
@pytest.mark.parametrize("at", (3, 100, 130, 299))
@pytest.mark.parametrize("where", ("k", "v", "q"))
def test_non_finite_values_stay_with_the_rows_that_see_them(where, at, bad, device):
    gen = torch.Generator(device).manual_seed(at)
    lens, hq, hkv, dim = [60, 300, 90], 8, 2, 128
    rows = sum(lens)
    cu = offsets(lens)
    q, k, v = randn(gen, rows, hq, dim), randn(gen, rows, hkv, dim), randn(gen, rows, hkv, dim)
    clean = ad.attention_prefill(q, k, v, ints(cu, device))
    token, head, column = cu[1] + at, 1, 17
    heads = slice(4, 8)  # the query heads of KV head 1
    {"k": k, "v": v, "q": q}[where][token, 5 if where == "q" else head, column] = bad
    out = ad.attention_prefill(q, k, v, ints(cu, device))
    touched = torch.zeros_like(out, dtype=torch.bool)
    if where == "q":
        touched[token, 5] = True
    elif where == "v":
        touched[token : cu[2], heads, column] = True
        got = out[token : cu[2], heads, column].float()
        assert torch.isnan(got).all() if math.isnan(bad) else (got == bad).all()
    else:
        touched[token : cu[2], heads] = True
    ref.check_close(out[~touched], clean[~touched].double(), 2.0**-6 * clean[~touched].double().abs() + 2.0**-6)
    if where == "k" and math.isnan(bad):
        assert torch.isnan(out[token : cu[2], heads].float()).all()
    before = out[: cu[1] + at]
    assert torch.isfinite(before).all() and torch.isfinite(out[cu[2] :]).all()


def make_pages(gen, lens, hkv, dim, page, layout, device, spare=3):
    cpu = torch.Generator().manual_seed(len(lens) + page)
    width = max(ref.pages_of(max(lens), page), 1) + 1
    table, refs = ref.random_rows(cpu, lens, width, spare, page, share=False)
    shape = (len(refs), hkv, page, dim) if layout == "HND" else (len(refs), page, hkv, dim)
    caches = [torch.full(shape, float("nan"), dtype=torch.bfloat16, device=device) for _ in range(2)]
    tokens = []
    for b, n in enumerate(lens):
        tokens.append((randn(gen, n, hkv, dim), randn(gen, n, hkv, dim)))
        ids = torch.tensor(table[b][: ref.pages_of(n, page)], dtype=torch.long, device=device)
        for cache, x in zip(caches, tokens[-1]):
            full = torch.full((len(ids) * page, hkv, dim), float("nan"), dtype=torch.bfloat16, device=device)
            full[:n] = x
            full = full.view(len(ids), page, hkv, dim)
            cache[ids] = full.transpose(1, 2) if layout == "HND" else full
    rows = torch.tensor(table, dtype=torch.int32)
    rows[rows < 0] = 10**6  # entries behind a row's pages are never followed
    return caches[0], caches[1], rows.to(device), tokens


def check_paged(out, q, tokens, new, total):
    cu = offsets(new)
    for b, n in enumerate(new):
        k, v = tokens[b]
        want, bound = ref.attend(q[cu[b] : cu[b + 1]], k, v, total[b] - n)
        ref.check_close(out[cu[b] : cu[b + 1]], want, bound)
    assert (out[cu[-1] :] == 0).all()


@gpu
@pytest.mark.parametrize("layout", ("HND", "NHD"))
@pytest.mark.parametrize("page", (8, 16, 64, 128, 512))
@pytest.mark.parametrize("hq,hkv,dim", ((32, 8, 128), (28, 4, 64), (8, 8, 64)))
def test_paged(layout, page, hq, hkv, dim, device):
    ad.read_error_flag(0)
    gen = torch.Generator(device).manual_seed(page)
    new = [1, 0, 5, 130, 1, 64, 3, 0]
    total = [1, 40, 700, 130, 257, 192, 2, 0]  # the last new tokens of row 6 outnumber its cache
    k_cache, v_cache, table, tokens = make_pages(gen, total, hkv, dim, page, layout, device)
    q = randn(gen, sum(new) + 5, hq, dim)
    out = ad.attention_prefill_paged(q, k_cache, v_cache, table, ints(offsets(new), device), ints(total, device), layout=layout)
    check_paged(out, q, tokens, new, total)
    assert ad.read_error_flag(0) == 0


@gpu
@pytest.mark.parametrize("layout", ("HND", "NHD"))
@pytest.mark.parametrize("new,total,hq,hkv,dim,page", (
    ([1], [20000], 8, 1, 128, 16),
    ([3, 1], [9000, 30001], 16, 2, 64, 64),
    ([600, 1, 1, 1], [9000, 17, 8000, 1], 8, 2, 128, 16),
    ([1] * 40, [50 * i + 1 for i in range(40)], 32, 8, 128, 32),
    ([200], [200], 4, 4, 128, 8),
    ([500], [90], 4, 4, 64, 16),  # most rows see no key, the first tiles none at all
    ([1] * 300 + [60], [7] * 300 + [5000], 4, 2, 64, 16),
    ([40, 300], [20000, 3000], 8, 1, 128, 16),
    ([2, 2, 2, 2], [1535, 1536, 1537, 40000], 2, 1, 64, 8),
))
def test_paged_long_or_mixed(layout, new, total, hq, hkv, dim, page, device):
    gen = torch.Generator(device).manual_seed(sum(total))
    k_cache, v_cache, table, tokens = make_pages(gen, total, hkv, dim, page, layout, device)
    q = randn(gen, sum(new), hq, dim)
    cu, lens = ints(offsets(new), device), ints(total, device)
    out = ad.attention_prefill_paged(q, k_cache, v_cache, table, cu, lens, layout=layout)
    check_paged(out, q, tokens, new, total)
    assert torch.equal(out, ad.attention_prefill_paged(q, k_cache, v_cache, table, cu, lens, layout=layout))


@gpu
@pytest.mark.parametrize("bad", (float("nan"), float("inf")))
@pytest.mark.parametrize("at", (5, 9000, 19950, 19999))
def test_non_finite_values_of_a_long_cache(at, bad, device):
    """One KV head and few rows: the cache is cut into parts, `at` lies in the first, a middle or the last one."""
    gen = torch.Generator(device).manual_seed(at)
    new, total, hq, dim, page = 100, 20000, 4, 128, 16
    k_cache, v_cache, table, tokens = make_pages(gen, [total], 1, dim, page, "HND", device)
    q = randn(gen, new, hq, dim)
    args = (table, ints([0, new], device), ints([total], device))
    clean = ad.attention_prefill_paged(q, k_cache, v_cache, *args)
    check_paged(clean, q, tokens, [new], [total])
    v_cache[table[0, at // page].long(), 0, at % page, 33] = bad
    out = ad.attention_prefill_paged(q, k_cache, v_cache, *args)
    first = max(0, at - (total - new))  # first new token that sees it
    touched = torch.zeros_like(out, dtype=torch.bool)
    touched[first:, :, 33] = True
    assert torch.equal(out[~touched], clean[~touched])
    got = out[first:, :, 33].float()
    assert torch.isnan(got).all() if math.isnan(bad) else (got == bad).all()


def scored(gen, heights, hq, hkv, dim):
    """q, k, v of which key j has a score of about heights[j], for every row."""
    n = len(heights)
    u = torch.randint(2, (dim,), generator=gen, device=gen.device).float() * 2 - 1
    q = (u * (1 + 0.25 * torch.randn(n, hq, dim, generator=gen, device=gen.device))).bfloat16()
    k = u * (heights.to(gen.device) / math.sqrt(dim))[:, None, None]
    k = (k + 0.5 * torch.randn(n, hkv, dim, generator=gen, device=gen.device)).bfloat16()
    return q, k, randn(gen, n, hkv, dim)


def heights(kind, n):
    """Scores that make the running maximum grow by far more than a factor of 2^8, several times, or not at all."""
    j = torch.arange(n).float()
    if kind == "rising":
        return -40 + 80 * torch.floor(12 * j / n) / 12
    if kind == "falling":
        return 40 - 80 * torch.floor(12 * j / n) / 12
    if kind == "waves":
        return 30 * torch.sin(j * (20 / n))
    at = {"first": 5, "middle": n // 2 - 100, "last": n - 10}[kind]
    return torch.where(j == at, 130.0, 0.0)  # by itself, whatever the others' weights: less than 2^-149 of its own


KINDS = ("rising", "falling", "waves", "first", "middle", "last")


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("hq,hkv,dim,lens", (
    (8, 2, 128, [700, 400]), (4, 4, 64, [900, 400]), (32, 4, 64, [500]), (2, 2, 128, [3000]), (4, 1, 64, [3500]),
))
def test_packed_growing_scores(kind, hq, hkv, dim, lens, device):
    gen = torch.Generator(device).manual_seed(lens[0])
    q, k, v = scored(gen, torch.cat([heights(kind, n) for n in lens]), hq, hkv, dim)
    check_packed(ad.attention_prefill(q, k, v, ints(offsets(lens), device)), q, k, v, lens)


@gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("page", (8, 16, 64))
@pytest.mark.parametrize("hq,hkv,dim,new,total", (
    (8, 2, 128, 150, 1100), (8, 8, 64, 150, 1100), (8, 2, 128, 3, 1100), (16, 2, 64, 3, 1100),
    (4, 1, 128, 100, 20000), (8, 1, 64, 5, 20000), (2, 2, 128, 200, 9000),
))
def test_paged_growing_scores(kind, page, hq, hkv, dim, new, total, device):
    """One and two tiles of rows, whole and cut into parts."""
    gen = torch.Generator(device).manual_seed(total + new)
    q, k, v = scored(gen, heights(kind, total), hq, hkv, dim)
    blocks = ref.pages_of(total, page)
    order = torch.randperm(blocks, generator=gen, device=device)
    caches = [torch.full((blocks, page, hkv, dim), float("nan"), dtype=torch.bfloat16, device=device) for _ in range(2)]
    at = torch.arange(total, device=device)
    for cache, x in zip(caches, (k, v)):
        cache[order[at // page], at % page] = x
    args = (*caches, order.int()[None], ints([0, new], device), ints([total], device))
    out = ad.attention_prefill_paged(q[-new:].contiguous(), *args, layout="NHD")
    check_paged(out, q[-new:], [(k, v)], [new], [total])


@gpu
@pytest.mark.parametrize("bad", (float("nan"), float("inf"), -float("inf")))
@pytest.mark.parametrize("hq,hkv,dim,page,new,total,seen,later,border", (
    (8, 8, 128, 16, 256, 8260, 8010, 8100, 8064), (8, 8, 64, 64, 256, 9316, 9100, 9300, 9216),
    (8, 2, 128, 8, 64, 9246, 9200, 9230, 9216), (8, 2, 64, 32, 64, 9246, 9200, 9230, 9216),
))
def test_non_finite_values_on_both_sides_of_a_part(hq, hkv, dim, page, new, total, seen, later, border, bad, device):
    """The last part starts at key `border`, among the new tokens: rows between see `seen`, no key of that part, and not
    its non-finite value either."""
    gen = torch.Generator(device).manual_seed(total)
    k_cache, v_cache, table, tokens = make_pages(gen, [total], hkv, dim, page, "HND", device)
    q = randn(gen, new, hq, dim)
    args = (table, ints([0, new], device), ints([total], device))
    clean = ad.attention_prefill_paged(q, k_cache, v_cache, *args)
    check_paged(clean, q, tokens, [new], [total])
    head, heads = hkv - 1, slice((hkv - 1) * (hq // hkv), hq)
    for key, column in ((seen, 33), (later, 50)):
        v_cache[table[0, key // page].long(), head, key % page, column] = bad
    out = ad.attention_prefill_paged(q, k_cache, v_cache, *args)
    touched = torch.zeros_like(out, dtype=torch.bool)
    first = {}
    for key, column in ((seen, 33), (later, 50)):
        first[column] = key - (total - new)
        touched[first[column] :, heads, column] = True
    assert first[33] < border - (total - new) <= first[50]
    assert torch.equal(out[~touched], clean[~touched])
    got = out[touched].float()
    assert torch.isnan(got).all() if math.isnan(bad) else (got == bad).all()


@gpu
def test_paged_agrees_with_decode(device):
    gen = torch.Generator(device).manual_seed(2)
    total = [1, 17, 1000, 4097, 64]
    k_cache, v_cache, table, tokens = make_pages(gen, total, 8, 128, 16, "HND", device)
    q = randn(gen, len(total), 32, 128)
    out = ad.attention_prefill_paged(q, k_cache, v_cache, table, ints(range(len(total) + 1), device), ints(total, device))
    check_paged(out, q, tokens, [1] * len(total), total)
    step = ad.attention_decode_paged(q[:, :, None], k_cache, v_cache, table, ints(total, device))
    check_paged(step[:, :, 0], q, tokens, [1] * len(total), total)


@gpu
def test_paged_bad_pages_count_as_zeros(device):
    ad.read_error_flag(0)
    gen = torch.Generator(device).manual_seed(4)
    k_cache, v_cache, table, tokens = make_pages(gen, [200], 2, 64, 16, "HND", device)
    blocks = k_cache.shape[0]
    table[0, 3], table[0, 7], table[0, 12] = -1, blocks, 2**31 - 1
    k, v = tokens[0]
    for j in (3, 7, 12):
        k[16 * j : 16 * j + 16] = 0
        v[16 * j : 16 * j + 16] = 0
    q = randn(gen, 150, 8, 64)
    out = ad.attention_prefill_paged(q, k_cache, v_cache, table, ints([0, 150], device), ints([200], device))
    check_paged(out, q, tokens, [150], [200])
    assert ad.read_error_flag(0) == 16


@gpu
def test_lengths_outside_their_range_are_clamped(device):
    gen = torch.Generator(device).manual_seed(6)
    q, k, v = randn(gen, 50, 4, 64), randn(gen, 50, 2, 64), randn(gen, 50, 2, 64)
    out = ad.attention_prefill(q, k, v, ints([0, 20, 90], device))  # ends behind the tensor
    check_packed(out, q, k, v, [20, 30])
    k_cache, v_cache, table, tokens = make_pages(gen, [32, 16], 2, 64, 16, "HND", device)
    table = table[:, :2].contiguous()  # room for 32 tokens
    out = ad.attention_prefill_paged(q, k_cache, v_cache, table, ints([0, 4, 6], device), ints([40, -3], device))
    check_paged(out, q, [tokens[0], tuple(x[:0] for x in tokens[1])], [4, 2], [32, 0])


@gpu
def test_paged_past_32_bit_offsets(device):
    hkv, page, dim = 8, 16, 128
    blocks = 2**31 // (hkv * page * dim) + 2
    gen = torch.Generator(device).manual_seed(9)
    k_cache = torch.empty(blocks, hkv, page, dim, dtype=torch.bfloat16, device=device)
    v_cache = torch.empty_like(k_cache)
    ids = [blocks - 1, 0, blocks - 2]
    k, v = randn(gen, 3 * page, hkv, dim), randn(gen, 3 * page, hkv, dim)
    table = ints([ids], device)
    ad.cache_write(k, v, k_cache, v_cache, table, ints([0, 3 * page], device), ints([0], device))
    q = randn(gen, 20, 32, dim)
    out = ad.attention_prefill_paged(q, k_cache, v_cache, table, ints([0, 20], device), ints([3 * page - 5], device))
    check_paged(out, q, [(k[:-5], v[:-5])], [20], [3 * page - 5])


@gpu
def test_captured_calls_follow_their_inputs(device):
    """Two captured graphs and eager calls between their replays, lengths changed in place."""
    gen = torch.Generator(device).manual_seed(8)
    q, k, v = randn(gen, 300, 8, 128), randn(gen, 300, 2, 128), randn(gen, 300, 2, 128)
    cu = ints([0, 100, 300], device)
    total, new = [6000, 300], [4, 2]
    k_cache, v_cache, table, tokens = make_pages(gen, total, 2, 128, 16, "NHD", device)
    step_q, step_cu, lens = randn(gen, 6, 8, 128), ints([0, 4, 6], device), ints(total, device)

    def packed():
        return ad.attention_prefill(q, k, v, cu)

    def paged():
        return ad.attention_prefill_paged(step_q, k_cache, v_cache, table, step_cu, lens, layout="NHD")

    packed(), paged()
    torch.cuda.synchronize()
    graphs = []
    for call in (packed, paged):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            result = call()
        graphs.append((graph, result))
    for cuts, sizes in (([0, 100, 300], total), ([0, 0, 257], [5999, 299]), ([0, 290, 291], [130, 2])):
        cu.copy_(ints(cuts, device))
        lens.copy_(ints(sizes, device))
        for graph, result in graphs:
            result.fill_(7)
            graph.replay()
        check_packed(graphs[0][1], q, k, v, [b - a for a, b in zip(cuts, cuts[1:])])
        cut = [tuple(x[:n] for x in t) for t, n in zip(tokens, sizes)]
        check_paged(graphs[1][1], step_q, cut, new, sizes)
        assert torch.equal(packed(), graphs[0][1]) and torch.equal(paged(), graphs[1][1])


@gpu
def test_streams_run_side_by_side(device):
    gen = torch.Generator(device).manual_seed(21)
    total = [12000]
    k_cache, v_cache, table, tokens = make_pages(gen, total, 2, 128, 16, "HND", device)
    q = [randn(gen, 2, 8, 128) for _ in range(4)]
    cu, lens = ints([0, 2], device), ints(total, device)
    streams = [torch.cuda.Stream(device) for _ in q]
    torch.cuda.synchronize()
    out = [[] for _ in q]
    for _ in range(20):
        for x, stream, results in zip(q, streams, out):
            with torch.cuda.stream(stream):
                results.append(ad.attention_prefill_paged(x, k_cache, v_cache, table, cu, lens))
    torch.cuda.synchronize()
    for x, results in zip(q, out):
        check_paged(results[0], x, tokens, [2], total)
        assert all(torch.equal(r, results[0]) for r in results)


@gpu
def test_no_tokens(device):
    empty = torch.empty(0, 8, 64, dtype=torch.bfloat16, device=device)
    assert ad.attention_prefill(empty, empty, empty, ints([0, 0], device)).shape == (0, 8, 64)
    some = torch.ones(3, 8, 64, dtype=torch.bfloat16, device=device)
    assert (ad.attention_prefill(some, some, some, ints([0], device)) == 0).all()
    assert (ad.attention_prefill(some, some, some, ints([0, 0, 0], device)) == 0).all()
    cache = torch.zeros(2, 8, 8, 64, dtype=torch.bfloat16, device=device)
    table = ints([[0]], device)
    assert ad.attention_prefill_paged(empty, cache, cache, table, ints([0, 0], device), ints([3], device)).numel() == 0
    assert (ad.attention_prefill_paged(some, cache, cache, table, ints([0, 0], device), ints([3], device)) == 0).all()


# ------------------------------------------------------------------ a serving loop
@gpu
@pytest.mark.parametrize("layout", ("HND", "NHD"))
def test_a_serving_loop(layout, device):
    """Prompts in, chunked; beams fork; rows finish; the pool is compacted; decode steps read the result.  The plain
    side keeps each row's K/V as one tensor."""
    ad.read_error_flag(0)
    gen = torch.Generator(device).manual_seed(31)
    hq, hkv, dim, page, rows, layers = 8, 2, 128, 16, 6, 2
    table = torch.full((rows, 40), -1, dtype=torch.int32, device=device)
    refs = torch.zeros(120, dtype=torch.int32, device=device)
    shape = (120, hkv, page, dim) if layout == "HND" else (120, page, hkv, dim)
    caches = [[torch.full(shape, float("nan"), dtype=torch.bfloat16, device=device) for _ in range(2)] for _ in range(layers)]
    lens = torch.zeros(rows, dtype=torch.int32, device=device)
    plain = [[(torch.empty(0, hkv, dim, dtype=torch.bfloat16, device=device),) * 2 for _ in range(rows)] for _ in range(layers)]

    def step(new, lens):
        count = [sum(new)]
        want = lens + ints(new, device)
        after = ad.cache_resize(table, lens, want, refs, page_size=page)
        assert torch.equal(after, want)
        cu = ints(offsets(new), device)
        for layer, (k_cache, v_cache) in enumerate(caches):
            q, k, v = randn(gen, count[0], hq, dim), randn(gen, count[0], hkv, dim), randn(gen, count[0], hkv, dim)
            ad.cache_write(k, v, k_cache, v_cache, table, cu, lens, layout=layout)
            at = offsets(new)
            for b, n in enumerate(new):
                old = plain[layer][b]
                plain[layer][b] = (torch.cat([old[0], k[at[b] : at[b + 1]]]), torch.cat([old[1], v[at[b] : at[b + 1]]]))
            out = ad.attention_prefill_paged(q, k_cache, v_cache, table, cu, after, layout=layout)
            check_paged(out, q, plain[layer], new, after.tolist())
            if all(n == 1 for n in new):
                single = ad.attention_decode_paged(q[:, :, None], k_cache, v_cache, table, after, layout=layout)
                check_paged(single[:, :, 0], q, plain[layer], new, after.tolist())
            if lens.sum() == 0:
                check_packed(ad.attention_prefill(q, k, v, cu), q, k, v, new)
        return after

    lens = step([100, 33, 0, 0, 0, 16], lens)
    lens = step([200, 1, 0, 0, 0, 1], lens)
    lens, src, dst = ad.cache_fork(table, lens, refs, ints([0, 1, 1], device), ints([3, 2, 4], device), page_size=page)
    for layer, (k_cache, v_cache) in enumerate(caches):
        ad.cache_copy_pages(k_cache, v_cache, src, dst)
        for a, b in ((0, 3), (1, 2), (1, 4)):
            plain[layer][b] = plain[layer][a]
    lens = step([1] * rows, lens)
    lens = step([1, 20, 5, 1, 0, 3], lens)
    gone = lens.clone()
    gone[0] = gone[4] = 0
    lens = ad.cache_resize(table, lens, gone, refs, page_size=page)
    for layer in range(layers):
        for b in (0, 4):
            plain[layer][b] = tuple(x[:0] for x in plain[layer][b])
    src, dst = ad.cache_compact(table, lens, refs, page_size=page)
    for k_cache, v_cache in caches:
        ad.cache_copy_pages(k_cache, v_cache, src, dst)
    live = int((refs > 0).sum())
    assert (refs[:live] > 0).all() and (refs[live:] == 0).all()
    lens = step([50, 1, 1, 1, 40, 1], lens)
    lens = step([1] * rows, lens)
    assert ad.read_error_flag(0) == 0


# ------------------------------------------------------------------ refusals (host)
def test_prefill_refusals():
    q, k = torch.zeros(6, 8, 64, dtype=torch.bfloat16), torch.zeros(6, 2, 64, dtype=torch.bfloat16)
    cu = torch.tensor([0, 6], dtype=torch.int32)
    good = dict(q=q, k=k, v=k, cu_seqlens=cu)
    for change, error, match in (
        (dict(q=None), TypeError, "Q must be a tensor"),
        (dict(q=q.half()), RuntimeError, "BF16"),
        (dict(q=q[0]), RuntimeError, "rank 3"),
        (dict(q=q.clone().requires_grad_()), RuntimeError, "forward inference only"),
        (dict(k=k[:5], v=k[:5]), RuntimeError, "tokens"),
        (dict(v=torch.zeros(6, 4, 64, dtype=torch.bfloat16)), RuntimeError, "shape"),
        (dict(q=torch.zeros(6, 9, 64, dtype=torch.bfloat16)), RuntimeError, "divisible"),
        (dict(q=torch.zeros(6, 8, 96, dtype=torch.bfloat16)), RuntimeError, "64 or 128"),
        (dict(q=torch.zeros(6, 8, 65, dtype=torch.bfloat16)[..., 1:]), RuntimeError, "multiple of 8"),
        (dict(cu_seqlens=cu.long()), RuntimeError, "int32"),
        (dict(cu_seqlens=cu[:0]), RuntimeError, "batch"),
        (dict(), ValueError, "CUDA"),
    ):
        with pytest.raises(error, match=match):
            ad.attention_prefill(**{**good, **change})
    cache = torch.zeros(4, 2, 8, 64, dtype=torch.bfloat16)
    table, lens = torch.zeros(1, 4, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    good = dict(q=q, k_cache=cache, v_cache=cache, block_table=table, cu_seqlens=cu, seqlens=lens)
    for change, error, match in (
        (dict(layout="DNH"), ValueError, "layout"),
        (dict(k_cache=cache.float()), RuntimeError, "BF16"),
        (dict(k_cache=cache[:2]), RuntimeError, "match"),
        (dict(k_cache=cache.transpose(1, 2), v_cache=cache.transpose(1, 2)), RuntimeError, "contiguous"),
        (dict(q=torch.zeros(6, 8, 128, dtype=torch.bfloat16)), RuntimeError, "head dimension"),
        (dict(q=torch.zeros(6, 7, 64, dtype=torch.bfloat16)), RuntimeError, "divisible"),
        (dict(block_table=table[0]), RuntimeError, "rank 2"),
        (dict(seqlens=torch.zeros(2, dtype=torch.int32)), RuntimeError, "1 entries"),
        (dict(cu_seqlens=torch.zeros(3, dtype=torch.int32)), RuntimeError, "2 entries"),
        (dict(), ValueError, "CUDA"),
    ):
        with pytest.raises(error, match=match):
            ad.attention_prefill_paged(**{**good, **change})


def test_c_entry_points_refuse_on_the_host():
    import ctypes

    from attention_decode import _lib

    lib = _lib.load_library()
    invalid, unsupported = _lib.ADB_ERR_INVALID_ARGUMENT, _lib.ADB_ERR_UNSUPPORTED
    p = 256  # an address that no refused call follows

    def packed(q=p, stride=512, total=6, batch=1, hq=8, hkv=2, dim=64, cu=p):
        return lib.adb_prefill(q, stride, 64, p, 128, 64, p, 128, 64, cu, p, total, batch, hq, hkv, dim, p, 0, 0, None)

    assert packed(q=None) == invalid and packed(cu=None) == invalid
    assert packed(q=264) == invalid and packed(stride=513) == invalid
    assert packed(total=0) == invalid and packed(batch=0) == invalid and packed(hq=9) == invalid
    assert packed(hq=130) == unsupported and b"64" in lib.adb_last_error()
    assert packed(dim=96) == unsupported and packed(total=2**29) == invalid

    def paged(table=p, page=8, layout=0, stride=4, blocks=9, width=4):
        return lib.adb_prefill_paged(p, 512, 64, p, p, table, stride, p, p, p, 6, 1, 8, 2, 64, blocks, page, width,
                                     layout, p, 0, 0, None)

    assert paged(table=None) == invalid and paged(layout=3) == invalid and paged(stride=3) == invalid
    assert paged(page=7) == unsupported and paged(page=24) == unsupported
    assert paged(blocks=0) == invalid and paged(blocks=2**30) == invalid and paged(width=2**28, stride=2**28) == invalid
    size = ctypes.c_size_t(0)
    assert lib.adb_prefill_workspace_size(6, 1, 9, 2, 64, 0, 0, ctypes.byref(size)) == invalid
    assert lib.adb_prefill_workspace_size(6, 1, 8, 2, 64, 0, 0, None) == invalid
    assert lib.adb_prefill_workspace_size(6, 1, 8, 2, 64, -1, 0, ctypes.byref(size)) == invalid
