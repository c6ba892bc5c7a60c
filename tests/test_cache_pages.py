"""The upkeep of a paged cache: writes, page copies, resize, fork and compact,
against plain Python on lists.  Every value is a copy or a whole number, so
results have to be equal."""

from __future__ import annotations

import os
import subprocess
import sys

import pytest
import torch

import attention_decode as ad
import serving_reference as ref

gpu = pytest.mark.gpu


def ints(values, device):
    return torch.tensor(values, dtype=torch.int32, device=device)


def flags():
    return ad.read_error_flag(torch.cuda.current_device())


def lengths(gen, rows, longest):
    """Lengths over the logarithm up to `longest`, some rows empty, some on page borders."""
    lens = (torch.rand(rows, generator=gen) * torch.log(torch.tensor(float(longest) + 1))).exp().int() - 1
    lens[torch.rand(rows, generator=gen) < 0.2] = 0
    lens[torch.rand(rows, generator=gen) < 0.2] = longest // 2
    return lens.tolist()


# ------------------------------------------------------------------ write
@gpu
@pytest.mark.parametrize("layout", ("HND", "NHD"))
@pytest.mark.parametrize("page,heads,dim", ((8, 8, 128), (16, 1, 64), (64, 3, 128), (256, 8, 64)))
def test_write_puts_tokens_in_their_pages(layout, page, heads, dim, device):
    flags()
    gen = torch.Generator().manual_seed(page + heads)
    new = [1, 0, 5, page + 3, 0, 2 * page, 1]
    starts = [0, 7, page - 2, 3 * page - 1, 0, page, 5 * page]
    table, refs = ref.random_rows(gen, [s + n for s, n in zip(starts, new)], 9, 3, page, share=False)
    shape = (len(refs), heads, page, dim) if layout == "HND" else (len(refs), page, heads, dim)
    k_cache, v_cache = (torch.randn(shape, generator=gen).to(device, torch.bfloat16) for _ in range(2))
    want = [k_cache.cpu(), v_cache.cpu()]
    rows = sum(new) + 4  # four rows of padding
    fused = torch.randn(rows, 2 * heads + 1, dim, generator=gen).to(torch.bfloat16)
    on = fused.to(device)
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    wide = torch.full((len(table), 12), 10**6, dtype=torch.int32)  # entries that no row has
    wide[:, :9] = ints(table, "cpu")
    ad.cache_write(on[:, 1 : heads + 1], on[:, heads + 1 :], k_cache, v_cache, wide.to(device)[:, :9], ints(cu, device),
                   ints(starts, device), layout=layout)
    for b, n in enumerate(new):
        for i in range(n):
            block, slot = table[b][(starts[b] + i) // page], (starts[b] + i) % page
            for cache, first in zip(want, (1, heads + 1)):
                place = cache[block, :, slot] if layout == "HND" else cache[block, slot]
                place.copy_(fused[cu[b] + i, first : first + heads])
    assert torch.equal(k_cache.cpu(), want[0]) and torch.equal(v_cache.cpu(), want[1])
    assert flags() == 0


@gpu
def test_write_leaves_out_tokens_without_a_page(device):
    flags()
    k_cache = torch.zeros(4, 2, 8, 64, dtype=torch.bfloat16, device=device)
    v_cache = torch.zeros_like(k_cache)
    k = torch.ones(6, 2, 64, dtype=torch.bfloat16, device=device)
    table = ints([[2, -1], [4, 0]], device)  # row 0 has one page, row 1's first is outside the pool
    ad.cache_write(k, k, k_cache, v_cache, table, ints([0, 4, 6], device), ints([6, 15], device))
    got = k_cache.float().sum((1, 3)).cpu()
    want = torch.zeros(4, 8)
    want[2, 6:] = 128  # positions 6, 7 of row 0; 8 and 9 have no page
    want[0, 7] = 128   # position 15 of row 1; 16 is behind the table
    assert torch.equal(got, want) and torch.equal(k_cache, v_cache)
    assert flags() == 16
    before = k_cache.clone()
    ad.cache_write(k[:2], k[:2], k_cache, v_cache, table, ints([0, 0, 2], device), ints([0, 0], device))
    ad.cache_write(k[:2], k[:2], k_cache, v_cache, table, ints([0, 2, 2], device), ints([-9, 0], device))
    assert torch.equal(k_cache, before) and flags() == 16


@gpu
def test_write_and_copy_past_32_bit_offsets(device):
    heads, page, dim = 8, 16, 128
    blocks = 2**31 // (heads * page * dim) + 3  # the last pages lie past 2^31 elements
    k_cache = torch.empty(blocks, heads, page, dim, dtype=torch.bfloat16, device=device)
    v_cache = torch.empty_like(k_cache)
    last = blocks - 1
    k = torch.randn(page, heads, dim, device=device).bfloat16()
    ad.cache_write(k, -k, k_cache, v_cache, ints([[last]], device), ints([0, page], device), ints([0], device))
    assert torch.equal(k_cache[last], k.transpose(0, 1)) and torch.equal(v_cache[last], -k.transpose(0, 1))
    ad.cache_copy_pages(k_cache, v_cache, ints([last, last], device), ints([0, last - 1], device))
    for b in (0, last - 1):
        assert torch.equal(k_cache[b], k_cache[last]) and torch.equal(v_cache[b], v_cache[last])


# ------------------------------------------------------------------ copies
@gpu
@pytest.mark.parametrize("shape", ((300, 1, 8, 64), (77, 8, 16, 128), (9, 4, 256, 128), (40, 3, 8, 64)))
@pytest.mark.parametrize("nhd", (False, True))
def test_copy_pages(shape, nhd, device):
    flags()
    blocks, heads, page, dim = shape
    shape = (blocks, page, heads, dim) if nhd else shape
    gen = torch.Generator().manual_seed(blocks)
    k_cache, v_cache = (torch.randn(shape, generator=gen).to(device, torch.bfloat16) for _ in range(2))
    want = [k_cache.clone(), v_cache.clone()]
    order = torch.randperm(blocks, generator=gen)
    half = blocks // 2
    src = order[:half][torch.randint(half, (blocks - half,), generator=gen)]  # sources may repeat
    dst = order[half:].clone()
    src[::3], dst[1::4] = -1, -1
    for a, b in zip(src.tolist(), dst.tolist()):
        if a >= 0 and b >= 0:
            for cache in want:
                cache[b] = cache[a]
    ad.cache_copy_pages(k_cache, v_cache, src.to(device, torch.int32), dst.to(device, torch.int32))
    assert torch.equal(k_cache, want[0]) and torch.equal(v_cache, want[1])
    assert flags() == 0
    ad.cache_copy_pages(k_cache, v_cache, ints([0, blocks, 1, -7], device), ints([blocks, 0, 1, 2], device))
    assert torch.equal(k_cache, want[0]) and torch.equal(v_cache, want[1])
    assert flags() == 16


# ------------------------------------------------------------------ bookkeeping
def state(gen, rows, longest, page, spare, device, width=None, share=True):
    lens = lengths(gen, rows, longest)
    width = width or ref.pages_of(longest, page) + 2
    table, refs = ref.random_rows(gen, lens, width, spare, page, share)
    return lens, table, refs, ints(table, device), ints(refs, device), ints(lens, device)


@gpu
@pytest.mark.parametrize("rows,longest,page,spare", (
    (1, 1, 8, 1), (1, 100, 8, 40), (7, 300, 16, 60), (33, 2000, 8, 3000), (300, 500, 64, 10), (3, 70000, 8, 20000),
    (2500, 40, 8, 4000), (64, 5000, 256, 100), (20, 900, 8, 300000), (16384, 9, 8, 9000),
))
@pytest.mark.parametrize("seed", (0, 1))
def test_resize(rows, longest, page, spare, seed, device):
    flags()
    gen = torch.Generator().manual_seed(1000 * seed + rows)
    lens, table, refs, dev_table, dev_refs, dev_lens = state(gen, rows, longest, page, spare, device)
    for step in range(4):
        want = list(lens)
        kinds = torch.rand(rows, generator=gen).tolist()
        amounts = torch.rand(rows, generator=gen).tolist()
        for b in range(rows):
            if kinds[b] < 0.15:
                want[b] = 0
            elif kinds[b] < 0.35:
                want[b] = int(amounts[b] * lens[b])
            elif kinds[b] < 0.8:
                want[b] = lens[b] + int(amounts[b] * (longest if kinds[b] < 0.5 else page))
            elif kinds[b] < 0.83:
                want[b] = -1
        after, bits = ref.resize(table, lens, want, refs, page)
        given = dev_lens.clone()
        got = ad.cache_resize(dev_table, dev_lens, ints(want, device), dev_refs, page_size=page)
        assert torch.equal(dev_lens, given)
        assert got.tolist() == after and dev_table.tolist() == table and dev_refs.tolist() == refs
        assert flags() == bits
        lens, dev_lens = after, got


@gpu
def test_resize_refuses_a_cut_into_a_page_that_another_row_holds(device):
    flags()
    table, refs = ints([[0, 1, -1], [0, 1, 2]], device), ints([2, 2, 1, 0], device)
    lens = ints([16, 20], device)
    got = ad.cache_resize(table, lens, ints([12, 8], device), refs, page_size=8)
    assert got.tolist() == [16, 8] and flags() == 64  # 8 is a border of pages
    assert table.tolist() == [[0, 1, -1], [0, -1, -1]] and refs.tolist() == [2, 1, 0, 0]
    got = ad.cache_resize(table, got, ints([12, 8], device), refs, page_size=8)
    assert got.tolist() == [12, 8] and flags() == 0
    # the row that leaves in the same call no longer holds it
    got = ad.cache_resize(table, got, ints([3, 0], device), refs, page_size=8)
    assert got.tolist() == [3, 0] and flags() == 0
    assert table.tolist() == [[0, -1, -1], [-1, -1, -1]] and refs.tolist() == [1, 0, 0, 0]


@gpu
def test_resize_follows_no_bad_page(device):
    flags()
    table, refs = ints([[5, -1, 0], [1, 2, -1]], device), ints([1, 0, 1], device)
    got = ad.cache_resize(table, ints([24, 16], device), ints([0, 0], device), refs, page_size=8)
    assert got.tolist() == [0, 0] and flags() == 16  # 5 and -1 are no pages, nobody held 1
    assert refs.tolist() == [0, 0, 0] and table.tolist() == [[-1, -1, -1]] * 2


@gpu
@pytest.mark.parametrize("rows,children,longest,page,spare", (
    (1, 1, 5, 8, 1), (2, 9, 100, 8, 4), (5, 40, 900, 16, 100), (8, 1500, 300, 64, 1400), (3, 30, 60000, 8, 29),
    (40, 1, 33, 32, 0), (3, 16381, 20, 8, 16000), (4, 20, 5000, 8, 300000),
))
def test_fork(rows, children, longest, page, spare, device):
    flags()
    gen = torch.Generator().manual_seed(rows + children)
    lens = lengths(gen, rows, longest) + [0] * children
    table, refs = ref.random_rows(gen, lens, ref.pages_of(longest, page) + 1, spare, page)
    dev_table, dev_refs, dev_lens = ints(table, device), ints(refs, device), ints(lens, device)
    parents = torch.randint(rows, (children,), generator=gen).tolist()
    kids = (rows + torch.randperm(children, generator=gen)).tolist()
    after, src, dst, bits = ref.fork(table, lens, refs, parents, kids, page)
    got, got_src, got_dst = ad.cache_fork(dev_table, dev_lens, dev_refs, ints(parents, device), ints(kids, device), page_size=page)
    assert got.tolist() == after and got_src.tolist() == src and got_dst.tolist() == dst
    assert dev_table.tolist() == table and dev_refs.tolist() == refs
    assert flags() == bits


@gpu
@pytest.mark.parametrize("call,sizes", (
    ("resize", ("4084", "4085", "4095", "4096", "4097")), ("fork", ("4084,4084", "4085,4084", "4095,4096", "4096,4096", "4097,4096")),
))
def test_rows_around_48_kb_of_shared_memory(call, sizes, device):
    """Three ints per row, or one per row and two per fork, beside what the kernel has of its own."""
    child = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cache_rows_child.py")
    proc = subprocess.run([sys.executable, child, call, *sizes], capture_output=True, text=True, timeout=600)
    assert proc.returncode == 0 and proc.stdout.split() == ["ok"], proc.stderr[-4000:]


@gpu
@pytest.mark.parametrize("page", (-1, -5, 9, 2**31 - 1))
def test_fork_follows_no_bad_page(page, device):
    """The parent's last, partly filled page is none of the pool: the child's own has no source."""
    flags()
    table, refs = ints([[3, page, -1], [-1, -1, -1]], device), ints([0, 0, 0, 1, 0, 0, 0, 0, 0], device)
    lens, src, dst = ad.cache_fork(table, ints([12, 0], device), refs, ints([0], device), ints([1], device), page_size=8)
    assert flags() == 16
    assert lens.tolist() == [12, 12] and src.tolist() == [-1] and dst.tolist() == [-1]
    assert table.tolist() == [[3, page, -1], [3, 0, -1]] and refs.tolist() == [1, 0, 0, 2, 0, 0, 0, 0, 0]


@gpu
def test_fork_refuses(device):
    """A child named twice, one that is not empty, rows that are not there, a row as its own child; a parent that is
    a child of the same call counts as empty."""
    flags()
    gen = torch.Generator().manual_seed(5)
    lens, page = [20, 9, 0, 0, 0, 0, 16], 8
    table, refs = ref.random_rows(gen, lens, 4, 6, page)
    parents = [0, 0, 1, 7, -1, 0, 2, 1, 6, 1]
    kids = [2, 2, 0, 3, 3, 7, 4, 1, 5, 3]
    dev_table, dev_refs = ints(table, device), ints(refs, device)
    after, src, dst, bits = ref.fork(table, lens, refs, parents, kids, page)
    got, got_src, got_dst = ad.cache_fork(dev_table, ints(lens, device), dev_refs, ints(parents, device), ints(kids, device), page_size=page)
    assert bits == 64 and flags() == 64
    assert got.tolist() == after and got_src.tolist() == src and got_dst.tolist() == dst
    assert dev_table.tolist() == table and dev_refs.tolist() == refs
    none = ints([], device)
    same, a, b = ad.cache_fork(dev_table, got, dev_refs, none, none, page_size=page)
    assert same.tolist() == after and a.numel() == b.numel() == 0


@gpu
@pytest.mark.parametrize("rows,longest,page,spare", (
    (1, 1, 8, 0), (1, 1, 8, 1), (1, 0, 8, 7), (6, 200, 8, 33), (30, 1000, 16, 2000), (500, 100, 8, 1), (4, 90000, 8, 9000),
    (30, 40000, 8, 250000),
))
def test_compact(rows, longest, page, spare, device):
    flags()
    gen = torch.Generator().manual_seed(rows + spare)
    lens, table, refs, dev_table, dev_refs, dev_lens = state(gen, rows, max(longest, 1), page, spare, device)
    if longest == 0:
        lens, table = [0] * rows, [[-1] * len(table[0]) for _ in table]
        refs = [0] * len(refs)
        dev_table, dev_refs, dev_lens = ints(table, device), ints(refs, device), ints(lens, device)
    if not refs:  # a pool without pages is refused
        with pytest.raises(RuntimeError, match="page_refs"):
            ad.cache_compact(dev_table, dev_lens, dev_refs, page_size=page)
        return
    if len(refs) > 3:  # a page that no row of the table holds, a prefix kept for later
        at = len(refs) - 1
        refs[at] += 1
        dev_refs[at] += 1
    src, dst = ref.compact(table, lens, refs, page)
    got_src, got_dst = ad.cache_compact(dev_table, dev_lens, dev_refs, page_size=page)
    assert got_src.tolist() == src and got_dst.tolist() == dst
    assert dev_table.tolist() == table and dev_refs.tolist() == refs
    assert flags() == 0
    again, _ = ad.cache_compact(dev_table, dev_lens, dev_refs, page_size=page)
    assert (again == -1).all() and dev_table.tolist() == table


@gpu
def test_rows_of_a_wider_table(device):
    """A view of a table, rows further apart than they are wide, another stream."""
    wide = torch.full((3, 10), 77, dtype=torch.int32, device=device)
    table = wide[:, 2:6]
    table.fill_(-1)
    refs, lens = torch.zeros(9, dtype=torch.int32, device=device), ints([0, 0, 0], device)
    side = torch.cuda.Stream(device)
    side.wait_stream(torch.cuda.current_stream(device))
    with torch.cuda.stream(side):
        lens = ad.cache_resize(table, lens, ints([9, 0, 8], device), refs, page_size=8)
        lens, src, dst = ad.cache_fork(table, lens, refs, ints([0], device), ints([1], device), page_size=8)
        lens = ad.cache_resize(table, lens, ints([0, 17, 8], device), refs, page_size=8)
        ad.cache_compact(table, lens, refs, page_size=8)
    side.synchronize()
    assert lens.tolist() == [0, 17, 8] and src.tolist() == [1] and dst.tolist() == [3]
    # after the resize: row 1 holds 0, 3 and 1 (freed by row 0), row 2 holds 2
    assert table.tolist() == [[-1] * 4, [0, 3, 1, -1], [2, -1, -1, -1]]
    assert refs.tolist() == [1, 1, 1, 1, 0, 0, 0, 0, 0]
    assert (wide[:, :2] == 77).all() and (wide[:, 6:] == 77).all()


# ------------------------------------------------------------------ refusals (host)
def cpu_state():
    table, lens, refs = torch.zeros(2, 4, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), torch.zeros(9, dtype=torch.int32)
    return table, lens, refs


def test_bookkeeping_refusals():
    table, lens, refs = cpu_state()
    with pytest.raises(TypeError, match="new_lens"):
        ad.cache_resize(table, lens, [1, 2], refs, page_size=8)
    with pytest.raises(RuntimeError, match="int32"):
        ad.cache_resize(table.long(), lens, lens, refs, page_size=8)
    with pytest.raises(RuntimeError, match="rank 2"):
        ad.cache_resize(lens, lens, lens, refs, page_size=8)
    with pytest.raises(RuntimeError, match="2 entries"):
        ad.cache_resize(table, refs, lens, refs, page_size=8)
    with pytest.raises(RuntimeError, match="contiguous"):
        ad.cache_resize(table.t(), torch.zeros(4, dtype=torch.int32), torch.zeros(4, dtype=torch.int32), refs, page_size=8)
    with pytest.raises(RuntimeError, match="distinct"):
        ad.cache_resize(table[:1].expand(2, 4), lens, lens, refs, page_size=8)
    with pytest.raises(RuntimeError, match="page_refs"):
        ad.cache_compact(table, lens, refs[:0], page_size=8)
    with pytest.raises(RuntimeError, match="children"):
        ad.cache_fork(table, lens, refs, lens, refs, page_size=8)
    for call in (
        lambda: ad.cache_resize(table, lens, lens, refs, page_size=8),
        lambda: ad.cache_fork(table, lens, refs, lens, lens, page_size=8),
        lambda: ad.cache_compact(table, lens, refs, page_size=8),
    ):
        with pytest.raises(ValueError, match="CUDA"):
            call()


def test_write_and_copy_refusals():
    table, lens, _ = cpu_state()
    cache = torch.zeros(4, 2, 8, 64, dtype=torch.bfloat16)
    k = torch.zeros(3, 2, 64, dtype=torch.bfloat16)
    cu = torch.zeros(3, dtype=torch.int32)
    good = dict(k=k, v=k, k_cache=cache, v_cache=cache, block_table=table, cu_seqlens=cu, starts=lens)
    for change, error, match in (
        (dict(layout="BHSD"), ValueError, "layout"),
        (dict(k=k.float()), RuntimeError, "BF16"),
        (dict(k=k[0]), RuntimeError, "rank 3"),
        (dict(v=k[:2]), RuntimeError, "shape"),
        (dict(v=torch.zeros(3, 64, 2, dtype=torch.bfloat16).transpose(1, 2)), RuntimeError, "contiguous"),
        (dict(k=torch.zeros(3, 2, 68, dtype=torch.bfloat16)[..., :64]), RuntimeError, "multiple of 8"),
        (dict(k=k[:1].expand(3, 2, 64)), RuntimeError, "expanded"),
        (dict(k=torch.zeros(3, 1, 64, dtype=torch.bfloat16), v=torch.zeros(3, 1, 64, dtype=torch.bfloat16)), RuntimeError, "heads"),
        (dict(k_cache=cache[:, :, :4]), RuntimeError, "match"),
        (dict(cu_seqlens=cu[:2]), RuntimeError, "3 entries"),
        (dict(starts=lens.long()), RuntimeError, "int32"),
        (dict(), ValueError, "CUDA"),
    ):
        with pytest.raises(error, match=match):
            ad.cache_write(**{**good, **change})
    with pytest.raises(RuntimeError, match="2 entries"):
        ad.cache_copy_pages(cache, cache, lens, cu)
    with pytest.raises(RuntimeError, match="shapes"):
        ad.cache_copy_pages(cache, cache[:2], lens, lens)
    with pytest.raises(ValueError, match="CUDA"):
        ad.cache_copy_pages(cache, cache, lens, lens)


def test_c_entry_points_refuse_on_the_host():
    from attention_decode import _lib

    lib = _lib.load_library()
    invalid, unsupported = _lib.ADB_ERR_INVALID_ARGUMENT, _lib.ADB_ERR_UNSUPPORTED
    p = 256  # an address that no refused call follows

    def resize(table=p, stride=4, batch=2, blocks=9, page=8, width=4, refs=p):
        return lib.adb_cache_resize(table, stride, p, p, refs, p, batch, blocks, page, width, 0, None)

    assert resize(table=None) == invalid and resize(refs=None) == invalid
    assert resize(stride=3) == invalid and b"stride" in lib.adb_last_error()
    assert resize(batch=0) == invalid and resize(batch=16385) == unsupported
    assert resize(page=12) == unsupported and b"power of two" in lib.adb_last_error()
    assert resize(page=4) == unsupported and resize(page=2**21) == unsupported
    assert resize(blocks=0) == invalid and resize(blocks=2**30 + 1) == invalid
    assert resize(stride=2**28, width=2**28) == invalid

    def fork(forks=1, children=p, dst=p):
        return lib.adb_cache_fork(p, 4, p, p, p, children, forks, p, p, dst, 2, 9, 8, 4, 0, None)

    assert fork(forks=0) == unsupported and fork(forks=16385) == unsupported
    assert fork(children=None) == invalid and fork(dst=None) == invalid
    assert lib.adb_cache_compact(p, 4, p, p, p, p, None, 2, 9, 8, 4, 0, None) == invalid
    assert lib.adb_cache_compact(p, 4, p, p, None, p, p, 2, 9, 8, 4, 0, None) == invalid

    def write(k=p, stride=128, heads=2, dim=64, layout=0, total=3, page=8):
        return lib.adb_cache_write(k, stride, 64, p, 128, 64, p, p, p, 4, p, p, total, 2, heads, dim, 9, page, 4, layout, 0, None)

    assert write(k=None) == invalid and write(k=264) == invalid and write(stride=100) == invalid
    assert write(layout=2) == invalid and write(dim=96) == unsupported and write(page=24) == unsupported
    assert write(total=0) == invalid and write(heads=0) == invalid

    def copy(k=p, count=1, size=2048):
        return lib.adb_cache_copy_pages(k, p, p, p, count, 9, size, 0, None)

    assert copy(k=None) == invalid and copy(count=0) == invalid and copy(size=100) == invalid and copy(k=8) == invalid


def test_write_refuses_more_heads_than_its_offsets_hold():
    from attention_decode import _lib

    lib = _lib.load_library()
    p = 256  # an address that no refused call follows

    def write(heads, blocks):
        return lib.adb_cache_write(p, heads * 64, 64, p, heads * 64, 64, p, p, p, 4, p, p, 3, 2, heads, 64, blocks, 8, 4, 0, 0, None)

    assert write(2**16 + 1, 9) == _lib.ADB_ERR_UNSUPPORTED and b"heads" in lib.adb_last_error()
    assert write(2**40, 2**30) == _lib.ADB_ERR_UNSUPPORTED
    assert write(2**16, 2**15) == _lib.ADB_ERR_INVALID_ARGUMENT  # num_blocks * heads
