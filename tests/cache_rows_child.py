"""Child process of tests/test_cache_pages.py.

What a kernel may use of shared memory stays set for the rest of a process, so
each size of a bookkeeping call is its kernel's first here: the sizes that need
48 KB together with the kernel's static shared memory, in ascending order.
Prints "ok" if every call did what it should.
"""

from __future__ import annotations

import os
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
for path in (os.path.dirname(HERE), os.path.join(os.path.dirname(HERE), "hpc-ops-sm120_b200"), HERE):
    if path not in sys.path:
        sys.path.insert(0, path)

import torch  # noqa: E402

import attention_decode as ad  # noqa: E402


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def resize(rows):
    table = torch.full((rows, 1), -1, dtype=torch.int32, device="cuda")
    refs = torch.zeros(rows, dtype=torch.int32, device="cuda")
    none = torch.zeros(rows, dtype=torch.int32, device="cuda")
    lens = ad.cache_resize(table, none, none + 3, refs, page_size=8)
    assert lens.tolist() == [3] * rows and refs.tolist() == [1] * rows
    assert table[:, 0].tolist() == list(range(rows))


def fork(rows, forks):
    table = torch.full((rows, 1), -1, dtype=torch.int32, device="cuda")
    table[0] = 0
    refs = torch.zeros(forks + 1, dtype=torch.int32, device="cuda")
    refs[0] = 1
    lens = torch.zeros(rows, dtype=torch.int32, device="cuda")
    lens[0] = 8
    children = ints(list(range(1, rows)) + [0] * (forks - rows + 1))  # the last ones are refused
    after, src, dst = ad.cache_fork(table, lens, refs, ints([0] * forks), children, page_size=8)
    assert after.tolist() == [8] * rows and table[:, 0].tolist() == [0] * rows
    assert refs[0].item() == rows and (src == -1).all() and (dst == -1).all()


if __name__ == "__main__":
    which, *sizes = sys.argv[1:]
    for size in sizes:
        {"resize": resize, "fork": fork}[which](*map(int, size.split(",")))
    print("ok")
