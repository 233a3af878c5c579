"""Calls that are the first of their process, at sizes where a block's shared memory
ends at the 48 KB that need no leave: the arrays that a kernel declares count
too. What a process ran before may raise a kernel's limit, so each case has its own.
Results are whole numbers and equal the definition's."""
import os
import subprocess
import sys

import pytest

import hkv_b200 as H

pytestmark = pytest.mark.gpu

START = f"""
import sys
sys.path.insert(0, {os.path.dirname(os.path.abspath(H.__file__))!r})
import torch
import hkv_b200 as H
def i32(*shape): return torch.zeros(shape, dtype=torch.int32, device="cuda")
"""

SORT = """
n, groups = {n}, {groups}
ids = torch.randint(0, groups, (n,), generator=torch.Generator().manual_seed(n))
offsets, positions, order = i32(groups + 1), i32(n), i32(n)
H.group_tokens(n, ids.cuda(), groups, offsets, positions, order)
want = torch.sort(ids, stable=True).indices
assert torch.equal(order.cpu().long(), want)
assert torch.equal(positions.cpu().long()[want], torch.arange(n))
assert torch.equal(offsets.cpu().long()[1:], torch.bincount(ids, minlength=groups).cumsum(0))
"""

RESIZE = """
rows = {rows}
pool = H.PagePool([torch.zeros((2 * rows, {width}), dtype=torch.uint8, device="cuda")], 4, rows, 2)
every = torch.arange(rows, device="cuda", dtype=torch.int32)
status = torch.zeros(rows, dtype=torch.bool, device="cuda")
pool.resize(rows, every, torch.full_like(every, 5), status)
assert status.all() and (pool.refs == 1).all() and (pool.lengths == 5).all()
assert torch.equal(pool.table.view(-1), torch.arange(2 * rows, device="cuda", dtype=torch.int32))
"""

FORK = """
rows = {rows}
pool = H.PagePool([], 4, rows, 17, num_pages=17 * rows)
every = torch.arange(rows, device="cuda", dtype=torch.int32)
pool.resize(rows, every, every % 69)
lengths, table = pool.lengths.clone(), pool.table.clone()
pool.fork(rows, every, every.flip(0).contiguous())
assert torch.equal(pool.lengths, lengths.flip(0))
held = torch.arange(17, device="cuda")[None] < ((pool.lengths + 3) // 4)[:, None]
assert torch.equal(pool.table[held], table.flip(0)[held])
"""


def first_call(code):
    done = subprocess.run([sys.executable, "-c", START + code], capture_output=True, text=True,
                          timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]


@pytest.mark.parametrize("n,groups", [(512, 1024), (960, 576), (8192, 428), (20000, 214),
                                      (40000, 1168)])
def test_group_tokens(n, groups):
    first_call(SORT.format(n=n, groups=groups))


@pytest.mark.parametrize("rows,width", [(12288, 16), (12221, 5)])
def test_resize(rows, width):
    first_call(RESIZE.format(rows=rows, width=width))


def test_fork():
    first_call(FORK.format(rows=945))
