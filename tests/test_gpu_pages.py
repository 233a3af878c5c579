"""The page pool against a model of its rules in plain Python, state for state
after every call. All results are whole numbers or copied bytes, so equal."""
import ctypes

import numpy as np
import pytest
import torch

import hkv_b200 as H

pytestmark = pytest.mark.gpu


def ceil_div(a, b):
    return -(-a // b)


class Model:
    """The rules of include/hkv_b200.h, one number at a time."""

    def __init__(self, pages, size, rows, width, planes):
        self.size, self.width = size, width
        self.refs = [0] * pages
        self.table = [[-1] * width for _ in range(rows)]
        self.lengths = [0] * rows
        self.planes = planes  # numpy [planes, pages, bytes]

    def held(self, row):
        return self.table[row][:ceil_div(self.lengths[row], self.size)]

    def count(self, pages, by):
        for p in pages:
            if 0 <= p < len(self.refs):
                self.refs[p] += by

    def copy(self, src, dst):
        before = self.planes.copy()
        for s, d in zip(src, dst):
            if 0 <= s < len(self.refs) and 0 <= d < len(self.refs):
                self.planes[:, d] = before[:, s]

    def entries(self, rows):
        """List entries that count: rows that exist, the last of each."""
        last = {r: k for k, r in enumerate(rows)}
        return [k for k, r in enumerate(rows) if 0 <= r < len(self.lengths) and last[r] == k]

    def fork(self, src, dst):
        rows = [list(r) for r in self.table]
        lengths = list(self.lengths)
        for k in self.entries(dst):
            s, d = src[k], dst[k]
            if not 0 <= s < len(lengths):
                continue
            new = rows[s][:ceil_div(lengths[s], self.size)]
            self.count(new, 1)
            self.count(rows[d][:ceil_div(lengths[d], self.size)], -1)
            self.table[d][:len(new)] = new
            self.lengths[d] = lengths[s]

    def resize(self, rows, lengths):
        refs = list(self.refs)
        free = [p for p, c in enumerate(refs) if c == 0]
        counts, status, wanted = set(self.entries(rows)), [], 0
        for k, (r, n) in enumerate(zip(rows, lengths)):
            if k not in counts or n < 0 or n > self.width * self.size:
                status.append(False)
                continue
            old, have = self.lengths[r], self.held(r)
            want = ceil_div(n, self.size)
            shared = n > old and old % self.size and refs[have[-1]] > 1
            need = max(0, want - len(have)) + bool(shared)
            wanted += need
            status.append(need == 0 or wanted <= len(free))
            if not status[-1]:
                continue
            given = free[wanted - need:wanted]
            if shared:
                page = given.pop(0)
                self.planes[:, page] = self.planes[:, have[-1]]
                self.refs[have[-1]] -= 1
                self.refs[page] = 1
                self.table[r][len(have) - 1] = page
            for j, page in zip(range(len(have), want), given):
                self.table[r][j] = page
                self.refs[page] = 1
            self.count(have[want:], -1)
            self.lengths[r] = n
        return status

    def free(self, rows):
        for r in rows:
            if 0 <= r < len(self.lengths):
                self.count(self.held(r), -1)
                self.lengths[r] = 0

    def compact(self):
        live = sum(c > 0 for c in self.refs)
        holes = [p for p in range(live) if self.refs[p] == 0]
        movers = [p for p in range(live, len(self.refs)) if self.refs[p] > 0]
        page_map = [p if c > 0 else -1 for p, c in enumerate(self.refs)]
        for to, page in zip(holes, movers):
            page_map[page] = to
            self.planes[:, to] = self.planes[:, page]
            self.refs[to], self.refs[page] = self.refs[page], 0
        for r in range(len(self.lengths)):
            held = self.held(r)
            self.table[r][:len(held)] = [page_map[p] if 0 <= p < len(page_map) else -1
                                         for p in held]
        return page_map


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


class Both:
    """A pool and its model, compared after each call."""

    def __init__(self, pages, size, rows, width, plane_bytes=(64, 48), seed=0, allocator=None):
        rng = np.random.default_rng(seed)
        sizes = list(plane_bytes)
        self.tensors = [torch.from_numpy(rng.integers(0, 256, (pages, b), dtype=np.uint8)).cuda()
                        for b in sizes]
        self.pool = H.PagePool(self.tensors, size, rows, width, num_pages=pages,
                               allocator=allocator)
        self.models = [t.cpu().numpy() for t in self.tensors]
        joined = np.concatenate(self.models, 1)[None] if sizes else np.zeros((1, pages, 0), np.uint8)
        self.model = Model(pages, size, rows, width, joined)

    def check(self):
        m, p = self.model, self.pool
        assert p.refs.tolist() == m.refs
        assert p.lengths.tolist() == m.lengths
        assert p.table.tolist() == m.table
        if self.tensors:
            got = np.concatenate([t.cpu().numpy() for t in self.tensors], 1)
            assert np.array_equal(got, m.planes[0])

    def fork(self, src, dst):
        self.pool.fork(len(src), i32(src), i32(dst))
        self.model.fork(src, dst)
        self.check()

    def resize(self, rows, lengths):
        status = torch.ones(len(rows) + 2, dtype=torch.bool, device="cuda")
        self.pool.resize(len(rows), i32(rows), i32(lengths), status)
        want = self.model.resize(rows, lengths)
        self.check()
        assert status.tolist() == want + [True, True]
        return want

    def free(self, rows):
        self.pool.free(len(rows), i32(rows))
        self.model.free(rows)
        self.check()

    def hold(self, pages, delta):
        self.pool.hold(len(pages), i32(pages), delta)
        self.model.count(pages, delta)
        self.check()

    def copy(self, src, dst):
        self.pool.copy(len(src), i32(src), i32(dst))
        self.model.copy(src, dst)
        self.check()

    def compact(self, beside=False):
        page_map = i32([-9] * self.pool.num_pages)
        if beside:
            table, refs = torch.full_like(self.pool.table, -5), torch.full_like(self.pool.refs, -5)
            before = self.pool.table.clone(), self.pool.refs.clone()
            self.pool.compact(page_map, table, refs)
            assert torch.equal(self.pool.table, before[0]) and torch.equal(self.pool.refs, before[1])
            want = self.model.compact()
            assert refs.tolist() == self.model.refs
            for r in range(len(self.model.lengths)):
                held = self.model.held(r)
                assert table[r].tolist() == held + [-5] * (self.model.width - len(held))
                self.pool.table[r, :len(held)] = table[r, :len(held)]
            self.pool.refs.copy_(refs)
        else:
            self.pool.compact(page_map)
            want = self.model.compact()
        self.check()
        assert page_map.tolist() == want


def test_take_branch_write_and_give_back():
    b = Both(16, 4, 4, 5)
    assert b.resize([0], [6]) == [True]  # pages 0 and 1, the second half full
    assert b.pool.table[0].tolist() == [0, 1, -1, -1, -1]
    b.fork([0, 0], [1, 2])
    assert b.pool.refs.tolist()[:3] == [3, 3, 0]
    b.resize([1, 2, 0], [7, 9, 8])  # each gets its own copy of page 1
    assert b.pool.table[1].tolist()[:2] == [0, 2] and b.pool.table[2].tolist()[:3] == [0, 3, 4]
    assert b.pool.refs[1] == 0
    b.resize([1], [4])  # back to the shared page
    b.resize([1], [5])  # a full last page is shared without a copy
    b.free([0, 0, 1])  # listed twice: given back once
    b.resize([2], [0])
    assert not any(b.pool.refs.tolist())


def test_permuted_in_place_and_listed_twice():
    b = Both(40, 4, 5, 6)
    b.resize([0, 1, 2, 3], [5, 9, 0, 22])
    b.fork([1, 0, 3], [0, 1, 3])  # swapped, and one onto itself
    b.fork([0, 1, 2], [4, 4, 4])  # the last one counts: an empty row
    b.fork([3, 0], [4, 4])
    b.fork([-1, 0, 7, 2], [0, 9, 2, -3])  # nothing of it exists
    b.fork([4, 0, 1, 2, 3], [0, 1, 2, 3, 4])  # a rotation
    b.free([0, 1, 2, 3, 4])
    assert not any(b.pool.refs.tolist())


def test_resize_refuses_entries():
    b = Both(8, 4, 4, 4)
    assert b.resize([0, 1, 2], [16, 12, 8]) == [True, True, False]  # 4 + 3, then 2 of 1
    assert b.resize([2, 3], [8, 4]) == [False, False]  # in order: the first wants too much
    assert b.resize([3, 2], [4, 8]) == [True, False]
    assert b.resize([0, 0, 1], [1, 4, 3]) == [False, True, True]  # shrinking, twice listed
    assert b.resize([0, 9, -1], [17, 4, 4]) == [False, False, False]
    assert b.resize([0, 1], [-1, 16]) == [False, True]
    assert b.resize([0, 1, 2, 3], [4, 16, 0, 4]) == [True] * 4  # nothing to do
    # what is given back in a call is not there to be taken in it
    assert b.resize([1, 2], [4, 16]) == [True, False]
    assert b.resize([2], [16]) == [True]


@pytest.mark.parametrize("plane_bytes", [(), (16,), (20, 8), (7,), (16384 * 2 + 16, 48), (1040,) * 9])
def test_copy_pages(plane_bytes):
    b = Both(30, 4, 1, 4, plane_bytes)
    order = np.random.default_rng(3).permutation(30).tolist()
    b.copy(order[:12], order[12:24])
    b.copy([3, -1, 30, 5, 4], [3, 7, 8, 1 << 30, -1])  # onto itself, and nothing that exists
    b.copy([9] * 5, [10, 11, 12, 13, 14])  # one page to many
    b.copy([], [])


def test_hold_keeps_pages():
    b = Both(12, 4, 3, 4)
    b.resize([0], [10])
    b.hold([0, 1, 1, -1, 99], 1)
    b.free([0])
    assert b.pool.refs.tolist()[:3] == [1, 2, 0]
    b.resize([1], [16])  # takes pages 2 to 5
    b.compact()
    b.hold([1], -2)
    b.compact(beside=True)


def test_compact_edges():
    b = Both(9, 4, 2, 9)
    b.compact()  # nothing in use
    b.resize([0], [36])
    b.compact()  # everything in use
    b.fork([0], [1])
    b.resize([0, 1], [0, 4])
    b.compact(beside=True)
    b.hold([8], 1)  # one page at the end, held by nothing else
    b.compact()
    assert b.pool.refs.tolist() == [1, 1] + [0] * 7


def test_table_entries_out_of_range_are_passed_over():
    b = Both(8, 4, 3, 4)
    b.resize([0, 1], [12, 8])
    b.pool.table[0, 1] = b.model.table[0][1] = -7
    b.pool.table[0, 2] = b.model.table[0][2] = 1 << 30
    b.model.refs[1] = b.model.refs[2] = 0
    b.pool.refs[1:3] = 0
    b.fork([0], [2])
    b.free([2])
    b.compact()
    assert b.pool.table[0].tolist()[:3] == [0, -1, -1]
    b.free([0])


@pytest.mark.parametrize("seed,pages,size,rows,width,plane_bytes", [
    (1, 40, 4, 7, 9, (32, 5)), (2, 4100, 16, 60, 40, (16,)), (3, 9000, 8, 300, 64, (16, 16)),
    (4, 5, 1, 3, 5, (48,)), (5, 130, 64, 33, 4, ()), (6, 3000, 3, 9, 1500, (20,)), (7, 3000, 3, 40, 1500, (20,))])
def test_any_order_of_calls(seed, pages, size, rows, width, plane_bytes):
    rng = np.random.default_rng(seed)
    b = Both(pages, size, rows, width, plane_bytes, seed)

    def some_rows(out_of_range=True):
        n = int(rng.integers(0, rows + 1))
        low, high = (-1, rows + 1) if out_of_range and rng.random() < 0.3 else (0, rows)
        return rng.integers(low, high, n).tolist()

    for _ in range(30):
        what = rng.integers(0, 10)
        if what < 3:
            dst = some_rows()
            b.fork(rng.integers(0, rows, len(dst)).tolist(), dst)
        elif what < 7:
            # mostly small steps, so that shared last pages occur
            who = some_rows()
            now = [b.model.lengths[r] if 0 <= r < rows else 0 for r in who]
            top = width * size
            to = [int(min(top + 1, max(-1, n + rng.integers(-size, 2 * size)))) if rng.random() < 0.7
                  else int(rng.integers(0, top + 1) * min(1.0, pages / rows / width)) for n in now]
            b.resize(who, to)
        elif what < 8:
            b.free(some_rows())
        else:
            b.compact(beside=bool(rng.integers(0, 2)))
    assert all(c >= 0 for c in b.pool.refs.tolist())


@pytest.mark.parametrize("rows", [4000, 6000, 60000])
def test_many_rows(rows):
    """Lists and pools of the size where the calls take their scratch elsewhere."""
    rng = np.random.default_rng(rows)
    b = Both(40000, 4, rows, 3, (16,), rows)
    some = rng.permutation(rows)[:rows // 2].tolist()
    b.resize(some, rng.integers(0, 9, len(some)).tolist())
    every = rng.integers(-1, rows + 1, rows).tolist()
    b.fork(every, rng.permutation(rows).tolist())
    b.resize(every, rng.integers(-1, 14, rows).tolist())
    b.fork(rng.permutation(rows).tolist(), every)
    b.free(some)
    b.compact()
    b.fork([1, 2], [2, 1])


def test_time_of_a_fork_grows_with_its_list():
    """No faster than the list: 32 times the entries take 64 times as long at most,
    where comparing every entry with every other would take a thousand times."""
    rows = 1 << 18
    pool = H.PagePool([], 4, rows, 1, num_pages=8)
    order = torch.randperm(rows, device="cuda").to(torch.int32)

    def milliseconds(n):
        times = []
        for _ in range(7):
            begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            begin.record()
            pool.fork(n, order, order)
            end.record()
            torch.cuda.synchronize()
            times.append(begin.elapsed_time(end))
        return sorted(times)[3]

    milliseconds(rows)
    assert milliseconds(rows) <= 64 * milliseconds(rows >> 5)


def test_long_lists_of_long_rows():
    """Thousands of entries, rows of more than one block's columns, destinations named
    several times and numbers that no row has; forked again and again."""
    rng = np.random.default_rng(11)
    rows, width = 2500, 1100
    b = Both(30000, 4, rows, width, ())
    some = rng.permutation(rows)[:40].tolist()
    b.resize(some, rng.integers(0, 4 * width + 1, 20).tolist() + rng.integers(0, 9, 20).tolist())
    for low, high in ((0, rows), (-2, rows + 2), (0, 30)):
        dst = rng.integers(low, high, rows).tolist()
        dst[-1] = dst[0]
        b.fork(rng.integers(-1, rows + 1, rows).tolist(), dst)
        b.fork(rng.permutation(rows).tolist(), rng.permutation(rows).tolist())


def test_long_list_captured_and_replayed():
    rng = np.random.default_rng(12)
    rows = 2600
    b = Both(9000, 4, rows, 3, (), 12)
    b.resize(list(range(rows)), rng.integers(0, 13, rows).tolist())
    src, dst = i32(rng.permutation(rows).tolist()), i32([0] * rows)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b.pool.fork(rows, src, dst)
    for low, high in ((0, rows), (0, 9), (-3, rows)):
        dst.copy_(i32(rng.integers(low, high, rows).tolist()))
        graph.replay()
        b.model.fork(src.tolist(), dst.tolist())
        b.check()


def test_pages_of_several_chunks_and_many_entries():
    """Page copies that a few blocks of an entry take in steps."""
    b = Both(2700, 4, 1300, 2, (33000, 16), 4)
    first = list(range(0, 1300, 2))
    b.resize(first, [6] * 650)
    b.fork(first, [r + 1 for r in first])
    b.resize([r + 1 for r in first], [7] * 650)
    b.compact()


def test_two_pools_on_two_streams():
    """Pools share nothing: their calls may overlap."""
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    pools = [Both(5000, 4, 200, 12, (4096,), k) for k in range(2)]
    lists = [i32(list(range(200))), i32([30] * 200), i32(list(range(100, 200)) + list(range(100)))]
    torch.cuda.synchronize()
    for _ in range(3):
        for b, s in zip(pools, streams):
            b.pool.resize(200, lists[0], lists[1], stream=s)
            b.pool.fork(200, lists[0], lists[2], stream=s)
            b.pool.compact(stream=s)
            b.pool.free(100, lists[2], stream=s)
    torch.cuda.synchronize()
    for b in pools:
        for _ in range(3):
            b.model.resize(lists[0].tolist(), lists[1].tolist())
            b.model.fork(lists[0].tolist(), lists[2].tolist())
            b.model.compact()
            b.model.free(lists[2].tolist()[:100])
        b.check()


def test_wide_table_rows_and_given_state():
    """A table inside a wider tensor; what lies beside it stays."""
    wide = torch.full((3, 12), -8, dtype=torch.int32, device="cuda")
    refs, lengths = torch.zeros(20, dtype=torch.int32, device="cuda"), i32([0, 0, 0])
    plane = torch.zeros((20, 32), dtype=torch.int16, device="cuda")
    pool = H.PagePool([plane], 4, refs=refs, table=wide[:, 2:8], lengths=lengths)
    pool.resize(2, i32([0, 2]), i32([9, 24]))
    pool.fork(1, i32([2]), i32([1]))
    assert wide[1].tolist() == [-8] * 2 + [3, 4, 5, 6, 7, 8] + [-8] * 4
    pool.free(1, i32([0]))
    pool.compact()
    # pages 3 to 8 in use: 0, 1, 2 are filled by 6, 7, 8
    assert wide[2].tolist() == [-8] * 2 + [3, 4, 5, 0, 1, 2] + [-8] * 4
    assert refs.tolist() == [2] * 6 + [0] * 14 and lengths.tolist() == [0, 24, 24]
    with pytest.raises(H.HkvException):
        pool.compact(None, torch.zeros((3, 6), dtype=torch.int32, device="cuda"))
    with pytest.raises(H.HkvException):
        pool.fork(4, i32([0] * 4), i32([1] * 4))  # more entries than rows
    with pytest.raises(H.HkvException):
        pool.resize(2, i32([0]), i32([1, 2]))
    with pytest.raises(H.HkvException):
        pool.free(1, i32([0]).long())
    with pytest.raises(H.HkvException):
        pool.free(1, i32([0]).cpu())


def test_pages_behind_32_bits():
    pages, size = (1 << 16) + 9, 1 << 16
    plane = torch.zeros((pages, size), dtype=torch.uint8, device="cuda")
    plane[-1], plane[3] = 5, 6
    pool = H.PagePool([plane], 4, 1, 4)
    pool.copy(2, i32([pages - 1, 3]), i32([0, pages - 2]))
    assert (plane[0] == 5).all() and (plane[pages - 2] == 6).all() and not plane[pages - 3].any()
    pool.hold(2, i32([pages - 1, pages - 2]))
    pool.compact()
    assert (plane[0] == 6).all() and (plane[1] == 5).all()  # in rising order
    assert pool.refs.tolist()[:3] == [1, 1, 0]


def test_captured_and_replayed():
    """A decode step with branches in a graph, replayed twice against the model."""
    b = Both(64, 4, 6, 8)
    b.resize([0, 1], [7, 11])
    src, dst = i32([0, 0, 1, 1]), i32([2, 3, 4, 5])
    longer, status = i32([8, 8, 12, 13]), torch.zeros(4, dtype=torch.bool, device="cuda")
    ended = i32([3, 4])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b.pool.fork(4, src, dst)
        b.pool.resize(4, dst, longer, status)
        b.pool.free(2, ended)
        b.pool.compact()
    b.check()  # nothing ran yet
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        b.model.fork(src.tolist(), dst.tolist())
        assert status.tolist() == b.model.resize(dst.tolist(), longer.tolist())
        b.model.free(ended.tolist())
        b.model.compact()
        b.check()


def test_on_another_stream():
    b = Both(32, 4, 4, 8)
    s = torch.cuda.Stream()
    rows, lengths = i32([0, 1]), i32([13, 6])
    s.wait_stream(torch.cuda.current_stream())
    b.pool.resize(2, rows, lengths, stream=s)
    b.pool.fork(1, rows, i32([3]), stream=s.cuda_stream)
    torch.cuda.synchronize()
    b.model.resize([0, 1], [13, 6])
    b.model.fork([0], [3])
    b.check()


def test_scratch_from_a_given_allocator():
    made = H.TorchAllocator()
    b = Both(32, 4, 4, 8, allocator=made)
    assert len(made.blocks) == 1
    b.resize([0, 1], [13, 6])
    b.compact()
    b.pool.close()
    assert not made.blocks


def test_scratch_that_pending_work_still_writes():
    """A pool made on a side stream gets memory that a kernel before it, not yet run,
    writes: in the order of that stream this comes first."""
    def state():
        return dict(refs=i32([0] * 40), table=i32([[-1] * 8] * 3000), lengths=i32([0] * 3000))

    first = H.TorchAllocator()
    like = H.PagePool([], 4, allocator=first, **state())
    (size,) = [block.numel() for block in first.blocks.values()]
    like.close()
    given, side, made = state(), torch.cuda.Stream(), H.TorchAllocator()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        pending = torch.empty(size, dtype=torch.uint8, device="cuda")
        address = pending.data_ptr()
        torch.cuda._sleep(100_000_000)
        pending.fill_(3)
        del pending
        pool = H.PagePool([], 4, allocator=made, **given)
    assert list(made.blocks) == [address]
    for n in (3, 3000):  # both forms of a fork
        given["lengths"][:2] = i32([9, 32])
        pool.fork(n, i32([0, 1] + [1] * (n - 2)), i32([1, 0] + list(range(2, n))))
        assert pool.lengths[:n].tolist() == [32, 9] + [32] * (n - 2)


def test_failing_allocator():
    class Nothing:
        def alloc(self, memory_type, size, flags):
            raise MemoryError

        def free(self, memory_type, address):
            pass

    with pytest.raises(H.CudaException):
        H.PagePool([], 4, 2, 4, num_pages=8, allocator=Nothing())
    assert ctypes.sizeof(H._PagesOptions) == 72


def test_prefix_index_of_a_cache():
    """The table as the index of a paged cache: blocks of prompts found again by
    their hash, their pages shared, pages of evicted blocks let go."""
    size, rows, pages = 4, 8, 128
    plane = torch.arange(pages, device="cuda", dtype=torch.int32)[:, None].repeat(1, 8)
    pool = H.PagePool([plane], size, rows, 16)
    index = H.HashTable(H.EvictStrategy.kLru, value_dtype="uint32")
    index.init(H.HashTableOptions(init_capacity=128, max_capacity=128,
                                  max_hbm_for_vectors=1 << 20, dim=1))
    hashes = torch.arange(1, 13, device="cuda", dtype=torch.int64) * 7919  # 12 blocks
    pool.resize(1, i32([0]), i32([12 * size]))
    first = pool.table[0, :12].contiguous()
    index.insert_or_assign(12, hashes, first)
    pool.hold(12, first)  # the index's own references
    pool.free(1, i32([0]))
    assert pool.refs.sum() == 12
    # another request with the same first eight blocks
    found, got = torch.zeros(10, dtype=torch.bool, device="cuda"), i32([-1] * 10)
    asked = torch.cat([hashes[:8], hashes[:2] + 1])
    index.find(10, asked, got, found)
    assert found.tolist() == [True] * 8 + [False] * 2
    pool.table[3, :8] = got[:8]
    pool.lengths[3] = 8 * size
    pool.hold(8, got)
    pool.resize(1, i32([3]), i32([9 * size + 1]))  # its own blocks behind them
    # the index loses blocks: evicted values are pages to let go
    more = torch.arange(1000, 1128, device="cuda", dtype=torch.int64) * 104729
    held = i32([-1] * 128)  # blocks whose pages live elsewhere
    gone = torch.zeros(128, dtype=torch.int64, device="cuda")
    lost = i32([-1] * 128)
    n = index.insert_and_evict(128, more, held, None, gone, lost)
    pool.hold(n, lost, -1)
    kept = sorted(set(range(12)) - set(lost.tolist()))
    want = [0] * pages
    for p in kept:
        want[p] += 1
    for p in pool.table[3, :10].tolist():
        want[p] += 1
    assert pool.refs.tolist() == want
    # compaction, and the index told of the new numbers
    marks = plane[pool.table[3, :10].long(), 0].tolist()
    page_map = i32([0] * pages)
    pool.compact(page_map)
    assert plane[pool.table[3, :10].long(), 0].tolist() == marks
    live = sum(c > 0 for c in want)
    assert (pool.refs[:live] > 0).all() and not pool.refs[live:].any()
    keys, values = torch.zeros(128, dtype=torch.int64, device="cuda"), i32([0] * 128)
    scores = torch.zeros(128, dtype=torch.int64, device="cuda")
    m = index.export_batch(128, 0, keys, values, scores)
    here = values[:m] >= 0
    moved = torch.where(here, page_map[values[:m].clamp(min=0).long()], values[:m])
    index.insert_or_assign(m, keys, moved, None)
    index.find(12, hashes, got_all := i32([-1] * 12), f := torch.zeros(12, dtype=torch.bool, device="cuda"))
    for k in range(12):
        if f[k]:
            assert plane[got_all[k], 0] == first[k]
    index.close()


def test_prefix_index_that_loses_half_of_its_blocks():
    """Six of twelve blocks evicted: their pages are let go, the others are found and
    hold what they held, before and after a compaction."""
    size, pages = 4, 64
    plane = torch.arange(pages, device="cuda", dtype=torch.int32)[:, None].repeat(1, 8)
    pool = H.PagePool([plane], size, 2, 16)
    index = H.HashTable(H.EvictStrategy.kLru, value_dtype="uint32")
    index.init(H.HashTableOptions(init_capacity=128, max_capacity=128,
                                  max_hbm_for_vectors=1 << 20, dim=1))
    hashes = torch.arange(1, 13, device="cuda", dtype=torch.int64) * 7919
    pool.resize(2, i32([0, 1]), i32([5 * size, 12 * size]))
    pool.free(1, i32([0]))
    first = pool.table[1, :12].contiguous()
    assert first.tolist() == list(range(5, 17))
    index.insert_or_assign(12, hashes, first)
    pool.hold(12, first)
    pool.free(1, i32([1]))
    n = 128 - 12 + 6
    more = torch.arange(1000, 1000 + n, device="cuda", dtype=torch.int64) * 104729
    gone, lost = torch.zeros(n, dtype=torch.int64, device="cuda"), i32([-1] * n)
    count = index.insert_and_evict(n, more, i32([-1] * n), None, gone, lost)
    assert count == 6 and all(5 <= p < 17 for p in lost[:6].tolist())
    pool.hold(count, lost, -1)
    found, got = torch.zeros(12, dtype=torch.bool, device="cuda"), i32([-1] * 12)
    index.find(12, hashes, got, found)
    kept = [k for k in range(12) if found[k]]
    assert len(kept) == 6
    assert [got[k].item() for k in kept] == [first[k].item() for k in kept]
    assert sorted(first[k].item() for k in kept) == pool.refs.nonzero()[:, 0].tolist()
    page_map = i32([0] * pages)
    pool.compact(page_map)
    assert pool.refs.tolist() == [1] * 6 + [0] * (pages - 6)
    assert [plane[page_map[first[k]], 0].item() for k in kept] == [first[k].item() for k in kept]
    index.close()
