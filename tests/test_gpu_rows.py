"""Tokens sorted by group and back with weights, and both gradients, against
their definitions in 64 bits.

Tolerances: u = 2^-24 bounds a float32 rounding, h = eps / 2 the rounding to the
result's type (both relative), `tiny` half of the smallest float16 step, where
the relative bound ends.
* combine_rows: slots fused multiply-adds in float32, each rounding a partial
  sum of magnitude at most M = sum |w y|, then one rounding:
  slots u M + h (|out| + slots u M).
* grad_rows: a product rounded to float32, then to the type: (u + h (1 + u)) |w g|.
* grad_weights: dim products and additions in any order, dim u sum |g y|, then
  one rounding.
"""
import threading

import numpy as np
import pytest
import torch

import hkv_b200 as H

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TINY = 2.0 ** -25
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def seeded(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def randn(g, *shape, dtype=F32):
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def i32(*shape, fill=0):
    return torch.full(shape, fill, dtype=torch.int32, device="cuda")


# ---- group_tokens ------------------------------------------------------------


def sorted_reference(ids, groups):
    """offsets, positions, order by the definition."""
    ids = ids.cpu().numpy().astype(np.int64).reshape(-1)
    kept = np.flatnonzero((ids >= 0) & (ids < groups))
    order = kept[np.argsort(ids[kept], kind="stable")]
    positions = np.full(ids.size, -1, np.int64)
    positions[order] = np.arange(order.size)
    offsets = np.concatenate([[0], np.cumsum(np.bincount(ids[kept], minlength=groups))])
    return offsets, positions, np.concatenate([order, np.full(ids.size - order.size, -1)])


def check_sort(ids, groups, **kw):
    n = ids.numel()
    offsets, positions, order = i32(groups + 1, fill=-7), i32(n + 3, fill=-7), i32(n + 3, fill=-7)
    H.group_tokens(n, ids, groups, offsets, positions, order, **kw)
    want = sorted_reference(ids, groups)
    assert np.array_equal(offsets.cpu().numpy(), want[0])
    assert np.array_equal(positions.cpu().numpy()[:n], want[1])
    assert np.array_equal(order.cpu().numpy()[:n], want[2])
    assert (positions[n:] == -7).all() and (order[n:] == -7).all()


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("groups", [1, 2, 31, 64, 257, 1024, 1025, 4096])
@pytest.mark.parametrize("n", [0, 1, 31, 33, 500, 1023, 4096, 4097, 8192, 8193, 50001])
def test_group_tokens(n, groups, dtype):
    ids = torch.randint(0, groups, (n,), generator=seeded(n + groups), device="cuda")
    check_sort(ids.to(dtype), groups)


@pytest.mark.parametrize("n,groups", [(300007, 8), (1300003, 100), (2500000, 4096), (70000, 1)])
def test_group_tokens_long(n, groups):
    g = seeded(n)
    skew = torch.rand(n, generator=g, device="cuda") ** 4
    ids = (skew * groups).long().clamp(max=groups - 1)
    ids[torch.rand(n, generator=g, device="cuda") < 0.1] = -1
    check_sort(ids, groups)
    check_sort(ids.to(torch.int32), groups)


@pytest.mark.parametrize("n", [1, 77, 5000, 40000])
def test_group_tokens_drops_what_is_outside(n):
    g = seeded(n)
    ids = torch.randint(-3, 13, (n,), generator=g, device="cuda")
    ids[::3] = (1 << 32) + 2  # looks like group 2 in its low 32 bits
    ids[1::7] = -(1 << 63)
    check_sort(ids, 9)
    check_sort(torch.full((n,), -1, device="cuda"), 9)  # nothing is kept
    check_sort(torch.full((n,), 8, device="cuda"), 9)  # one group has all
    check_sort(torch.full((n,), 0, dtype=torch.int32, device="cuda"), 9)


def test_group_tokens_without_order_and_with_workspace():
    n, groups = 9001, 40
    ids = torch.randint(0, groups, (n,), device="cuda")
    work = torch.full((H.group_workspace(n, groups) + 16,), 0xAB, dtype=torch.uint8, device="cuda")
    offsets, positions = i32(groups + 1), i32(n)
    H.group_tokens(n, ids, groups, offsets, positions, workspace=work)
    want = sorted_reference(ids, groups)
    assert np.array_equal(positions.cpu().numpy(), want[1])
    assert np.array_equal(offsets.cpu().numpy(), want[0])
    assert (work[-16:] == 0xAB).all()


def test_group_tokens_on_other_streams():
    ids = torch.randint(0, 50, (6000,), device="cuda")
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    offsets, positions, order = i32(51), i32(6000), i32(6000)
    torch.cuda.synchronize()
    H.group_tokens(6000, ids, 50, offsets, positions, order, stream=s)
    s.synchronize()
    want = sorted_reference(ids, 50)
    assert np.array_equal(order.cpu().numpy(), want[2])
    order.zero_()
    torch.cuda.synchronize()
    H.group_tokens(6000, ids, 50, offsets, positions, order, stream=s.cuda_stream)
    torch.cuda.synchronize()
    assert np.array_equal(order.cpu().numpy(), want[2])


def test_group_tokens_on_two_streams_at_once():
    n, groups = 300000, 100
    ids = [torch.randint(0, groups, (n,), generator=seeded(k), device="cuda") for k in range(2)]
    out = [(i32(groups + 1), i32(n), i32(n)) for _ in ids]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(5):
        for k, s in enumerate(streams):  # each call its own scratch, from its stream's pool
            H.group_tokens(n, ids[k], groups, *out[k], stream=s)
    torch.cuda.synchronize()
    for k in range(2):
        want = sorted_reference(ids[k], groups)
        assert np.array_equal(out[k][1].cpu().numpy(), want[1])
        assert np.array_equal(out[k][2].cpu().numpy(), want[2])


@pytest.mark.parametrize("groups", [64, 3000])
def test_scratch_of_the_largest_batch(groups):
    """Scratch sized once serves every smaller call."""
    largest = 200000
    scratch = torch.zeros(H.group_workspace(largest, groups), dtype=torch.uint8, device="cuda")
    for n in (0, 1, 1000, 1024, 1025, 32768, 32769, 150000, 151552, 151553, largest):
        ids = torch.randint(-1, groups, (n,), generator=seeded(n), device="cuda")
        check_sort(ids, groups, workspace=scratch)


@pytest.mark.parametrize("n,first,second", [(30000, 300, 400), (40000, 1500, 4000)])
def test_group_tokens_from_host_threads(n, first, second):
    """Host threads, each with a stream and a workspace, launch the same kernels with
    more than 48 KB of shared memory, of two sizes. The library's calls are made
    one right after the other, so that they meet."""
    calls, work = 3000, []
    for groups in (first, second) * 2:
        ids = torch.randint(0, groups, (n,), generator=seeded(groups), device="cuda")
        scratch = torch.zeros(H.group_workspace(n, groups), dtype=torch.uint8, device="cuda")
        work.append((ids, groups, (i32(groups + 1), i32(n), i32(n)), scratch, torch.cuda.Stream()))
    torch.cuda.synchronize()
    ready, statuses = threading.Barrier(len(work), timeout=60), []

    def sort(ids, groups, out, scratch, stream):
        call = H.lib().hkv_group_tokens
        args = (n, ids.data_ptr(), 1, groups, *(t.data_ptr() for t in out), scratch.data_ptr(),
                scratch.numel(), stream.cuda_stream)
        ready.wait()
        statuses.extend([call(*args) for _ in range(calls)])

    threads = [threading.Thread(target=sort, args=w) for w in work]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert len(statuses) == calls * len(work) and not any(statuses)
    for ids, groups, out, _, _ in work:
        want = sorted_reference(ids, groups)
        assert all(np.array_equal(g.cpu().numpy(), w) for g, w in zip(out, want))


# ---- dispatch_rows -----------------------------------------------------------


def places(g, n, slots, rows, dropped):
    """Distinct rows for n * slots places, some without one."""
    at = torch.randperm(rows, generator=g, device="cuda")[:n * slots].to(torch.int32)
    at = torch.cat([at, i32(n * slots - at.numel(), fill=-1)])
    at = at[torch.randperm(n * slots, generator=g, device="cuda")]
    at[torch.rand(n * slots, generator=g, device="cuda") < dropped] = -1
    return at.view(n, slots)


@pytest.mark.parametrize("dtype", [F32, F16, BF16, torch.float64, torch.int64, torch.int8])
@pytest.mark.parametrize("n,slots,dim,dropped", [(1, 1, 1, 0), (1, 8, 64, 0), (37, 3, 129, 0.3),
                                                 (5, 2, 4096, 0.5), (300, 5, 40, 0),
                                                 (2000, 1, 1, 0.1), (9, 4, 7, 1.0)])
def test_dispatch_rows(n, slots, dim, dropped, dtype):
    g = seeded(n * slots + dim)
    rows = n * slots + 2
    at = places(g, n, slots, rows, dropped)
    at[-1, -1] = rows + 5  # outside: passed over
    x = torch.randint(-100, 100, (n, dim), generator=g, device="cuda").to(dtype)
    out = torch.full((rows, dim), 77, dtype=dtype, device="cuda")
    want = out.clone()
    H.dispatch_rows(n, x, at, out)
    for t, s in (((at >= 0) & (at < rows)).nonzero()).tolist()[:20000]:
        want[at[t, s]] = x[t]
    assert torch.equal(out, want)


@pytest.mark.parametrize("dtype,dim,stride,first", [(F32, 12, 20, 0), (BF16, 8, 11, 0),
                                                    (BF16, 16, 24, 4), (F16, 6, 6, 1),
                                                    (torch.int8, 16, 20, 4)])
def test_rows_with_strides_and_odd_starts(dtype, dim, stride, first):
    """Rows inside wider tensors, at addresses that allow narrower words only."""
    n, slots = 50, 3
    g = seeded(dim)
    at = places(g, n, slots, n * slots, 0.2)
    wide = torch.randint(-50, 50, (n, stride + first), generator=g, device="cuda").to(dtype)
    x = wide[:, first:first + dim]
    room = torch.zeros((n * slots, stride + first), dtype=dtype, device="cuda")
    H.dispatch_rows(n, x, at, room[:, first:first + dim])
    want = torch.zeros_like(room)
    for t, s in (at >= 0).nonzero().tolist():
        want[at[t, s], first:first + dim] = x[t]
    assert torch.equal(room, want)
    if dtype == torch.int8:
        return
    back = torch.zeros((n, stride + first), dtype=dtype, device="cuda")
    H.combine_rows(n, room[:, first:first + dim], at, None, back[:, first:first + dim])
    kept = (at >= 0).sum(1, keepdim=True).to(torch.float64)
    assert torch.equal(back[:, first:first + dim].double(), x.double() * kept)
    assert not back[:, :first].any() and not back[:, first + dim:].any()


# ---- combine_rows and its gradients ---------------------------------------------


def combine_reference(rows, at, weights, grad_out):
    """out, M, grad_rows, |w g|, grad_weights, sum |g y| in 64 bits."""
    n, slots = at.shape
    has = (at >= 0) & (at < rows.shape[0])
    y = rows.double()[at.clamp(0, rows.shape[0] - 1).long()]
    y = torch.where(has[:, :, None], y, 0.0)
    w = torch.ones(at.shape, dtype=torch.float64, device="cuda") if weights is None \
        else weights.double()
    w = torch.where(has, w, 0.0)
    out, mass = (w[:, :, None] * y).sum(1), (w[:, :, None] * y).abs().sum(1)
    g = grad_out.double()
    dots, dot_mass = (g[:, None] * y).sum(2), (g[:, None] * y).abs().sum(2)
    return out, mass, w[:, :, None] * g[:, None], dots, dot_mass, has


def near(got, want, slack):
    """|got - want| <= slack before the rounding to got's type, that rounding added."""
    bound = slack + half_step(got.dtype) * (want.abs() + slack) + TINY
    off = (got.double() - want).abs()
    assert not torch.isnan(off).any()
    assert (off <= bound).all(), float((off - bound).max())


def check_combine(g, n, slots, dim, dtype, weight, dropped, identity=False, extra=0):
    count = n * slots + extra
    rows = randn(g, count, dim, dtype=dtype)
    at = places(g, n, slots, count, dropped)
    if identity:
        at = torch.arange(n * slots, device="cuda", dtype=torch.int32).view(n, slots)
    weights = None if weight is None else randn(g, n, slots, dtype=weight)
    grad_out = randn(g, n, dim, dtype=dtype)
    out = torch.full((n + 1, dim), 9.0, dtype=dtype, device="cuda")
    grad_rows = torch.full((count, dim), 9.0, dtype=dtype, device="cuda")
    grad_weights = torch.full((n, slots), 9.0, dtype=weight or F32, device="cuda")
    given, more = (None, {"slots": slots}) if identity else (at, {})
    H.combine_rows(n, rows, given, weights, out, **more)
    H.combine_rows_backward(n, rows, given, weights, grad_out, grad_rows, grad_weights, **more)
    want, mass, spread, dots, dot_mass, has = combine_reference(rows, at, weights, grad_out)
    near(out[:n], want, slots * U * mass)
    assert (out[n:] == 9).all()
    near(grad_weights, dots, dim * U * dot_mass)
    at_rows = at[has].long()
    near(grad_rows[at_rows], spread[has], U * spread[has].abs())
    rest = torch.ones(count, dtype=torch.bool, device="cuda")
    rest[at_rows] = False
    assert (grad_rows[rest] == 9).all()
    # either gradient alone gives the same bits
    alone_rows, alone_weights = torch.full_like(grad_rows, 9.0), torch.zeros_like(grad_weights)
    H.combine_rows_backward(n, None, given, weights, grad_out, alone_rows, None, **more)
    H.combine_rows_backward(n, rows, given, weights, grad_out, None, alone_weights, **more)
    assert torch.equal(alone_rows, grad_rows) and torch.equal(alone_weights, grad_weights)


@pytest.mark.parametrize("dtype,weight", [(F32, F32), (F32, None), (F16, F32), (F16, F16),
                                          (BF16, F32), (BF16, BF16), (BF16, None)])
@pytest.mark.parametrize("n,slots,dim,dropped", [(1, 1, 1, 0), (1, 1, 8192, 0), (1, 7, 64, 0.4),
                                                 (33, 3, 129, 0.3), (700, 20, 64, 0.4),
                                                 (64, 4, 1024, 0), (5, 33, 40, 0.2),
                                                 (3, 2, 5000, 0.5), (11, 2, 24, 1.0),
                                                 (260, 8, 520, 0.1)])
def test_combine_and_gradients(n, slots, dim, dropped, dtype, weight):
    check_combine(seeded(n + slots + dim), n, slots, dim, dtype, weight, dropped, extra=3)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,slots,dim", [(1, 1, 32), (50, 19, 64), (7, 1, 130)])
def test_combine_by_place(n, slots, dim, dtype):
    check_combine(seeded(slots), n, slots, dim, dtype, F32, 0, identity=True)
    check_combine(seeded(slots), n, slots, dim, dtype, None, 0, identity=True)


def test_positions_outside_of_fewer_rows():
    """By place, rows that are not there add nothing."""
    rows = torch.ones((5, 8), device="cuda")
    out = torch.full((3, 8), 9.0, device="cuda")
    H.combine_rows(3, rows, None, torch.ones((3, 2), device="cuda"), out)
    assert out[:, 0].tolist() == [2, 2, 1]
    none = torch.zeros((0, 8), device="cuda")
    H.combine_rows(3, none, i32(3, 2), None, out)
    assert not out.any()


def test_nothing_of_a_place_without_a_row_is_read():
    """NaN and infinities in weights of places without a row, and in rows that no
    place has, reach nothing."""
    rows = torch.full((8, 16), float("nan"), device="cuda")
    rows[2], rows[5] = 1.0, 2.0
    at = torch.tensor([[2, -1], [-1, 5], [-1, -1], [8, 1 << 30]], dtype=torch.int32, device="cuda")
    bad = float("nan")
    weights = torch.tensor([[1.0, bad], [float("inf"), 0.5], [bad, bad], [bad, bad]], device="cuda")
    out, grad_out = torch.full((4, 16), bad, device="cuda"), torch.ones((4, 16), device="cuda")
    H.combine_rows(4, rows, at, weights, out)
    assert out[:, 0].tolist() == [1, 1, 0, 0] and not torch.isnan(out).any()
    grad_rows, grad_weights = torch.zeros_like(rows), torch.full_like(weights, bad)
    H.combine_rows_backward(4, rows, at, weights, grad_out, grad_rows, grad_weights)
    assert grad_weights.tolist() == [[16, 0], [0, 32], [0, 0], [0, 0]]
    assert grad_rows[:, 0].tolist() == [0, 0, 1, 0, 0, 0.5, 0, 0]


def test_infinities_of_a_used_row_arrive():
    rows = torch.tensor([[float("inf"), 1.0], [2.0, float("nan")]], device="cuda")
    out = torch.zeros((1, 2), device="cuda")
    H.combine_rows(1, rows, i32(1, 2) + torch.tensor([0, 1], device="cuda").int(), None, out)
    assert out[0, 0] == float("inf") and torch.isnan(out[0, 1])


def test_gradient_against_differences():
    """The analytic gradients against central differences of combine_rows in
    float32. The sum is linear in rows and in weights, so a difference of two
    losses over twice the step is off by one loss's rounding at most: (slots +
    1) u M per output, M <= slots * size. The gradient itself is off by dim u
    size per unit of grad_out. Together (slots (slots + 1) + dim) u size sum
    |grad_out|, below the bound taken."""
    g = seeded(4)
    n, slots, dim, step = 6, 3, 5, 1.0
    rows, at = randn(g, n * slots, dim), places(g, n, slots, n * slots, 0.2)
    weights, grad_out = randn(g, n, slots), randn(g, n, dim)
    grad_rows, grad_weights = torch.zeros_like(rows), torch.zeros_like(weights)
    H.combine_rows_backward(n, rows, at, weights, grad_out, grad_rows, grad_weights)

    def loss(r, w):
        out = torch.zeros_like(grad_out)
        H.combine_rows(n, r, at, w, out)
        return float((out.double() * grad_out.double()).sum())

    size = (weights.abs().max() + step) * (rows.abs().max() + step)
    bound = float((2 * slots + 1) * U * slots * size * grad_out.abs().sum()) / step
    for i in range(n * slots):
        t, s = divmod(i, slots)
        a, b = weights.clone(), weights.clone()
        a[t, s] += step
        b[t, s] -= step
        moved = float(a[t, s].double() - b[t, s].double())
        assert abs((loss(rows, a) - loss(rows, b)) / moved - float(grad_weights[t, s])) <= bound
        a, b = rows.clone(), rows.clone()
        a[i, i % dim] += step
        b[i, i % dim] -= step
        moved = float(a[i, i % dim].double() - b[i, i % dim].double())
        assert abs((loss(a, weights) - loss(b, weights)) / moved - float(grad_rows[i, i % dim])) <= bound


def test_offsets_over_32_bits():
    """Rows whose elements lie behind the first 2^32."""
    dim, rows = 1 << 16, (1 << 16) + 3
    big = torch.zeros((rows, dim), dtype=torch.int8, device="cuda")
    x = torch.arange(2 * dim, device="cuda").view(2, dim).to(torch.int8)
    at = torch.tensor([[rows - 1], [rows - 3]], dtype=torch.int32, device="cuda")
    H.dispatch_rows(2, x, at, big)
    assert torch.equal(big[rows - 1], x[0]) and torch.equal(big[rows - 3], x[1])
    assert not big[rows - 2].any() and not big[0].any() and not big[rows - 1 - (1 << 16)].any()
    del big
    rows16 = torch.zeros(((1 << 17) + 2, 1 << 15), dtype=BF16, device="cuda")
    rows16[-1] = 3.0
    at = torch.tensor([[0, rows16.shape[0] - 1]], dtype=torch.int32, device="cuda")
    out = torch.zeros((1, 1 << 15), dtype=BF16, device="cuda")
    H.combine_rows(1, rows16, at, None, out)
    assert (out == 3).all()
    grad, dots = torch.ones_like(out), torch.zeros((1, 2), device="cuda")
    H.combine_rows_backward(1, rows16, at, None, grad, None, dots)
    assert dots.tolist() == [[0, 3 << 15]]
    H.combine_rows_backward(1, None, at, None, grad, rows16, None)  # rows16 takes the gradient
    assert (rows16[-1] == 1).all() and (rows16[0] == 1).all() and not rows16[1].any()


def test_more_words_than_32_bits_number():
    """Rows of an odd number of 2-byte elements, 2^31 of them and some more, which
    take more than one launch: all rows there and back, by position and by place."""
    dim = 4097
    n = (1 << 31) // dim + 50
    x = torch.randint(-128, 128, (n, dim), generator=seeded(1), device="cuda", dtype=torch.int8)
    x = x.to(BF16)
    at = torch.arange(n - 1, -1, -1, device="cuda", dtype=torch.int32).view(n, 1)
    at[5] = at[n - 5] = -1
    rows = torch.zeros((n, dim), dtype=BF16, device="cuda")
    H.dispatch_rows(n, x, at, rows)
    x[5], x[n - 5] = 0, 0
    assert torch.equal(rows.flip(0), x)
    out = torch.full((n, dim), 7.0, dtype=BF16, device="cuda")
    H.combine_rows(n, rows, at, None, out)
    assert torch.equal(out, x)
    del rows, at
    two = torch.stack([x, x], 1).view(2 * n, dim)
    two = two[:2 * n - 1]  # the last place has no row
    out.fill_(7.0)
    H.combine_rows(n, two, None, None, out, slots=2)
    x[:n - 1] *= 2
    assert torch.equal(out, x)


def test_captured_and_replayed():
    """The whole way there and back in a graph, replayed on other inputs."""
    n, slots, groups, dim = 96, 4, 16, 64
    ids, x = torch.zeros((n, slots), dtype=torch.int64, device="cuda"), torch.zeros((n, dim), device="cuda")
    weights = torch.zeros((n, slots), device="cuda")
    offsets, at, order = i32(groups + 1), i32(n, slots), i32(n * slots)
    rows, out = torch.zeros((n * slots, dim), device="cuda"), torch.zeros((n, dim), device="cuda")
    grads = torch.zeros_like(rows), torch.zeros_like(weights)

    def step():
        H.group_tokens(n * slots, ids, groups, offsets, at, order)
        H.dispatch_rows(n, x, at, rows)
        H.combine_rows(n, rows, at, weights, out)
        H.combine_rows_backward(n, rows, at, weights, x, *grads)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for seed in (1, 2):
        g = seeded(seed)
        ids.copy_(torch.randint(0, groups, (n, slots), generator=g, device="cuda"))
        x.copy_(randn(g, n, dim))
        weights.copy_(randn(g, n, slots))
        graph.replay()
        torch.cuda.synchronize()
        want = sorted_reference(ids, groups)
        assert np.array_equal(at.cpu().numpy().reshape(-1), want[1])
        assert torch.equal(rows, x[torch.from_numpy(want[2]).cuda() // slots])
        total = weights.double().sum(1, keepdim=True)
        mass = weights.double().abs().sum(1, keepdim=True) * x.double().abs()
        near(out, x.double() * total, slots * U * mass)
        square = (x.double() ** 2).sum(1, keepdim=True)
        near(grads[1], square.expand(n, slots), dim * U * square.expand(n, slots))


def test_captured_between_branches_copies_and_other_kernels():
    """Nodes before and after the calls that are no kernels of this library, and
    two streams that join: each call sees what came before it."""
    n, groups = 70000, 32
    source = torch.zeros(n, dtype=torch.int32, device="cuda")
    first, second = i32(n), i32(n)
    out = [(i32(groups + 1), i32(n), i32(n)) for _ in range(3)]
    moved, pool_rows = torch.zeros((n, 1), device="cuda"), torch.zeros((n, 1), device="cuda")
    side = torch.cuda.Stream()
    H.group_tokens(n, source, groups, *out[0])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        main = torch.cuda.current_stream()
        side.wait_stream(main)
        with torch.cuda.stream(side):
            second.copy_(source)
            second.add_(1).remainder_(groups)
            H.group_tokens(n, second, groups, *out[1])
        first.copy_(source)  # a copy node, then the call
        H.group_tokens(n, first, groups, *out[0])
        main.wait_stream(side)
        H.group_tokens(n, second, groups, *out[2])  # after the join
        pool_rows.zero_()
        H.dispatch_rows(n, source.view(torch.float32).view(n, 1), out[2][1].view(n, 1), pool_rows)
        moved.copy_(pool_rows)
    for seed in (5, 6):
        source.copy_(torch.randint(0, groups, (n,), generator=seeded(seed), device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        later = (source + 1) % groups
        for ids, got in ((source, out[0]), (later, out[1]), (later, out[2])):
            want = sorted_reference(ids, groups)
            assert all(np.array_equal(g.cpu().numpy(), w) for g, w in zip(got, want))
        order = out[2][2].long()
        assert torch.equal(moved.view(torch.int32).view(-1), source[order])


def test_default_stream_by_its_number():
    ids = torch.randint(0, 50, (6000,), device="cuda")
    out = i32(51), i32(6000), i32(6000)
    H.group_tokens(6000, ids, 50, *out, stream=0)
    torch.cuda.synchronize()
    assert all(np.array_equal(g.cpu().numpy(), w) for g, w in zip(out, sorted_reference(ids, 50)))


def test_same_bits_every_time():
    g = seeded(8)
    n, slots, dim = 500, 6, 200
    rows, at = randn(g, n * slots, dim, dtype=BF16), places(g, n, slots, n * slots, 0.1)
    weights, grad = randn(g, n, slots), randn(g, n, dim, dtype=BF16)
    got = []
    for _ in range(3):
        out, dw = torch.zeros_like(grad), torch.zeros_like(weights)
        H.combine_rows(n, rows, at, weights, out)
        H.combine_rows_backward(n, rows, at, weights, grad, None, dw)
        got.append((out, dw))
    assert all(torch.equal(a, b) for k in (1, 2) for a, b in zip(got[0], got[k]))


def test_keys_to_tables_and_bags_back():
    """A model with a table per feature: keys sorted by table, each table asked for
    its own run, rows back to the tokens with weights, the gradient to the tables."""
    tables, dim, n, slots = 3, 16, 200, 4
    g = seeded(21)
    keys = torch.randperm(5000, generator=g, device="cuda")[:n * slots].view(n, slots) + 1
    which = torch.randint(0, tables, (n, slots), generator=g, device="cuda")
    which[torch.rand((n, slots), generator=g, device="cuda") < 0.2] = -1  # shorter bags
    values = randn(g, 5001, dim)
    made = []
    for t in range(tables):
        table = H.HashTable(H.EvictStrategy.kLru)
        table.init(H.HashTableOptions(init_capacity=8192, max_capacity=8192,
                                      max_hbm_for_vectors=1 << 30, dim=dim))
        mine = keys[which == t].contiguous()
        table.insert_or_assign(mine.numel(), mine, values[mine].contiguous())
        made.append(table)
    offsets, at, sorted_keys = i32(tables + 1), i32(n, slots), torch.zeros((n * slots, 1), dtype=torch.int64, device="cuda")
    H.group_tokens(n * slots, which, tables, offsets, at)
    # a key is a row of one 64-bit element, each place a token of its own
    H.dispatch_rows(n * slots, keys.view(-1, 1), at.view(-1, 1), sorted_keys)
    rows, found = torch.zeros((n * slots, dim), device="cuda"), torch.zeros(n * slots, dtype=torch.bool, device="cuda")
    cut = offsets.tolist()
    for t, table in enumerate(made):
        a, b = cut[t], cut[t + 1]
        table.find(b - a, sorted_keys[a:b], rows[a:b], found[a:b])
    assert found[:cut[-1]].all() and not found[cut[-1]:].any()
    weights = randn(g, n, slots)
    out, grad_out = torch.zeros((n, dim), device="cuda"), randn(g, n, dim)
    H.combine_rows(n, rows, at, weights, out)
    kept = (which >= 0)[:, :, None]
    terms = torch.where(kept, weights.double()[:, :, None] * values.double()[keys], 0.0)
    near(out, terms.sum(1), slots * U * terms.abs().sum(1))
    # one step down the gradient, row by row through accum_or_assign
    grad_rows, grad_weights = torch.zeros_like(rows), torch.zeros_like(weights)
    H.combine_rows_backward(n, rows, at, weights, grad_out, grad_rows, grad_weights)
    for t, table in enumerate(made):
        a, b = cut[t], cut[t + 1]
        here = torch.ones(b - a, dtype=torch.bool, device="cuda")
        table.accum_or_assign(b - a, sorted_keys[a:b], grad_rows[a:b].contiguous(), here)
        after = torch.zeros((b - a, dim), device="cuda")
        table.find(b - a, sorted_keys[a:b], after, found[a:b])
        assert torch.equal(after, rows[a:b] + grad_rows[a:b])
        table.close()
