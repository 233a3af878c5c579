"""What the row operators and the page pool refuse, and the calls that do nothing:
checked on the host before any CUDA call, so on CPU."""
import ctypes

import pytest
import torch

import hkv_b200 as H

SOME = 4096  # an aligned address that is never read: every call below is refused first


def status(name, *args):
    return getattr(H.lib(), name)(*args)


def i32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


@pytest.mark.parametrize("n,groups", [(0, 1), (1, 1), (4096, 64), (4097, 4096),
                                      ((1 << 31) - 1, 8)])
def test_group_workspace(n, groups):
    size = H.group_workspace(n, groups)
    assert 0 < size < 1 << 30


@pytest.mark.parametrize("n,groups", [(1, 0), (1, 4097), (1 << 31, 4), (-1, 4), (1, -1),
                                      (1, 1 << 32)])
def test_group_workspace_refuses(n, groups):
    with pytest.raises(H.HkvException):
        H.group_workspace(n, groups)


@pytest.mark.parametrize("groups", [1, 8, 64, 428, 1168, 3000, 4096])
def test_group_workspace_never_falls(groups):
    """Scratch for n places serves every call with fewer. The borders of the forms
    and of the tiles' sizes lie at multiples of 512."""
    borders = sorted({max(0, k * step + d) for step in (512, 4096, 75776, 303104)
                      for k in range(0, 40) for d in (-1, 0, 1)} | {1 << 24, (1 << 31) - 1})
    sizes = [H.group_workspace(n, groups) for n in borders]
    assert all(a <= b for a, b in zip(sizes, sizes[1:]))
    # nor with more groups
    assert all(H.group_workspace(n, groups) <= H.group_workspace(n, 4096) for n in borders)


@pytest.mark.parametrize("groups", [8 - (1 << 32), 8 + (1 << 32), -1, 0, 4097])
@pytest.mark.parametrize("scratch", [None, 1 << 16])
def test_group_tokens_refuses_numbers_of_groups(groups, scratch):
    """Before offsets, which are num_groups + 1, are looked at."""
    work = None if scratch is None else torch.zeros(scratch, dtype=torch.uint8)
    offsets = i32(max(groups + 1, 1) if groups < 1 << 20 else 16)
    with pytest.raises(H.HkvException, match="num_groups must be 1 to 4096"):
        H.group_tokens(8, i32(8), groups, offsets, i32(8), workspace=work)


def test_slots_beyond_32_bits():
    rows, x = torch.zeros(8, 8), torch.zeros(4, 8)
    for slots in (1 << 31, (1 << 32) + 2, (1 << 64) + 2):
        with pytest.raises(H.HkvException, match="slots"):
            H.combine_rows(4, rows, None, None, x, slots=slots)
        with pytest.raises(H.HkvException, match="slots"):
            H.combine_rows_backward(4, None, None, None, x, rows, slots=slots)
    for n in (1 << 31, (1 << 64) + 5):
        with pytest.raises(H.HkvException):
            H.group_workspace(n, 8)


GROUP = dict(n=4, groups=SOME, id_type=0, num_groups=8, offsets=SOME, positions=SOME, order=SOME,
             workspace=SOME, workspace_bytes=1 << 20, stream=None)


@pytest.mark.parametrize("change", [
    dict(id_type=2), dict(id_type=-1), dict(num_groups=0), dict(num_groups=4097),
    dict(n=1 << 31), dict(offsets=None), dict(positions=None), dict(groups=None),
    dict(workspace=None), dict(workspace_bytes=8), dict(workspace=SOME + 4),
    dict(groups=SOME + 2), dict(groups=SOME + 4, id_type=1), dict(order=SOME + 1)])
def test_group_tokens_abi_refuses(change):
    assert status("hkv_group_tokens", *{**GROUP, **change}.values()) == H.HKV_ERR_INVALID
    assert H.lib().hkv_last_error()


DISPATCH = dict(n=4, slots=2, dim=8, value_type=0, x=SOME, x_stride=0, positions=SOME,
                num_rows=8, rows=SOME, rows_stride=0, stream=None)


@pytest.mark.parametrize("change", [
    dict(slots=0), dict(dim=0), dict(value_type=8), dict(value_type=-1), dict(x=None),
    dict(positions=None), dict(rows=None), dict(x_stride=7), dict(rows_stride=7),
    dict(n=1 << 30), dict(num_rows=1 << 31), dict(dim=1 << 31), dict(slots=1 << 40),
    dict(x=SOME + 2), dict(rows=SOME + 1), dict(positions=SOME + 2)])
def test_dispatch_rows_abi_refuses(change):
    assert status("hkv_dispatch_rows", *{**DISPATCH, **change}.values()) == H.HKV_ERR_INVALID


@pytest.mark.parametrize("change", [dict(n=0), dict(num_rows=0), dict(n=0, x=None, rows=None)])
def test_dispatch_rows_abi_empty(change):
    assert status("hkv_dispatch_rows", *{**DISPATCH, **change}.values()) == H.HKV_OK


COMBINE = dict(n=4, slots=2, dim=8, value_type=2, rows=SOME, rows_stride=0, num_rows=8,
               positions=SOME, weights=SOME, weight_type=0, out=SOME, out_stride=0, stream=None)


@pytest.mark.parametrize("change,code", [
    (dict(value_type=3), H.HKV_ERR_UNSUPPORTED), (dict(value_type=7), H.HKV_ERR_UNSUPPORTED),
    (dict(value_type=9), H.HKV_ERR_INVALID), (dict(weight_type=1), H.HKV_ERR_INVALID),
    (dict(value_type=0, weight_type=2), H.HKV_ERR_INVALID), (dict(rows=None), H.HKV_ERR_INVALID),
    (dict(out=None), H.HKV_ERR_INVALID), (dict(slots=0), H.HKV_ERR_INVALID),
    (dict(out_stride=4), H.HKV_ERR_INVALID), (dict(rows_stride=4), H.HKV_ERR_INVALID),
    (dict(weights=SOME + 2), H.HKV_ERR_INVALID), (dict(out=SOME + 1), H.HKV_ERR_INVALID),
    (dict(positions=SOME + 1), H.HKV_ERR_INVALID), (dict(n=1 << 31), H.HKV_ERR_INVALID)])
def test_combine_rows_abi_refuses(change, code):
    assert status("hkv_combine_rows", *{**COMBINE, **change}.values()) == code


BACKWARD = dict(n=4, slots=2, dim=8, value_type=2, rows=SOME, rows_stride=0, num_rows=8,
                positions=SOME, weights=SOME, weight_type=0, grad_out=SOME, grad_out_stride=0,
                grad_rows=SOME, grad_rows_stride=0, grad_weights=SOME, stream=None)


@pytest.mark.parametrize("change,code", [
    (dict(value_type=3), H.HKV_ERR_UNSUPPORTED), (dict(weight_type=1), H.HKV_ERR_INVALID),
    (dict(weights=None, weight_type=1), H.HKV_ERR_INVALID), (dict(rows=None), H.HKV_ERR_INVALID),
    (dict(grad_out=None), H.HKV_ERR_INVALID), (dict(grad_rows_stride=3), H.HKV_ERR_INVALID),
    (dict(grad_weights=SOME + 2), H.HKV_ERR_INVALID), (dict(dim=0), H.HKV_ERR_INVALID),
    (dict(grad_rows=None, grad_weights=None), H.HKV_OK), (dict(n=0), H.HKV_OK)])
def test_combine_rows_backward_abi_refuses(change, code):
    assert status("hkv_combine_rows_backward", *{**BACKWARD, **change}.values()) == code


def test_python_refuses_shapes_types_and_devices():
    x, rows, at = torch.zeros(4, 8), torch.zeros(8, 8), i32(4, 2)
    bad = [
        lambda: H.dispatch_rows(5, x, at, rows),  # more tokens than there are
        lambda: H.dispatch_rows(-1, x, at, rows),
        lambda: H.dispatch_rows(4, x, at.long(), rows),
        lambda: H.dispatch_rows(4, x, at[:, :0], rows),
        lambda: H.dispatch_rows(4, x, at.t().contiguous().t(), rows),
        lambda: H.dispatch_rows(4, x.half(), at, rows),
        lambda: H.dispatch_rows(4, x[:, :4], at, rows),
        lambda: H.dispatch_rows(4, x.t(), at, rows),
        lambda: H.dispatch_rows(4, x[:1].expand(4, 8), at, rows),
        lambda: H.dispatch_rows(4, x.bool(), at, rows.bool()),
        lambda: H.dispatch_rows(4, x, at, rows),  # not on a GPU
        lambda: H.combine_rows(4, rows, at, torch.zeros(4, 3), x),
        lambda: H.combine_rows(4, rows, at, torch.zeros(4, 2).half(), x),
        lambda: H.combine_rows(4, rows, at, torch.zeros(2, 4).t(), x),
        lambda: H.combine_rows(4, rows, None, None, x),
        lambda: H.combine_rows(4, rows, None, None, x, slots=0),
        lambda: H.combine_rows(4, rows, None, torch.zeros(4, 2), x, slots=3),
        lambda: H.combine_rows_backward(4, rows, None, None, x, rows),
        lambda: H.combine_rows(4, rows, at, None, x.half()),
        lambda: H.combine_rows(4, rows, at, None, x),  # not on a GPU
        lambda: H.combine_rows_backward(4, None, at, None, x, None, torch.zeros(4, 2)),
        lambda: H.combine_rows_backward(4, rows, at, torch.zeros(4, 2), x.half(), rows),
        lambda: H.combine_rows_backward(4, rows[:6], at, None, x, rows),
        lambda: H.combine_rows_backward(4, rows, at, None, x[:1].expand(4, 8), rows),
        lambda: H.group_tokens(9, i32(8), 4, i32(5), i32(8)),
        lambda: H.group_tokens(8, i32(8), 4, i32(4), i32(8)),
        lambda: H.group_tokens(8, i32(8).short(), 4, i32(5), i32(8)),
        lambda: H.group_tokens(8, i32(8), 4, i32(5), i32(8).long()),
        lambda: H.group_tokens(8, i32(16)[::2], 4, i32(5), i32(8)),
        lambda: H.group_tokens(8, i32(8), 4, i32(5), i32(8)),  # not on a GPU
    ]
    for call in bad:
        with pytest.raises(H.HkvException):
            call()
    # f16 rows with bf16 weights
    with pytest.raises(H.HkvException):
        H.combine_rows(4, rows.half(), at, torch.zeros(4, 2).bfloat16(), x.half())


POOL = dict(num_pages=8, page_tokens=4, num_rows=2, max_pages=3, table_stride=0, refs=SOME,
            table=SOME, lengths=SOME, num_planes=1, device_id=-1)


@pytest.mark.parametrize("change", [
    dict(num_pages=0), dict(page_tokens=0), dict(num_rows=0), dict(max_pages=0), dict(refs=None),
    dict(table=None), dict(lengths=None), dict(refs=SOME + 4), dict(table=SOME + 2),
    dict(table_stride=2), dict(num_planes=129), dict(max_pages=1 << 20, page_tokens=1 << 12),
    dict(num_pages=1 << 31), dict(num_rows=1 << 31), dict(max_pages=1 << 27, page_tokens=1),
    dict(num_rows=1 << 28, max_pages=1 << 10), dict(no_planes=True), dict(plane=None),
    dict(page_bytes=0), dict(page_bytes=(1 << 40) + 1), dict(page_bytes=1 << 32)])
def test_pool_abi_refuses(change):
    v = {**POOL, **change}
    plane = (ctypes.c_void_p * 1)(change.get("plane", SOME))
    size = (ctypes.c_uint64 * 1)(change.get("page_bytes", 64))
    for k in ("no_planes", "plane", "page_bytes"):
        v.pop(k, None)
    o = H._PagesOptions(**v)
    if not change.get("no_planes"):
        o.planes, o.page_bytes = plane, size
    out = ctypes.c_void_p()
    assert status("hkv_pages_create", ctypes.byref(o), None,
                  ctypes.byref(out)) == H.HKV_ERR_INVALID
    assert not out.value


def test_pool_abi_null_handles():
    for name, args in (("hkv_pages_copy", (1, SOME, SOME, None)),
                       ("hkv_pages_fork", (1, SOME, SOME, None)),
                       ("hkv_pages_resize", (1, SOME, SOME, None, None)),
                       ("hkv_pages_free", (1, SOME, None)),
                       ("hkv_pages_hold", (1, SOME, 1, None)),
                       ("hkv_pages_compact", (None, None, None, None))):
        assert status(name, None, *args) == H.HKV_ERR_INVALID
    assert status("hkv_pages_destroy", None) == H.HKV_OK
    assert status("hkv_pages_create", None, None, None) == H.HKV_ERR_INVALID


def test_pool_python_refuses():
    plane = torch.zeros(8, 4, 4)
    for make in (
            lambda: H.PagePool([plane], 4),  # no rows
            lambda: H.PagePool([plane, plane[:7]], 4, 2, 3),
            lambda: H.PagePool([plane.transpose(1, 2).transpose(0, 1)], 4, 2, 3),
            lambda: H.PagePool([plane[:, 1:]], 4, 2, 3),
            lambda: H.PagePool([plane[:, :0]], 4, 2, 3),
            lambda: H.PagePool([plane], 0, 2, 3),
            lambda: H.PagePool([plane], 4, 2, 0),
            lambda: H.PagePool([plane], 4, table=i32(2, 3).long(), lengths=i32(2)),
            lambda: H.PagePool([plane], 4, 3, 3, table=i32(2, 3)),
            lambda: H.PagePool([plane], 4, 2, 3, refs=i32(7)),
            lambda: H.PagePool([plane], 4, 2, 3, lengths=i32(1)),
            lambda: H.PagePool([plane], 4, 2, 3)):  # not on a GPU
        with pytest.raises(H.HkvException):
            make()
