"""Routing operators: what the C interface refuses, before it touches a GPU."""
import ctypes as C

import pytest

INVALID, UNSUPPORTED = 1, 8
A, B, D = 1 << 20, 1 << 21, 1 << 22   # aligned addresses that nothing reads


@pytest.fixture(scope="module")
def L(built_lib):
    from ugache_b200 import _lib
    return _lib.lib()


def plan(L, device=0, ids=A, id_bytes=8, tokens=4, k=2, groups=8, offsets=B, order=B, position=B, space=None, size=0):
    return L.ugc_route_plan(device, ids, id_bytes, tokens, k, groups, offsets, order, position, space, size, None)


@pytest.mark.parametrize("kw", [dict(ids=None), dict(ids=A + 4), dict(id_bytes=2), dict(k=0), dict(groups=0), dict(groups=-1),
                                dict(groups=1025), dict(tokens=1 << 28, k=2), dict(tokens=1 << 63, k=2), dict(offsets=None),
                                dict(order=None), dict(position=B + 2), dict(tokens=1 << 20),   # wants a workspace
                                dict(tokens=1 << 20, space=A, size=64)])
def test_plan(L, kw):
    assert plan(L, **kw) == INVALID
    assert L.ugc_last_error()


def test_plan_workspace(L):
    n = C.c_size_t(1)
    assert L.ugc_route_plan_workspace(0, 1, 1, C.byref(n)) == 0 and n.value == 0
    assert L.ugc_route_plan_workspace(64, 8, 1024, C.byref(n)) == 0 and n.value == 0
    assert L.ugc_route_plan_workspace(1 << 25, 8, 1024, C.byref(n)) == 0 and n.value > 0
    assert L.ugc_route_plan_workspace(1, 1, 1, None) == INVALID
    assert L.ugc_route_plan_workspace(1, 0, 1, C.byref(n)) == INVALID


def rows_call(L, call, elem=0, tokens=4, k=2, dim=8, a=A, a_stride=8, b=A, b_stride=8, w=D, position=D, routed=D, out=B, out_stride=8,
              dw=None):
    if call == "dispatch":
        return L.ugc_route_dispatch(0, elem, a, a_stride, w, position, routed, tokens, k, dim, out, out_stride, None)
    if call == "dispatch_grad":
        return L.ugc_route_dispatch_grad(0, elem, a, a_stride, b, b_stride, w, position, tokens, k, dim, out, out_stride, dw, None)
    if call == "combine":
        return L.ugc_route_combine(0, elem, a, a_stride, w, position, tokens, k, dim, out, out_stride, None)
    return L.ugc_route_combine_grad(0, elem, a, a_stride, b, b_stride, w, position, routed, tokens, k, dim, out, out_stride, dw, None)


@pytest.mark.parametrize("call", ["dispatch", "dispatch_grad", "combine", "combine_grad"])
@pytest.mark.parametrize("kw", [dict(elem=3), dict(elem=-1), dict(k=0), dict(dim=0), dict(dim=1 << 29), dict(tokens=1 << 28, k=2),
                                dict(a=None), dict(a=A + 2), dict(a_stride=7), dict(a_stride=-8), dict(out=None), dict(out_stride=0),
                                dict(w=D + 1), dict(position=None), dict(position=D + 1)])
def test_rows(L, call, kw):
    assert rows_call(L, call, **kw) == INVALID
    assert L.ugc_last_error()


@pytest.mark.parametrize("call", ["dispatch_grad", "combine_grad"])
@pytest.mark.parametrize("kw", [dict(b=None), dict(b_stride=7), dict(dw=D + 2)])
def test_rows_with_products(L, call, kw):
    assert rows_call(L, call, **{"dw": D, **kw}) == INVALID


@pytest.mark.parametrize("call", ["dispatch", "dispatch_grad", "combine", "combine_grad"])
def test_no_tokens(L, call):
    assert rows_call(L, call, tokens=0, a=None, b=None, w=None, position=None, routed=None, out=None) == 0


def adapter(L, elem=2, base=A, base_stride=8, x=A, x_stride=16, down=A, down_stride=64, up=A, up_stride=64, scale=None, offsets=D,
            order=D, tokens=4, groups=3, rank=4, dim=16, out_dim=8, out=B, out_stride=8,
            space=None, size=0):
    return L.ugc_adapter_add(0, elem, base, base_stride, x, x_stride, down, down_stride, up, up_stride, scale, offsets, order,
                             tokens, groups, rank, dim, out_dim, out, out_stride, space, size, None)


@pytest.mark.parametrize("kw,status", [
    (dict(elem=3), INVALID), (dict(elem=7), INVALID), (dict(rank=0), INVALID), (dict(rank=129), UNSUPPORTED),
    (dict(dim=0), INVALID), (dict(out_dim=0), INVALID), (dict(groups=0), INVALID), (dict(groups=1025), INVALID),
    (dict(tokens=(1 << 28) + 1), INVALID), (dict(base=None), INVALID), (dict(x=A + 1), INVALID), (dict(x_stride=15), INVALID),
    (dict(base_stride=7), INVALID), (dict(out=None), INVALID), (dict(down=None), INVALID), (dict(down_stride=63), INVALID),
    (dict(up_stride=31), INVALID), (dict(offsets=None), INVALID), (dict(order=None), INVALID), (dict(scale=D + 2), INVALID),
    (dict(out=A, out_stride=16), INVALID), (dict(tokens=8192), INVALID), (dict(tokens=8192, space=A, size=1 << 10), INVALID),
    (dict(tokens=8192, space=A + 8, size=1 << 30), INVALID)])
def test_adapter(L, kw, status):
    assert adapter(L, **kw) == status
    assert L.ugc_last_error()


def test_adapter_workspace(L):
    n = C.c_size_t(1)
    assert L.ugc_adapter_workspace(4, 3, 4, 16, 8, C.byref(n)) == 0 and n.value == 0
    assert L.ugc_adapter_workspace(8192, 3, 4, 16, 8, C.byref(n)) == 0 and n.value > 0
    assert L.ugc_adapter_workspace(8192, 3, 4, 16, 8, None) == INVALID
    assert L.ugc_adapter_stalled(0, None) == INVALID


def test_adapter_no_tokens(L):
    assert adapter(L, tokens=0, base=None, x=None, down=None, up=None, offsets=None, order=None, out=None) == 0

