"""Plan, dispatch and combine where sizes and addresses decide what is read and added when."""
import numpy as np
import pytest

from tests.test_gpu_routing import Case, check_plan

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def rt(built_lib):
    from ugache_b200 import runtime
    return runtime


@pytest.mark.parametrize("elem,dim", [("f16", 1001), ("bf16", 77), ("bf16", 4097), ("f32", 255), ("f32", 9), ("f16", 6), ("bf16", 2050)])
@pytest.mark.parametrize("k", [1, 3, 6])
def test_products_of_odd_rows_do_not_depend_on_the_batch(rt, elem, dim, k):
    """A token's weights' gradients are the same bit for bit wherever its rows stand: alone, and in a batch whose other
    tokens move its rows to other addresses.  So are its rows."""
    c = Case(rt, 900, k, dim, elem, G=7, dropped=0.1)
    ids = torch.full((900, k), -1, dtype=torch.int64, device="cuda")
    starts = c.plan.offsets.long()
    ids[c.taken] = torch.bucketize(c.pos[c.taken], starts[1:], right=True)
    assert torch.equal(rt.route_plan(ids, 7).position, c.plan.position)
    dx, dw = rt.route_dispatch_grad(c.rows, c.plan, weights=c.w, x=c.x)
    drows, dw2 = rt.route_combine_grad(c.x, c.plan, weights=c.w, rows=c.rows)
    c.check_gathered(dx)
    c.check_dots(dw)
    c.check_spread(drows)
    assert torch.equal(dw, dw2)
    for first, n in ((0, 5), (3, 8), (450, 1), (877, 23)):
        part = slice(first, first + n)
        plan = rt.route_plan(ids[part].contiguous(), 7)
        at, whole = plan.position[plan.position >= 0].long(), c.pos[part][c.taken[part]]
        rows = torch.zeros((n * k, dim), dtype=c.ty, device="cuda")
        rows[at] = c.rows[whole]
        x, w = c.x[part].clone(), c.w[part].clone()
        one = rt.route_dispatch_grad(rows, plan, weights=w, x=x)
        two = rt.route_combine_grad(x, plan, weights=w, rows=rows)
        assert torch.equal(one[0], dx[part]) and torch.equal(one[1], dw[part])
        assert torch.equal(two[0][at], drows[whole]) and torch.equal(two[1], dw[part])


# one CTA up to 1024 ids, a cluster of eight up to 65,536 (its tiles full there), parts beyond
@pytest.mark.parametrize("n", [65528, 65535, 65536, 151552, 151553])
@pytest.mark.parametrize("G", [1, 256, 1024])
def test_plans_at_the_largest_cluster(rt, n, G):
    check_plan(rt, np.random.default_rng(n + G).integers(-1, G + 1, n), G)


# From 148 * 2048 * 4 pieces of 16 bytes on a thread has several: four with up to two choices and where pieces come in
# fours, else two, else one.
@pytest.mark.parametrize("elem,dim", [("bf16", 2048), ("f16", 2064), ("bf16", 2056), ("f32", 1024), ("f32", 1032), ("f32", 1028)])
@pytest.mark.parametrize("k", [1, 2, 3, 5])
@pytest.mark.parametrize("weighted", [True, False])
def test_rows_of_large_batches(rt, elem, dim, k, weighted):
    T = 4900
    c = Case(rt, T, k, dim, elem, G=5, dropped=0.1, weighted=weighted)
    assert T * (dim * c.ty.itemsize // 16) >= 148 * 2048 * 4
    y = rt.route_combine(c.rows, c.plan, weights=c.w)
    dx, none = rt.route_dispatch_grad(c.rows, c.plan, weights=c.w)
    assert none is None and torch.equal(dx, y)
    c.check_gathered(y)
    # the same tokens in a small batch: bit for bit
    ids = torch.full((T, k), -1, dtype=torch.int64, device="cuda")
    ids[c.taken] = torch.bucketize(c.pos[c.taken], c.plan.offsets.long()[1:], right=True)
    for part in (slice(0, 9), slice(T - 20, T)):
        plan = rt.route_plan(ids[part].contiguous(), 5)
        rows = torch.zeros((ids[part].numel(), dim), dtype=c.ty, device="cuda")
        rows[plan.position[plan.position >= 0].long()] = c.rows[c.pos[part][c.taken[part]]]
        assert torch.equal(rt.route_combine(rows, plan, weights=None if c.w is None else c.w[part].contiguous()), y[part])
