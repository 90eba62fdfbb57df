"""Plan, dispatch and combine where sizes and addresses decide what is read and added when."""
import pytest

from tests.test_gpu_routing import Case

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
