"""What the routing calls do when autograd is watching: they record nothing, say so, and tell it what they changed."""
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def rt(built_lib):
    from ugache_b200 import runtime
    return runtime


@pytest.fixture(scope="module")
def t(rt):
    torch.manual_seed(2)

    class T:
        plan = rt.route_plan(torch.randint(0, 4, (12, 2), device="cuda"), 4)
        one = rt.route_plan(torch.randint(0, 4, (12,), device="cuda"), 4)
        x, rows, w = torch.randn(12, 16, device="cuda"), torch.randn(24, 16, device="cuda"), torch.rand(12, 2, device="cuda")
        base, down, up = torch.randn(12, 8, device="cuda"), torch.randn(4, 3, 16, device="cuda"), torch.randn(4, 8, 3, device="cuda")
        scale = torch.rand(4, device="cuda")
    return T


def calls(rt, t):
    """(call, its tensors) of all five."""
    return ((lambda x, w: rt.route_dispatch(x, t.plan, weights=w), (t.x, t.w)),
            (lambda rows, w, x: rt.route_dispatch_grad(rows, t.plan, weights=w, x=x), (t.rows, t.w, t.x)),
            (lambda rows, w: rt.route_combine(rows, t.plan, weights=w), (t.rows, t.w)),
            (lambda x, w, rows: rt.route_combine_grad(x, t.plan, weights=w, rows=rows), (t.x, t.w, t.rows)),
            (lambda base, x, down, up, scale: rt.adapter_add(base, x, down, up, t.one, scale=scale), (t.base, t.x, t.down, t.up, t.scale)))


def first(y):
    return y[0] if isinstance(y, tuple) else y


def test_a_gradient_that_would_be_lost_is_refused(rt, t):
    for call, args in calls(rt, t):
        want = first(call(*args))
        for i in range(len(args)):
            leaf = [a.clone().requires_grad_() if j == i else a for j, a in enumerate(args)]
            made = [a * 1 for a in leaf]        # not a leaf: it has a history
            for given in (leaf, made):
                with pytest.raises(ValueError, match="requires a gradient"):
                    call(*given)
                with torch.no_grad():
                    assert torch.equal(first(call(*given)), want)
                with torch.inference_mode():
                    assert torch.equal(first(call(*given)), want)


def test_inside_a_function_of_its_own(rt, t):
    class Dispatch(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x):
            return rt.route_dispatch(x, t.plan)

        @staticmethod
        def backward(ctx, g):
            return rt.route_dispatch_grad(g, t.plan)[0]

    x = t.x.clone().requires_grad_()
    Dispatch.apply(x).sum().backward()
    assert torch.equal(x.grad, torch.full_like(x, 2.0))


def test_what_is_written_counts_as_changed(rt, t):
    """An output of the caller that a graph has saved: its backward pass says that the value is gone."""
    outs = ((lambda o: rt.route_dispatch(t.x, t.plan, out=o), t.rows), (lambda o: rt.route_dispatch_grad(t.rows, t.plan, dx=o), t.x),
            (lambda o: rt.route_combine(t.rows, t.plan, out=o), t.x), (lambda o: rt.route_combine_grad(t.x, t.plan, drows=o), t.rows),
            (lambda o: rt.adapter_add(o, t.x, t.down, t.up, t.one, out=o), t.base))
    for call, like in outs:
        out, leaf = like.clone(), torch.ones_like(like).requires_grad_()
        y = (out * leaf).sum()
        before = out._version
        call(out)
        assert out._version == before + 1
        with pytest.raises(RuntimeError, match="inplace"):
            y.backward()
        with torch.inference_mode():
            made = like.clone()
            call(made)
        call(made)      # a tensor without a version takes it as before


def test_an_output_that_requires_a_gradient_is_refused(rt, t):
    with pytest.raises(ValueError, match="requires a gradient"):
        rt.route_combine(t.rows, t.plan, out=t.x.clone().requires_grad_())
