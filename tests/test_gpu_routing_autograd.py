"""What the routing calls do when autograd is watching: they tell it what they changed."""
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
