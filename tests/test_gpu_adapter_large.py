"""Prompt batches so large that every CTA has several tiles: buffers and barriers of the ring come round again."""
import pytest

from tests.test_gpu_adapter import Case

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def rt(built_lib):
    from ugache_b200 import runtime
    return runtime


# 148 CTAs: 45,000 tokens are 352 tiles of 128 or more
@pytest.mark.parametrize("elem", ["bf16", "f16"])
@pytest.mark.parametrize("rank", [16, 24, 64, 128])
@pytest.mark.parametrize("dim,out_dim", [(128, 136), (520, 64)])
def test_several_tiles_a_cta(rt, rank, elem, dim, out_dim):
    c = Case(rt, 45000, 7, rank, dim, out_dim, elem)
    first = c.check(rt)
    base = c.base.clone()
    assert torch.equal(rt.adapter_add(base, c.x, c.down, c.up, c.plan, scale=c.scale, out=base), first)


@pytest.mark.parametrize("G", [40, 1024])
def test_many_groups_that_end_inside_a_tile(rt, G):
    Case(rt, 70000, G, 16, 64, 72, "bf16").check(rt)


# more tiles than 148 CTAs keep a list of
def test_more_ctas_than_the_gpu_holds(rt):
    Case(rt, 700000, 5, 16, 64, 64, "bf16").check(rt)


def test_the_same_again_and_again(rt):
    """Bit for bit, with other work in between and on another stream beside it."""
    c, d = Case(rt, 45000, 24, 64, 512, 256, "bf16"), Case(rt, 20000, 3, 128, 256, 512, "f16")
    call = lambda c: rt.adapter_add(c.base, c.x, c.down, c.up, c.plan, scale=c.scale)  # noqa: E731
    want = call(c), call(d)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for _ in range(20):
        with torch.cuda.stream(side):
            other = call(d)
        assert torch.equal(call(c), want[0])
        side.synchronize()
        assert torch.equal(other, want[1])
