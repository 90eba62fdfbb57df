"""Low-rank adapters against the formula in 64 bits.

Bound: the first product's sum of dim terms (and of the 16 partial sums or fewer that it is cut into) is off by at most (dim + 16) * 2^-23 of the sum of its magnitudes (products of
16-bit values are exact in fp32; an addition inside a matrix instruction may truncate, 2^-23), the scale by 2^-24, the two 16-bit terms by 2^-16 of the
value (2^-8 of 2^-8) and, below the type's normal range, 2^-24 of the token's largest one; the second sum of 2 * rank terms by
2 * rank * 2^-23 of its magnitudes, the result by eps / 2.  fp32: fused multiply-adds, so 2^-24 for 2^-23, and no terms."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


@pytest.fixture(scope="module")
def rt(built_lib):
    from ugache_b200 import runtime
    return runtime


def formula(base, x, down, up, ids, scale):
    """(result, bound) in 64 bits, adapter by adapter."""
    want, slack = base.double(), torch.zeros_like(base, dtype=torch.float64)
    rank, dim = down.shape[1], down.shape[2]
    f = torch.finfo(base.dtype)
    full = base.dtype == torch.float32          # fused multiply-adds, no terms of 16 bits
    add, term, least, sums = (2.0 ** -24, 0.0, 0.0, rank) if full else (2.0 ** -23, 2.0 ** -16, 2.0 ** -24, 2 * rank)
    for a in range(down.shape[0]):
        t = torch.nonzero(ids == a).reshape(-1)
        if not t.numel():
            continue
        s = 1.0 if scale is None else float(scale[a].double())
        d, u = down[a].double(), up[a].double()
        inner = x[t].double() @ d.t() * s
        off = ((dim + 16) * add + 2.0 ** -24) * (x[t].double().abs() @ d.abs().t()) * abs(s)
        off = off + term * inner.abs() + least * inner.abs().amax(1, keepdim=True)
        want[t] += inner @ u.t()
        slack[t] += off @ u.abs().t() + sums * add * ((inner.abs() + off) @ u.abs().t())
    slack = slack + f.eps / 2 * (want.abs() + slack) + (0.0 if full else add) * (want.abs() + slack) + f.smallest_normal * f.eps / 2
    return want, slack


class Case:
    def __init__(self, rt, T, G, rank, dim, out_dim, elem, none=0.2, scaled=True, ids=None, seed=0):
        g = torch.Generator(device="cuda")
        g.manual_seed(seed + T + 7 * rank)
        ty = TYPES[elem]

        def normal(*size):
            return torch.randn(*size, generator=g, device="cuda")

        if ids is None:
            ids = torch.randint(0, G, (T,), generator=g, device="cuda")
            ids[torch.rand(T, generator=g, device="cuda") < none] = -1
        self.ids, self.G = ids, G
        self.plan = rt.route_plan(ids, G)
        self.base, self.x = normal(T, out_dim).to(ty), normal(T, dim).to(ty)
        self.down, self.up = (normal(G, rank, dim) / dim ** 0.5).to(ty), normal(G, out_dim, rank).to(ty)
        self.scale = normal(G) if scaled else None

    def check(self, rt, **kw):
        want, slack = formula(self.base, self.x, self.down, self.up, self.ids, self.scale)
        got = rt.adapter_add(self.base, self.x, self.down, self.up, self.plan, scale=self.scale, **kw)
        assert got.dtype == self.base.dtype and got.shape == self.base.shape
        assert bool(((got.double() - want).abs() <= slack).all())
        assert torch.equal(got[self.ids < 0], self.base[self.ids < 0])
        return got


@pytest.mark.parametrize("elem", sorted(TYPES))
@pytest.mark.parametrize("rank", [1, 4, 8, 12, 16, 24, 32, 40, 64, 72, 128])
@pytest.mark.parametrize("T", [77, 2700])   # single tokens, prompts
def test_ranks(rt, rank, elem, T):
    Case(rt, T, 5, rank, 512, 320, elem).check(rt)


@pytest.mark.parametrize("dim,out_dim", [(1, 1), (8, 8), (33, 17), (256, 256), (264, 1000), (1001, 77), (4096, 40), (72, 4096), (2048, 2056)])
@pytest.mark.parametrize("T,rank", [(1, 16), (40, 16), (700, 64), (2600, 16)])
def test_dims(rt, dim, out_dim, T, rank):
    Case(rt, T, 3, rank, dim, out_dim, "bf16").check(rt)


@pytest.mark.parametrize("T", [0, 1, 15, 16, 17, 31, 64, 127, 128, 129, 255, 256, 257, 1000, 4099])
@pytest.mark.parametrize("G,rank", [(1, 8), (6, 8), (300, 8), (6, 128)])
def test_tokens(rt, T, G, rank):
    Case(rt, T, G, rank, 192, 264, "bf16", scaled=T % 2 == 0).check(rt)


@pytest.mark.parametrize("rank", [16, 64])
@pytest.mark.parametrize("what", ["one adapter", "own adapters", "none", "ragged", "no one without"])
@pytest.mark.parametrize("G", [32, 1024])   # prompts, single tokens
def test_groupings(rt, what, rank, G):
    T = 700
    i = torch.arange(T, device="cuda")
    ids = {"one adapter": torch.full_like(i, G - 1), "own adapters": i % G, "none": torch.full_like(i, -1),
           "ragged": (i.float().sqrt() * 1.3).long(), "no one without": i % 3}[what]
    c = Case(rt, T, G, rank, 256, 128, "f16", ids=ids)
    c.check(rt)


@pytest.mark.parametrize("elem", sorted(TYPES))
@pytest.mark.parametrize("T", [150, 2600])
def test_in_place_and_strided(rt, elem, T):
    c = Case(rt, T, 4, 16, 256, 192, elem)
    want, slack = formula(c.base, c.x, c.down, c.up, c.ids, c.scale)
    base = c.base.clone()
    got = rt.adapter_add(base, c.x, c.down, c.up, c.plan, scale=c.scale, out=base)
    assert got.data_ptr() == base.data_ptr() and bool(((base.double() - want).abs() <= slack).all())
    for pad in (8, 1):     # on and off the 16-byte boundaries
        wide = torch.full((T, 192 + 2 * pad), 3.0, dtype=c.base.dtype, device="cuda")
        view = wide[:, pad:pad + 192]
        view.copy_(c.base)
        x = torch.zeros((T, 256 + pad), dtype=c.base.dtype, device="cuda")[:, :256]
        x.copy_(c.x)
        rt.adapter_add(view, x, c.down, c.up, c.plan, scale=c.scale, out=view)
        assert bool(((view.double() - want).abs() <= slack).all())
        view.fill_(3.0)
        assert bool((wide == 3.0).all())


@pytest.mark.parametrize("T", [90, 3000])
def test_both_matrices_in_one_row(rt, T):
    """An adapter as a row of a table: down and up behind one another."""
    G, r, H, N = 7, 16, 320, 256
    c = Case(rt, T, G, r, H, N, "bf16")
    table = torch.cat([c.down.reshape(G, -1), c.up.reshape(G, -1)], 1)
    want = rt.adapter_add(c.base, c.x, c.down, c.up, c.plan, scale=c.scale)
    c.down, c.up = table[:, :r * H].view(G, r, H), table[:, r * H:].view(G, N, r)
    assert c.down.stride(0) == r * (H + N)
    assert torch.equal(c.check(rt), want)


@pytest.mark.parametrize("elem", sorted(TYPES))
@pytest.mark.parametrize("T", [60, 2600])
def test_magnitudes(rt, elem, T):
    """Rank products far above and below the type's range; the result is in it."""
    for factor in (2.0 ** 17, 2.0 ** -20):
        c = Case(rt, T, 3, 16, 256, 128, elem, scaled=False)
        c.scale = torch.full((3,), factor, device="cuda")
        c.up = (c.up.float() * (2.0 ** -14 if factor > 1 else 1)).to(c.up.dtype)
        c.check(rt)


@pytest.mark.parametrize("T", [64, 2900])
def test_non_finite_values_stay_with_their_token(rt, T):
    c = Case(rt, T, 3, 16, 256, 128, "bf16", none=0.0)
    clean = rt.adapter_add(c.base, c.x, c.down, c.up, c.plan)
    c.x[5, 3], c.x[6, 7] = float("nan"), float("inf")
    got = rt.adapter_add(c.base, c.x, c.down, c.up, c.plan)
    rest = torch.arange(T, device="cuda")
    rest = rest[(rest != 5) & (rest != 6)]
    assert torch.equal(got[rest], clean[rest])
    assert bool(torch.isnan(got[5]).all()) and not bool(torch.isfinite(got[6]).any())


@pytest.mark.parametrize("T", [64, 2900])
def test_adapters_that_no_token_names_are_not_read(rt, T):
    c = Case(rt, T, 4, 16, 256, 128, "bf16")
    c.ids = torch.where(c.ids == 2, torch.full_like(c.ids, 1), c.ids)
    c.plan = rt.route_plan(c.ids, 4)
    c.down[2], c.up[2] = float("nan"), float("nan")
    c.check(rt)


@pytest.mark.parametrize("T", [300, 5000])
def test_same_results_again(rt, T):
    c = Case(rt, T, 5, 16, 512, 256, "bf16", none=0.0)
    whole = rt.adapter_add(c.base, c.x, c.down, c.up, c.plan, scale=c.scale)
    assert torch.equal(whole, rt.adapter_add(c.base, c.x, c.down, c.up, c.plan, scale=c.scale))


@pytest.mark.parametrize("T", [40, 2700])
def test_far_adapters(rt, T):
    """Adapter offsets beyond 32 bits."""
    c = Case(rt, T, 3, 8, 64, 64, "f16")
    stride = (1 << 30) + 64
    room = torch.empty(3 * stride, dtype=torch.float16, device="cuda")
    down, up = room.as_strided((3, 8, 64), (stride, 64, 1)), room.as_strided((3, 64, 8), (stride, 8, 1), 1024)
    down.copy_(c.down)
    up.copy_(c.up)
    c.down, c.up = down, up
    c.check(rt)


@pytest.mark.parametrize("elem", sorted(TYPES))
def test_far_rows(rt, elem):
    """Row offsets beyond 32 bits, in elements and in bytes; prompts."""
    c = Case(rt, 2600, 2, 16, 64, 64, elem)
    stride = (1 << 21) + 8           # 2600 rows of it pass 2^32 elements
    room = torch.empty(2600 * stride, dtype=c.base.dtype, device="cuda")
    base, x = room.as_strided((2600, 64), (stride, 1)), room.as_strided((2600, 64), (stride, 1), 1024)
    base.copy_(c.base)
    x.copy_(c.x)
    want, slack = formula(c.base, c.x, c.down, c.up, c.ids, c.scale)
    rt.adapter_add(base, x, c.down, c.up, c.plan, scale=c.scale, out=base)
    assert bool(((base.double() - want).abs() <= slack).all())
    few = rt.route_plan(c.ids[-20:], 2)                        # single tokens: the last rows of the room
    got = rt.adapter_add(c.base[-20:], x[-20:], c.down, c.up, few, scale=c.scale)
    assert bool(((got.double() - want[-20:]).abs() <= slack[-20:]).all())


def test_no_wait_ran_out(rt):
    import ctypes as C

    from ugache_b200 import _lib
    n = C.c_uint32(7)
    _lib.check(_lib.lib().ugc_adapter_stalled(0, C.byref(n)))
    assert n.value == 0


def test_refusals(rt):
    c = Case(rt, 16, 3, 8, 64, 32, "bf16")
    b, x, d, u, p = c.base, c.x, c.down, c.up, c.plan
    for call, error in (
            (lambda: rt.adapter_add(b.cpu(), x, d, u, p), ValueError), (lambda: rt.adapter_add(b, x[:9], d, u, p), ValueError),
            (lambda: rt.adapter_add(b, x.half(), d, u, p), TypeError), (lambda: rt.adapter_add(b, x, d.half(), u, p), TypeError),
            (lambda: rt.adapter_add(b, x, d[0], u, p), ValueError), (lambda: rt.adapter_add(b, x, d, u[:2], p), ValueError),
            (lambda: rt.adapter_add(b, x, d[:, :, :32], u, p), ValueError), (lambda: rt.adapter_add(b, x, d[:, :4], u, p), ValueError),
            (lambda: rt.adapter_add(b, x, d[:2], u[:2], p), ValueError), (lambda: rt.adapter_add(b, x, d, u, p, scale=torch.ones(2, device="cuda")), ValueError),
            (lambda: rt.adapter_add(b, x, d, u, p, scale=torch.ones(3, device="cuda").half()), TypeError),
            (lambda: rt.adapter_add(b.double(), x.double(), d.double(), u.double(), p), TypeError),
            (lambda: rt.adapter_add(b, x, torch.zeros(3, 136, 64, dtype=b.dtype, device="cuda"), torch.zeros(3, 32, 136, dtype=b.dtype, device="cuda"), p), rt.UgcError),
            (lambda: rt.adapter_add(b, x, d, u, p, out=b[:, :16]), ValueError)):
        with pytest.raises(error):
            call()


@pytest.mark.parametrize("T", [64, 3000])
def test_captured_and_replayed(rt, T):
    c = Case(rt, T, 9, 16, 512, 256, "bf16")
    out = torch.empty_like(c.base)

    def step():
        plan = rt.route_plan(c.ids, 9)
        rt.adapter_add(c.base, c.x, c.down, c.up, plan, scale=c.scale, out=out)

    step()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    for i in range(3):
        c.ids.copy_(torch.randint(-1, 9, (T,), device="cuda"))
        c.x.normal_()
        g.replay()
        want, slack = formula(c.base, c.x, c.down, c.up, c.ids, c.scale)
        assert bool(((out.double() - want).abs() <= slack).all())


@pytest.mark.parametrize("T", [64, 2700])
def test_bad_plans_stay_in_bounds(rt, T):
    """Tokens outside the batch are skipped and offsets clamped, whatever a caller put there."""
    c = Case(rt, T, 4, 16, 256, 128, "bf16", none=0.0)
    want, slack = formula(c.base, c.x, c.down, c.up, c.ids, c.scale)
    order = c.plan.order.clone()
    gone = order[[1, T // 2, T - 1]].long()
    order[1], order[T // 2], order[T - 1] = -1, T, 1 << 30
    out = torch.full_like(c.base, 9.0)
    rt.adapter_add(c.base, c.x, c.down, c.up, c.plan._replace(order=order), scale=c.scale, out=out)
    kept = torch.ones(T, dtype=torch.bool, device="cuda")
    kept[gone] = False
    assert bool(((out.double() - want).abs() <= slack)[kept].all()) and bool((out[gone] == 9.0).all())
    offsets = c.plan.offsets.clone()
    offsets[-1] = 1 << 30        # beyond the batch: as if it were its end
    assert torch.equal(rt.adapter_add(c.base, c.x, c.down, c.up, c.plan._replace(offsets=offsets), scale=c.scale),
                       rt.adapter_add(c.base, c.x, c.down, c.up, c.plan, scale=c.scale))


def test_two_streams_at_once(rt):
    """Prompts and single tokens side by side: the calls share nothing."""
    big, small = Case(rt, 6000, 6, 64, 1024, 1024, "bf16"), Case(rt, 64, 9, 16, 1024, 1024, "bf16")
    run = lambda c: rt.adapter_add(c.base, c.x, c.down, c.up, c.plan, scale=c.scale)  # noqa: E731
    want = [run(big), run(small)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    got = []
    for i in range(24):
        with torch.cuda.stream(streams[i % 4]):
            got.append((i % 2, run((big, small)[i % 2])))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[k]) for k, y in got)


@pytest.mark.parametrize("T", [200, 3000])
def test_adapters_behind_the_cache(rt, T):
    """The run as a server makes it: adapters are rows of a table in host memory, the hot ones cached; a batch's
    distinct adapters are looked up once and applied through the lookup's own index."""
    A, r, H, N = 60, 16, 128, 192
    per = r * (H + N)
    g = torch.Generator()
    g.manual_seed(3)
    table = (torch.randn((A, per), generator=g) / 8).to(torch.float16).pin_memory()
    cache = rt.Cache(1, A, per * 2, 0.4, max_batch=4096)
    cache.set_placement(rt.solve_placement("rep", 1, np.arange(A, dtype=np.uint32), None, 40.0))
    cache.build(0, 0, table.data_ptr())
    names = torch.randint(0, A + 6, (T,), generator=g).cuda()     # some name no adapter of the table
    rows, _, inverse, _ = cache.lookup_unique(0, names)
    n = min(T, 1024)
    rows = rows[:n].view(torch.float16)
    down, up = rows[:, :r * H].view(n, r, H), rows[:, r * H:].view(n, N, r)
    plan = rt.route_plan(inverse, n)
    x, base = torch.randn((T, H), device="cuda").half(), torch.randn((T, N), device="cuda").half()
    got = rt.adapter_add(base, x, down, up, plan)
    dev = table.cuda()
    ids = torch.where(names < A, names, torch.full_like(names, -1))
    want, slack = formula(base, x, dev[:, :r * H].view(A, r, H), dev[:, r * H:].view(A, N, r), ids, None)
    assert bool(((got.double() - want).abs() <= slack).all())
    assert torch.equal(got[ids < 0], base[ids < 0]) and bool((ids < 0).any())
    cache.close()
