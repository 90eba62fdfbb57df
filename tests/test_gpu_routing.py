"""Plan, dispatch and combine with their gradients, against the formulas in 64 bits.

Bounds: a product or fused multiply-add in fp32 is off by at most 2^-24 of its value, a sum of n of them
by n * 2^-24 of the sum of the magnitudes, and the rounding to a row's type by eps / 2 of the result
(plus half its smallest subnormal)."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

U = 2.0 ** -24
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def rt(built_lib):
    from ugache_b200 import runtime
    return runtime


def sorted_plan(ids, G):
    flat = np.asarray(ids).reshape(-1).astype(np.int64)
    key = np.where((flat >= 0) & (flat < G), flat, G)
    order = np.argsort(key, kind="stable")
    offsets = np.concatenate([[0], np.cumsum(np.bincount(key, minlength=G + 1)[:G])])
    position = np.empty(len(flat), np.int64)
    position[order] = np.arange(len(flat))
    position[key == G] = -1
    return offsets, order, position.reshape(np.asarray(ids).shape)


def check_plan(rt, ids, G, dtype=torch.int64):
    p = rt.route_plan(torch.from_numpy(np.asarray(ids)).to(dtype).cuda(), G)
    for got, want in zip(p, sorted_plan(ids, G)):
        assert got.dtype == torch.int32 and got.shape == want.shape
        assert np.array_equal(got.cpu().numpy(), want)
    return p


# one part (a CTA) up to 8192 ids, 148 parts of one tile up to 1,212,416, more tiles a part beyond
@pytest.mark.parametrize("n", [0, 1, 2, 31, 32, 33, 127, 128, 129, 1000, 1024, 1025, 8191, 8192, 8193, 20000, 65537, 1212416, 1212417, 3000001])
@pytest.mark.parametrize("G", [1, 7, 256, 1024])
def test_plan(rt, n, G):
    rng = np.random.default_rng(n + G)
    ids = rng.integers(-1 if n % 2 else 0, G + (n % 3 == 0), n)   # ids outside on both sides, in some sizes
    check_plan(rt, ids, G, torch.int64 if n % 2 else torch.int32)


# shared memory of a CTA on both sides of what a launch gets without asking
@pytest.mark.parametrize("n", [30000, 36000, 40000, 42000, 44000, 46000, 48000, 50000])
@pytest.mark.parametrize("G", [1, 256, 500, 700])
def test_plan_shared_memory(rt, n, G):
    check_plan(rt, np.random.default_rng(n).integers(0, G, n), G)


@pytest.mark.parametrize("shape", [(5, 3), (4096, 8), (1, 1), (0, 4), (17, 20)])
def test_plan_shapes(rt, shape):
    check_plan(rt, np.random.default_rng(1).integers(0, 12, shape), 12)


@pytest.mark.parametrize("n", [300, 30000])
@pytest.mark.parametrize("what", ["one group", "all outside", "far outside", "sorted", "reversed", "runs"])
def test_plan_values(rt, n, what):
    G = 65
    i = np.arange(n)
    ids = {"one group": np.full(n, 64), "all outside": np.full(n, 65), "sorted": i * G // n, "reversed": (n - 1 - i) * G // n,
           "far outside": np.where(i % 3, i % G, (1 << 40) + i % G), "runs": (i // 100) % G}[what]
    check_plan(rt, ids, G)
    if what == "far outside":
        check_plan(rt, np.where(i % 3, i % G, -(1 << 40) + i % G), G)
        check_plan(rt, np.where(i % 3, i % G, -(1 << 31)), G, torch.int32)


def test_plan_refuses(rt):
    ids = torch.zeros((4, 2), dtype=torch.int64, device="cuda")
    for bad, error in ((ids.cpu(), ValueError), (ids.float(), TypeError), (ids.reshape(2, 2, 2), ValueError), ([1, 2], TypeError)):
        with pytest.raises(error):
            rt.route_plan(bad, 4)
    for G in (0, -1, 1025, 1 << 40):
        with pytest.raises(rt.UgcError):
            rt.route_plan(ids, G)
    with pytest.raises(rt.UgcError):
        rt.route_plan(ids[:, :0], 4)


def test_plan_strided_ids(rt):
    wide = torch.randint(0, 9, (50, 16), device="cuda")
    p, q = rt.route_plan(wide[:, ::2], 9), rt.route_plan(wide[:, ::2].contiguous(), 9)
    assert all(torch.equal(a, b) for a, b in zip(p, q))


# ---- rows ----------------------------------------------------------------------------------

class Case:
    """Inputs on the GPU, and what the formulas give for them in 64 bits."""

    def __init__(self, rt, T, k, dim, elem, G=9, dropped=0.2, weighted=True, seed=0):
        g = torch.Generator(device="cuda")
        g.manual_seed(seed + 1000 * T + k)
        self.T, self.k, self.dim, self.ty = T, k, dim, TYPES[elem]
        ids = torch.randint(0, G, (T, k), generator=g, device="cuda")      # the same group may come twice
        ids[torch.rand((T, k), generator=g, device="cuda") < dropped] = -1
        self.plan = rt.route_plan(ids, G)
        self.x = torch.randn((T, dim), generator=g, device="cuda").to(self.ty)
        self.rows = torch.randn((T * k, dim), generator=g, device="cuda").to(self.ty)
        self.w = torch.randn((T, k), generator=g, device="cuda") if weighted else None
        self.pos = self.plan.position.long()
        self.taken = self.pos >= 0
        w = torch.ones((T, k), dtype=torch.float64, device="cuda") if self.w is None else self.w.double()
        self.w64 = torch.where(self.taken, w, torch.zeros_like(w))

    def picked(self):
        return torch.where(self.taken[:, :, None], self.rows.double()[self.pos.clamp(min=0)], torch.zeros((), dtype=torch.float64, device="cuda"))

    def spread(self):
        want = torch.zeros((self.T * self.k, self.dim), dtype=torch.float64, device="cuda")
        want[self.pos[self.taken]] = (self.w64[:, :, None] * self.x.double()[:, None, :])[self.taken]
        return want

    def check_rounded(self, got, want, sums):
        """got: rounded to the rows' type; sums: magnitude of what was added up, times the additions."""
        f = torch.finfo(self.ty)
        own = 0.0 if self.ty == torch.float32 else f.eps / 2
        bound = own * (want.abs() + U * sums) + U * sums + f.smallest_normal * f.eps / 2 + 2.0 ** -149
        assert got.dtype == self.ty and got.shape == want.shape
        assert bool(((got.double() - want).abs() <= bound).all())

    def check_spread(self, got):
        want = self.spread()
        if self.w is None:
            assert got.dtype == self.ty and torch.equal(got.double(), want)
        else:
            self.check_rounded(got, want, want.abs())

    def check_gathered(self, got):
        parts = self.picked() * self.w64[:, :, None]
        self.check_rounded(got, parts.sum(1), self.k * parts.abs().sum(1))

    def check_dots(self, got):
        parts = self.picked() * self.x.double()[:, None, :]
        assert got.dtype == torch.float32 and got.shape == (self.T, self.k)
        assert bool(((got.double() - parts.sum(2)).abs() <= U * self.dim * parts.abs().sum(2) + 2.0 ** -149).all())
        assert bool((got[~self.taken] == 0).all())

    def check_all(self, rt):
        x, rows, w, plan = self.x, self.rows, self.w, self.plan
        self.check_spread(rt.route_dispatch(x, plan, weights=w))
        self.check_gathered(rt.route_combine(rows, plan, weights=w))
        dx, none = rt.route_dispatch_grad(rows, plan, weights=w)
        assert none is None
        self.check_gathered(dx)
        drows, none = rt.route_combine_grad(x, plan, weights=w)
        assert none is None
        self.check_spread(drows)
        dx, dw = rt.route_dispatch_grad(rows, plan, weights=w, x=x)
        self.check_gathered(dx)
        self.check_dots(dw)
        drows, dw = rt.route_combine_grad(x, plan, weights=w, rows=rows)
        self.check_spread(drows)
        self.check_dots(dw)


@pytest.mark.parametrize("elem", sorted(TYPES))
@pytest.mark.parametrize("dim", [1, 2, 3, 8, 36, 64, 100, 255, 1001, 2048, 4104])
def test_rows_by_dim(rt, dim, elem):
    Case(rt, 37, 3, dim, elem).check_all(rt)


@pytest.mark.parametrize("k", [1, 2, 4, 5, 8, 9, 20])
@pytest.mark.parametrize("weighted", [True, False])
def test_rows_by_choices(rt, k, weighted):
    Case(rt, 29, k, 264, "bf16", weighted=weighted).check_all(rt)


@pytest.mark.parametrize("T", [0, 1, 2, 300, 5000])
def test_rows_by_tokens(rt, T):
    Case(rt, T, 6, 128, "f16").check_all(rt)


@pytest.mark.parametrize("dropped", [0.0, 1.0])
def test_rows_dropped(rt, dropped):
    Case(rt, 65, 4, 520, "bf16", dropped=dropped).check_all(rt)


def test_rows_of_one_dimensional_ids(rt):
    ids = torch.tensor([3, 0, -1, 3, 1], device="cuda")
    plan = rt.route_plan(ids, 4)
    x = torch.randn(5, 24, device="cuda")
    out = rt.route_dispatch(x, plan)
    assert torch.equal(out, torch.cat([x[[1, 4, 0, 3]], torch.zeros(1, 24, device="cuda")]))
    back = rt.route_combine(out, plan)
    x[2] = 0
    assert torch.equal(back, x)


@pytest.mark.parametrize("elem", sorted(TYPES))
@pytest.mark.parametrize("offset,stride", [(0, 200), (1, 201), (2, 202), (8, 208), (3, 4096)])
def test_rows_strided(rt, elem, offset, stride):
    """Rows apart from one another and off the 16-byte boundaries; what lies between them stays as it was."""
    c = Case(rt, 33, 4, 192, elem)

    def within(t):
        big = torch.full((t.shape[0] + 1, stride), 7.0, dtype=t.dtype, device="cuda")
        view = big.reshape(-1)[offset:offset + t.shape[0] * stride].reshape(t.shape[0], stride)[:, :t.shape[1]]
        view.copy_(t)
        return big, view

    def untouched(big, view):
        view.fill_(7.0)
        return bool((big == 7.0).all())

    _, x = within(c.x)
    _, rows = within(c.rows)
    for spread in (lambda out: rt.route_dispatch(x, c.plan, weights=c.w, out=out),
                   lambda out: rt.route_combine_grad(x, c.plan, weights=c.w, drows=out)[0],
                   lambda out: rt.route_combine_grad(x, c.plan, weights=c.w, rows=rows, drows=out)[0]):
        big, out = within(torch.zeros_like(c.rows))
        got = spread(out)
        assert got.data_ptr() == out.data_ptr()
        c.check_spread(got)
        assert untouched(big, out)
    for gather in (lambda out: rt.route_combine(rows, c.plan, weights=c.w, out=out),
                   lambda out: rt.route_dispatch_grad(rows, c.plan, weights=c.w, dx=out)[0],
                   lambda out: rt.route_dispatch_grad(rows, c.plan, weights=c.w, x=x, dx=out)[0]):
        big, out = within(torch.zeros_like(c.x))
        got = gather(out)
        assert got.data_ptr() == out.data_ptr()
        c.check_gathered(got)
        assert untouched(big, out)


def test_rows_transposed_and_broadcast_inputs(rt):
    c = Case(rt, 40, 3, 64, "f32")
    x = c.x.t().contiguous().t()
    c.check_spread(rt.route_dispatch(x, c.plan, weights=c.w))
    one = torch.ones((), device="cuda").expand(40, 64)      # what the backward pass of a sum hands over
    c.x = one.contiguous()
    c.check_spread(rt.route_combine_grad(one, c.plan, weights=c.w)[0])
    c.check_dots(rt.route_combine_grad(one, c.plan, weights=c.w, rows=c.rows)[1])


def test_rows_behind_the_output_stay(rt):
    c = Case(rt, 20, 2, 48, "f16")
    out = torch.full((60, 48), 5.0, dtype=torch.float16, device="cuda")
    rt.route_dispatch(c.x, c.plan, weights=c.w, out=out)
    c.check_spread(out[:40])
    assert bool((out[40:] == 5.0).all())


def test_dropped_rows_are_not_read(rt):
    """Rows that no choice takes may hold anything."""
    c = Case(rt, 50, 4, 72, "bf16", dropped=0.4)
    routed = int(c.plan.offsets[-1])
    c.rows[routed:] = float("nan")
    c.check_gathered(rt.route_combine(c.rows[:, :], c.plan, weights=c.w))
    dx, dw = rt.route_dispatch_grad(c.rows, c.plan, weights=c.w, x=c.x)
    c.check_gathered(dx)
    c.check_dots(dw)
    assert bool(torch.isfinite(rt.route_combine_grad(c.x, c.plan, weights=c.w, rows=c.rows)[1]).all())


def test_non_finite_values_stay_with_their_token(rt):
    c = Case(rt, 30, 3, 40, "f32", dropped=0.0)
    c.x[4, 5] = float("inf")
    c.x[9, 1] = float("nan")
    out = rt.route_dispatch(c.x, c.plan)
    bad = torch.zeros(90, dtype=torch.bool, device="cuda")
    bad[c.pos[[4, 9]].reshape(-1)] = True
    assert torch.equal(~torch.isfinite(out).all(1), bad)
    y = rt.route_combine(out, c.plan)
    assert torch.equal(torch.nonzero(~torch.isfinite(y)).cpu(), torch.tensor([[4, 5], [9, 1]]))


def test_plain_arithmetic_is_the_definition(rt):
    """fp32 rows: the sums are fused multiply-adds in the order of the choices, nothing else."""
    c = Case(rt, 64, 5, 96, "f32", dropped=0.3)
    want = torch.zeros((64, 96), dtype=torch.float64, device="cuda")
    for j in range(5):
        t = c.taken[:, j]
        v = c.rows[c.pos[t, j]].double() * c.w[t, j, None].double()   # exact in 64 bits; the sum is rounded twice,
        want[t] = (want[t] + v).float().double()                       # which differs from once in about 2^-29 of cases
    got = rt.route_combine(c.rows, c.plan, weights=c.w)
    assert float((got.double() != want).double().mean()) < 1e-3


def test_gradients_against_differences(rt):
    """Directional derivatives of sum(c * combine(dispatch(x, v), w)); the function is linear in each argument, so a
    central difference has no error of its own.  fp32 bound: sums of dim * k * T terms, 2^-24 each, twice."""
    c = Case(rt, 24, 3, 40, "f32", dropped=0.25)
    v = torch.randn_like(c.w)
    up = torch.randn_like(c.x)

    def f(x, v, w):
        return rt.route_combine(rt.route_dispatch(x, c.plan, weights=v), c.plan, weights=w)

    rows = rt.route_dispatch(c.x, c.plan, weights=v)
    drows, dw = rt.route_combine_grad(up, c.plan, weights=c.w, rows=rows)
    dx, dv = rt.route_dispatch_grad(drows, c.plan, weights=v, x=c.x)
    size = float((c.x.abs().double().mean() * v.abs().double().max() * c.w.abs().double().max() * up.abs().double().max())) * 24 * 3 * 40
    for i, grad in enumerate((dx, dv, dw)):
        args = [c.x, v, c.w]
        d = torch.randn_like(args[i])
        hi, lo = list(args), list(args)
        hi[i], lo[i] = d, -d
        diff = float(((f(*hi).double() - f(*lo).double()) * up.double()).sum()) / 2
        want = float((grad.double() * d.double()).sum())
        assert abs(diff - want) <= 8 * U * 40 * size * float(d.abs().max())


@pytest.mark.parametrize("elem", ["bf16", "f32"])
def test_far_rows(rt, elem):
    """Row offsets beyond 32 bits, in elements and in bytes."""
    c = Case(rt, 5, 2, 64, elem, dropped=0.0)
    stride = (1 << 28) + 8          # 9 rows of it pass 2^31 elements
    room = torch.empty(10 * stride, dtype=c.ty, device="cuda")
    far = room.as_strided((10, 64), (stride, 1))
    far.copy_(c.rows)
    c.check_gathered(rt.route_combine(far, c.plan, weights=c.w))
    c.check_dots(rt.route_dispatch_grad(far, c.plan, weights=c.w, x=c.x)[1])
    c.check_spread(rt.route_dispatch(c.x, c.plan, weights=c.w, out=far))
    del room, far
    torch.cuda.empty_cache()


def test_bad_positions_are_dropped(rt):
    """A position outside the rows is a dropped choice, whatever a caller put there."""
    c = Case(rt, 16, 2, 32, "f32", dropped=0.0)
    pos = c.plan.position.clone()
    pos[3, 1], pos[7, 0], pos[9, 1] = 32, 1 << 30, -(1 << 31)
    plan = c.plan._replace(position=pos)
    c.taken = (pos >= 0) & (pos < 32)
    c.w64 = torch.where(c.taken, c.w64, torch.zeros_like(c.w64))
    c.check_gathered(rt.route_combine(c.rows, plan, weights=c.w))
    dx, dw = rt.route_dispatch_grad(c.rows, plan, weights=c.w, x=c.x)
    c.check_gathered(dx)
    c.check_dots(dw)


def test_rows_refuse(rt):
    c = Case(rt, 8, 2, 32, "f16")
    x, rows, w, p = c.x, c.rows, c.w, c.plan
    for call, error in (
            (lambda: rt.route_dispatch(x.cpu(), p), ValueError), (lambda: rt.route_dispatch(x[0], p), ValueError),
            (lambda: rt.route_dispatch(x[:7], p), ValueError), (lambda: rt.route_dispatch(x.double(), p), TypeError),
            (lambda: rt.route_dispatch(x, p, weights=w.half()), TypeError), (lambda: rt.route_dispatch(x, p, weights=w[:4]), ValueError),
            (lambda: rt.route_dispatch(x, p, out=rows[:15]), ValueError), (lambda: rt.route_dispatch(x, p, out=rows.float()), TypeError),
            (lambda: rt.route_dispatch(x, p, out=rows.t().contiguous().t()), ValueError),
            (lambda: rt.route_dispatch(x, p._replace(position=p.position.long())), TypeError),
            (lambda: rt.route_dispatch(x, p._replace(offsets=p.offsets.cpu())), ValueError),
            (lambda: rt.route_combine(rows[:15], p), ValueError), (lambda: rt.route_combine(rows[:, :0], p), ValueError),
            (lambda: rt.route_combine(rows, p, out=x[:, :16]), ValueError),
            (lambda: rt.route_combine(rows, p, out=x[:1].expand(8, 32)), ValueError),
            (lambda: rt.route_combine_grad(x, p, rows=rows.float()), TypeError),
            (lambda: rt.route_dispatch_grad(rows, p, x=x[:, :16]), ValueError),
            (lambda: rt.route_combine(list(rows), p), TypeError)):
        with pytest.raises(error):
            call()


# ---- streams, graphs -----------------------------------------------------------------------

def test_on_a_stream_of_their_own(rt):
    """Named by argument and as the current one; every tensor the calls make belongs to that stream."""
    c = Case(rt, 3000, 4, 256, "bf16")
    ids = torch.where(c.taken, torch.randint(0, 9, (3000, 4), device="cuda"), torch.full((), -1, device="cuda"))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for named in (True, False):
        for _ in range(5):
            with torch.cuda.stream(side if not named else torch.cuda.current_stream()):
                s = side.cuda_stream if named else None
                plan = rt.route_plan(ids[:, ::2], 9, stream=s)          # copied first: on the same stream
                out = rt.route_dispatch(c.x, plan, weights=c.w[:, ::2], stream=s)
                back = rt.route_combine(out, plan, stream=s)
            side.synchronize()
            p = rt.route_plan(ids[:, ::2].contiguous(), 9)
            o = rt.route_dispatch(c.x, p, weights=c.w[:, ::2].contiguous())
            assert torch.equal(plan.order, p.order) and torch.equal(out, o) and torch.equal(back, rt.route_combine(o, p))


def test_captured_and_replayed(rt):
    """The whole layer in one graph, replayed over other ids, rows and weights; a second graph beside it."""
    T, k, G, dim = 4096, 4, 16, 128
    x = torch.zeros((T, dim), device="cuda", dtype=torch.bfloat16)
    w = torch.zeros((T, k), device="cuda")
    ids = torch.zeros((T, k), device="cuda", dtype=torch.int64)

    def layer(x, w, ids):
        plan = rt.route_plan(ids, G)
        rows = rt.route_dispatch(x, plan)
        y = rt.route_combine(rows, plan, weights=w)
        drows, dw = rt.route_combine_grad(y, plan, weights=w, rows=rows)
        dx, _ = rt.route_dispatch_grad(drows, plan)
        return plan.position, y, dw, dx

    layer(x, w, ids)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = layer(x, w, ids)
        graphs.append((g, out))
    for i in range(4):
        x.copy_(torch.randn(T, dim, device="cuda"))
        w.copy_(torch.rand(T, k, device="cuda"))
        ids.copy_(torch.randint(-1, G, (T, k), device="cuda"))
        want = layer(x, w, ids)
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_behind_lookups_in_one_stream(rt):
    """Tokens' rows from the cache, routed, and looked up again from what the routing wrote: every kernel waits for the ones
    ahead of it, however they overlap."""
    N, dim, n = 4000, 64, 512
    table = torch.randn(N, dim).pin_memory()
    cache = rt.Cache(1, N, dim * 4, 0.9, max_batch=4096)
    cache.set_placement(rt.solve_placement("rep", 1, np.arange(N, dtype=np.uint32), None, 90.0))
    cache.build(0, 0, table.data_ptr())
    dev = table.cuda()
    keys = torch.randint(0, N, (n,), device="cuda")
    ids = torch.randint(0, 7, (n, 2), device="cuda")
    for _ in range(30):
        x = cache.lookup(0, keys).view(torch.float32)
        plan = rt.route_plan(ids, 7)
        y = rt.route_combine(rt.route_dispatch(x, plan), plan)
        again = cache.lookup(0, plan.order[:n] % N).view(torch.float32)     # keys that the plan has just written
        pooled = cache.lookup_pool(0, plan.order, bag_size=2)
        assert torch.equal(y, 2 * dev[keys])
        assert torch.equal(again, dev[plan.order[:n].long()])
        assert torch.equal(pooled, dev[plan.order.long()].view(n, 2, dim).sum(1))
        keys = plan.order[n:].long() % N
    out = torch.empty(n, dim, device="cuda")
    with pytest.raises(rt.UgcError):   # bf16 rows are routed, not pooled
        cache.lookup_pool_ptr(0, keys.data_ptr(), 8, n, 0, n, 1, 2, 0, out.data_ptr())
    cache.close()


def test_a_layer_under_autograd(rt):
    """Dispatch, experts and combine as a training step uses them, against the same layer in 64 bits.  Every value is
    sums of products of at most 7 factors: off by at most (terms + 8) * 2^-24 of what the layer gives for the magnitudes."""
    class Dispatch(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, plan):
            ctx.plan = plan
            return rt.route_dispatch(x, plan)

        @staticmethod
        def backward(ctx, g):
            return rt.route_dispatch_grad(g, ctx.plan)[0], None

    class Combine(torch.autograd.Function):
        @staticmethod
        def forward(ctx, rows, weights, plan):
            ctx.plan = plan
            ctx.save_for_backward(rows, weights)
            return rt.route_combine(rows, plan, weights=weights)

        @staticmethod
        def backward(ctx, g):
            rows, weights = ctx.saved_tensors
            return (*rt.route_combine_grad(g, ctx.plan, weights=weights, rows=rows), None)

    T, k, G, dim = 200, 3, 6, 72
    g = torch.Generator(device="cuda")
    g.manual_seed(11)
    ids = torch.randint(-1, G, (T, k), generator=g, device="cuda")
    plan = rt.route_plan(ids, G)
    routed = int(plan.offsets[-1])
    group = ids.reshape(-1)[plan.order[:routed].long()]
    x, w, expert, up = (torch.randn(*s, generator=g, device="cuda") for s in ((T, dim), (T, k), (G, dim), (T, dim)))

    def fused(x, w, expert):
        rows = Dispatch.apply(x, plan)
        out = torch.cat([rows[:routed] * expert[group], rows[routed:]])
        return Combine.apply(out, w, plan)

    def plain(x, w, expert):
        return sum(torch.where((ids[:, j] >= 0)[:, None], w[:, j, None] * (x * expert[ids[:, j].clamp(min=0)]), 0.0) for j in range(k))

    def gradients(layer, ty, change=lambda t: t):
        leaves = [change(t.to(ty)).detach().requires_grad_() for t in (x, w, expert)]
        y = layer(*leaves)
        y.backward(change(up.to(ty)))
        return [y.detach()] + [t.grad for t in leaves]

    got, want, size = gradients(fused, torch.float32), gradients(plain, torch.float64), gradients(plain, torch.float64, torch.abs)
    for a, b, m, terms in zip(got, want, size, (k, k, dim, T * k)):
        assert bool(((a.double() - b).abs() <= (terms + 8) * U * m).all())


def test_same_results_again(rt):
    c = Case(rt, 2000, 8, 1000, "f16")
    first = rt.route_dispatch_grad(c.rows, c.plan, weights=c.w, x=c.x)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, rt.route_dispatch_grad(c.rows, c.plan, weights=c.w, x=c.x)))


def test_token_results_do_not_depend_on_the_batch(rt):
    """One group: the plan is the identity, so the first tokens of a large batch are a small batch."""
    ids = torch.zeros((3000, 4), dtype=torch.int64, device="cuda")
    x, rows, w = torch.randn(3000, 768, device="cuda"), torch.randn(12000, 768, device="cuda"), torch.randn(3000, 4, device="cuda")
    whole, few = rt.route_plan(ids, 1), rt.route_plan(ids[:7], 1)
    for a, b in zip(rt.route_dispatch_grad(rows, whole, weights=w, x=x), rt.route_dispatch_grad(rows[:28], few, weights=w[:7], x=x[:7])):
        assert torch.equal(a[:7], b)
    for (a, n), (b, _) in zip(zip(rt.route_combine_grad(x, whole, weights=w, rows=rows), (28, 7)),
                              zip(rt.route_combine_grad(x[:7], few, weights=w[:7], rows=rows[:28]), (28, 7))):
        assert torch.equal(a[:n], b)
    assert torch.equal(rt.route_combine(rows, whole, weights=w)[:7], rt.route_combine(rows[:28], few, weights=w[:7]))


@pytest.mark.skipif(not torch.cuda.is_available() or torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_on_another_device(rt):
    with torch.cuda.device(0):
        ids = torch.randint(0, 9, (100, 3), device="cuda:1")
        x = torch.randn(100, 64, device="cuda:1")
        plan = rt.route_plan(ids, 9)
        y = rt.route_combine(rt.route_dispatch(x, plan), plan)
        assert torch.cuda.current_device() == 0
        assert torch.allclose(y, 3 * x)
        with pytest.raises(ValueError):
            rt.route_dispatch(x.to("cuda:0"), plan)
