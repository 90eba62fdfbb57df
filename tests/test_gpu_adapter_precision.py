"""What the rank products of 16-bit adapters keep between the two products: 24 significand bits, as an fp32 sum has.

Inputs are chosen so that both sums are exact in fp32 (whole numbers below 2^24, or one term a sum), so that what is
left is the way the rank products are handed over and the result's one rounding."""
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def rt(built_lib):
    from ugache_b200 import runtime
    return runtime


def run(rt, base, x, down, up, ids, **kw):
    return rt.adapter_add(base, x, down, up, rt.route_plan(ids, down.shape[0]), **kw)


@pytest.mark.parametrize("rank", [8, 16, 24, 64, 72, 128])
@pytest.mark.parametrize("T", [50, 6000])   # single tokens, prompts
def test_whole_numbers_are_exact(rt, rank, T):
    """Rank products of 18 to 20 bits; `base` takes away all that the result's type could hide."""
    g = torch.Generator(device="cuda")
    g.manual_seed(T + rank)
    G, dim, out_dim = 3, 64, 136

    def whole(low, high, *size):
        return torch.randint(low, high + 1, size, generator=g, device="cuda")

    x, down = whole(0, 127, T, dim), whole(0, 127, G, rank, dim)       # sums up to 64 * 127^2 < 2^20
    up = torch.zeros((G, out_dim, rank), dtype=torch.int64, device="cuda")
    for _ in range(4):                                                 # at most four ranks an output, each at most 3 in the end
        up.scatter_(2, whole(0, rank - 1, G, out_dim, 1), whole(-1, 1, G, out_dim, 1))
    ids = whole(0, G - 1, T)
    delta = torch.einsum("tr,tnr->tn", torch.einsum("td,trd->tr", x.double(), down[ids].double()), up[ids].double())
    assert float(delta.abs().max()) < 2 ** 23
    ty = torch.bfloat16
    base = (-delta).to(ty)
    got = run(rt, base, x.to(ty), down.to(ty), up.to(ty), ids)
    want = (base.double() + delta).to(ty)
    assert bool((want != 0).any()) and torch.equal(got, want)


@pytest.mark.parametrize("elem", sorted(TYPES))
@pytest.mark.parametrize("rank", [8, 16, 24, 64, 128])
@pytest.mark.parametrize("T", [50, 6000])
def test_ranks_of_far_magnitudes(rt, rank, T, elem):
    """Rank product r of a token is m * 2^-e(r), m of up to 11 bits in [1, 2) and e from 0 to 20; output n takes one rank
    alone and scales it back.  Two roundings: a rank product's to 24 bits (2^-23 of it, whatever cuts them off; or 2^-38 of the
    token's largest, 2, where the type ends below it) and the result's, by eps / 2."""
    g = torch.Generator(device="cuda")
    g.manual_seed(T + 3 * rank)
    G, ty = 2, TYPES[elem]
    dim = out_dim = max(rank, 16)
    e = (torch.arange(rank, device="cuda") * 7) % 21
    m = (1 + torch.rand((T, dim), generator=g, device="cuda")).to(ty)
    down = torch.zeros((G, rank, dim), device="cuda")
    up = torch.zeros((G, out_dim, rank), device="cuda")
    r = torch.arange(rank, device="cuda")
    down[:, r, r] = 2.0 ** -e.float()
    n = torch.arange(out_dim, device="cuda")
    up[:, n, n % rank] = (2.0 ** e[n % rank].float()).clamp(max=2.0 ** 15)
    ids = torch.randint(0, G, (T,), generator=g, device="cuda")
    assert torch.equal(down.to(ty).float(), down) and torch.equal(up.to(ty).float(), up)
    got = run(rt, torch.zeros((T, out_dim), dtype=ty, device="cuda"), m, down.to(ty), up.to(ty), ids)
    inner = torch.zeros((T, rank), dtype=torch.float64, device="cuda")
    inner[:] = m[:, :rank].double() * 2.0 ** -e.double()
    want = inner @ up[0].double().t()
    off = (2.0 ** -23 * inner + 2.0 ** -38 * 2) @ up[0].double().t()
    assert bool(((got.double() - want).abs() <= off + torch.finfo(ty).eps / 2 * (want + off)).all())


@pytest.mark.parametrize("elem", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("rank", [1, 4, 8, 12, 16, 24, 40, 72, 128])
@pytest.mark.parametrize("T", [50, 6000])
def test_an_infinite_input_is_an_infinite_result(rt, rank, T, elem):
    """All factors of a token's infinite element are positive, and so is every product that `up` makes of an output's
    sign: the formula has infinities of one sign in each output, and no NaN, whatever the rank is padded to."""
    g = torch.Generator(device="cuda")
    g.manual_seed(rank)
    ty = torch.float32 if elem == "f32" else TYPES[elem]
    x, base = torch.rand((T, 64), generator=g, device="cuda"), torch.randn((T, 72), generator=g, device="cuda")
    down, up = 0.5 + torch.rand((2, rank, 64), generator=g, device="cuda"), 0.5 + torch.rand((2, 72, rank), generator=g, device="cuda")
    up[:, 1::2] *= -1
    x[3, 10], x[T - 1, 63] = float("inf"), float("-inf")
    ids = torch.randint(0, 2, (T,), generator=g, device="cuda")
    got = run(rt, base.to(ty), x.to(ty), down.to(ty), up.to(ty), ids)
    sign = torch.ones(72, device="cuda")
    sign[1::2] = -1
    inf = float("inf")
    assert torch.equal(got[3].float(), inf * sign) and torch.equal(got[T - 1].float(), -inf * sign)
    rest = torch.ones(T, dtype=torch.bool, device="cuda")
    rest[3], rest[T - 1] = False, False
    assert bool(torch.isfinite(got[rest]).all())


@pytest.mark.parametrize("elem", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("T,rank", [(50, 16), (50, 3), (6000, 16)])
def test_tokens_without_an_adapter_keep_their_bits(rt, T, rank, elem):
    """Negative zeros, subnormals and infinities among them."""
    ty = torch.float32 if elem == "f32" else TYPES[elem]
    base = torch.randn(T, 88, device="cuda").to(ty)
    base[:, ::4], base[:, 1::8] = -0.0, float("-inf")
    base[:, 2::8] = torch.finfo(ty).smallest_normal / 4
    ids = torch.randint(0, 3, (T,), device="cuda")
    ids[::2] = -1
    x, down, up = torch.randn(T, 48, device="cuda").to(ty), torch.randn(3, rank, 48, device="cuda").to(ty), torch.randn(3, 88, rank, device="cuda").to(ty)
    got = run(rt, base, x, down, up, ids)
    bits = torch.int32 if elem == "f32" else torch.int16
    assert torch.equal(got[::2].view(bits), base[::2].view(bits))


@pytest.mark.parametrize("rank", [16, 64, 128])
@pytest.mark.parametrize("T", [50, 6000])
def test_long_sums_of_one_sign(rt, T, rank):
    """Every factor is positive, so that whatever a sum cuts off adds up; `up` hands the rank products out one by one and
    `base` takes away what the result's type could hide.  Bound, of the sum: 2^-23 for each instruction of a matrix unit's
    own sum (prompts: 8; single tokens: 4, at rank 16 the 32 that a warp has of a row), 2^-24 for each fp32 addition behind it
    (prompts: 128 steps and at most 8 parts; single tokens: the sums of a warp, and those of 16 warps and 8 CTAs at most),
    2^-23 for each of the three terms and for the scale."""
    g = torch.Generator(device="cuda")
    g.manual_seed(T + rank)
    G, dim = 2, 16384
    x, down = torch.rand((T, dim), generator=g, device="cuda").half(), (torch.rand((G, rank, dim), generator=g, device="cuda") / 64).half()
    up = torch.eye(rank, device="cuda").expand(G, rank, rank).contiguous().half()
    ids = torch.randint(0, G, (T,), generator=g, device="cuda")
    delta = torch.stack([x.double() @ down[a].double().t() for a in range(G)])[ids, torch.arange(T, device="cuda")]
    base = (-delta).half()
    got = run(rt, base, x, down, up, ids)
    want = base.double() + delta
    own, added = (8, 136) if T > 1000 else (32, 24) if rank == 16 else (4, {64: 16, 128: 32}[rank] + 24)
    off = (own * 2.0 ** -23 + added * 2.0 ** -24 + 4 * 2.0 ** -23) * delta
    assert bool(((got.double() - want).abs() <= off + torch.finfo(torch.float16).eps / 2 * (want.abs() + off) + 2.0 ** -25).all())
