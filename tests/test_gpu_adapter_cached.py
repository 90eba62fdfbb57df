"""Adapters as rows of a cached table, looked up by request: more requests, and more adapters, than a plan has groups."""
import numpy as np
import pytest

from tests.test_gpu_adapter import formula

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.mark.parametrize("n_requests,T", [(1, 1), (24, 3000), (1024, 1024), (1500, 4000)])
def test_every_request_gets_its_adapter(built_lib, n_requests, T):
    from ugache_b200 import runtime as rt
    A, r, H, N = 2000, 8, 64, 72
    per = r * (H + N)
    g = torch.Generator()
    g.manual_seed(n_requests)
    table = (torch.randn((A, per), generator=g) / 8).to(torch.bfloat16).pin_memory()
    cache = rt.Cache(1, A, per * 2, 0.4, max_batch=4096)
    cache.set_placement(rt.solve_placement("rep", 1, np.arange(A, dtype=np.uint32), None, 40.0))
    cache.build(0, 0, table.data_ptr())
    names = torch.randperm(A, generator=g)[:n_requests].cuda()          # all distinct
    if n_requests > 30:
        names[::7] = names[0]                                           # some the same,
        names[3::50] = A + 5                                            # some of no adapter
    of_token = torch.sort(torch.randint(0, n_requests, (T,), generator=g)).values.cuda()
    x, base = torch.randn((T, H), device="cuda").bfloat16(), torch.randn((T, N), device="cuda").bfloat16()
    y = base.clone()
    for first in range(0, n_requests, 1024):
        part = names[first:first + 1024]
        n = part.numel()
        rows, _, inverse, _ = cache.lookup_unique(0, part)
        rows = rows.view(torch.bfloat16)
        down, up = rows[:, :r * H].view(n, r, H), rows[:, r * H:].view(n, N, r)
        here = of_token - first
        ids = torch.where((here >= 0) & (here < n), inverse[here.clamp(0, n - 1)], -1)
        y = rt.adapter_add(y, x, down, up, rt.route_plan(ids, n), out=y)
    dev = table.cuda()
    ids = names[of_token]
    ids = torch.where(ids < A, ids, torch.full_like(ids, -1))
    if n_requests == 1500:
        assert ids.unique().numel() > 1024
    want, slack = formula(base, x, dev[:, :r * H].view(A, r, H), dev[:, r * H:].view(A, N, r), ids, None)
    assert bool(((y.double() - want).abs() <= slack).all())
    assert torch.equal(y[ids < 0], base[ids < 0])
    cache.close()
