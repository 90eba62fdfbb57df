"""Calls from several host threads at once, each on a stream of its own: they share nothing, on the host neither."""
import threading

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.fixture(scope="module")
def rt(built_lib):
    from ugache_b200 import runtime
    return runtime


def together(calls, rounds):
    """Every call in a thread, over and over; its first result came alone."""
    want = [call() for call in calls]
    torch.cuda.synchronize()
    failed, start = [], threading.Barrier(len(calls))

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                start.wait()
                for _ in range(rounds):
                    got = calls[i]()
                if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                    failed.append("call %d gave something else" % i)
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # handed on: an exception would end in the thread
            failed.append("call %d: %r" % (i, e))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(calls))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed


def test_plans_of_several_sizes(rt):
    """One kernel whose launches want 43 to 74 KB of shared memory."""
    torch.manual_seed(5)
    sizes = [(1024, 1024), (1024, 600), (1000, 800), (900, 700), (1024, 50)]
    ids = [torch.randint(0, G, (n,), device="cuda") for n, G in sizes]
    together([lambda i=i, G=G: rt.route_plan(i, G) for i, (_, G) in zip(ids, sizes)], 20000)


@pytest.mark.parametrize("elem", [torch.bfloat16, torch.float16])
def test_adapters_of_several_batches(rt, elem):
    """One kernel whose launches want 54 to 200 KB of shared memory."""
    torch.manual_seed(6)
    G, rank, dim = 64, 16, 256
    down, up = torch.randn(G, rank, dim, device="cuda").to(elem), torch.randn(G, 320, rank, device="cuda").to(elem)
    calls = []
    for T in (1, 20, 60, 200, 1, 900):
        x, base = torch.randn(T, dim, device="cuda").to(elem), torch.randn(T, 320, device="cuda").to(elem)
        plan = rt.route_plan(torch.randint(-1, G, (T,), device="cuda"), G)
        calls.append(lambda x=x, base=base, plan=plan: (rt.adapter_add(base, x, down, up, plan),))
    together(calls, 3000)
