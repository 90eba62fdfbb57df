"""The count of waits that ran out, through the Python face."""
import ctypes as C

import pytest


@pytest.fixture(scope="module")
def rt(built_lib):
    from ugache_b200 import runtime
    return runtime


def test_the_count_is_read_and_errors_are_raised(rt, monkeypatch):
    """Against a stand-in for the library: what the GPU counted arrives, what the call refuses is an exception."""
    asked = []

    class Lib:
        def ugc_adapter_stalled(self, device, count):
            asked.append(device)
            C.cast(count, C.POINTER(C.c_uint32))[0] = 3
            return 0 if device < 2 else 2

        def ugc_last_error(self):
            return b"no such device"

    monkeypatch.setattr(rt._lib, "lib", lambda: Lib())
    assert rt.adapter_stalled() == 3 and rt.adapter_stalled(1) == 3
    with pytest.raises(rt.UgcError):
        rt.adapter_stalled(2)
    assert asked == [0, 1, 2]


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 40, 900])
def test_no_wait_runs_out(rt, T):
    torch = pytest.importorskip("torch")
    base, x = torch.randn(T, 4096, device="cuda").bfloat16(), torch.randn(T, 512, device="cuda").bfloat16()
    down, up = torch.randn(3, 64, 512, device="cuda").bfloat16(), torch.randn(3, 4096, 64, device="cuda").bfloat16()
    rt.adapter_add(base, x, down, up, rt.route_plan(torch.randint(-1, 3, (T,), device="cuda"), 3))
    assert rt.adapter_stalled() == 0
