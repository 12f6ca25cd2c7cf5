"""A host thread's first use of the device may be one of the library's calls:
its tensor maps need a current context, which the CUDA runtime makes only at
the thread's first call that works on the device."""
import threading

import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def env():
    import torch
    import whirlwind_trt_plugins_b200 as ww
    return torch, ww


def _in_thread(fn):
    got = []

    def work():
        try:
            got.append(fn())
        except Exception as e:  # noqa: BLE001 -- the finding
            got.append(e)

    t = threading.Thread(target=work)
    t.start()
    t.join()
    if isinstance(got[0], Exception):
        raise got[0]
    return got[0]


@pytest.mark.parametrize("Lq", [2, 90])
def test_attention(env, Lq):
    torch, ww = env
    q = torch.randn((1, Lq, 2, 64), device="cuda").half()
    k = torch.randn((1, 100, 2, 64), device="cuda").half()
    out, lse = ww.cross_attention(q, k, k, return_lse=True)
    grads = ww.cross_attention_backward(q, q, k, k, out, lse)
    torch.cuda.synchronize()
    again, _ = _in_thread(lambda: ww.cross_attention(q, k, k, return_lse=True))
    more = _in_thread(lambda: ww.cross_attention_backward(q, q, k, k, out, lse))
    torch.cuda.synchronize()
    assert torch.equal(out, again)
    assert all(torch.equal(x, y) for x, y in zip(grads[:3], more[:3]))


def test_fused_stem(env):
    torch, ww = env
    left, right = (torch.randn((1, 32, 16, 64), device="cuda").half() for _ in range(2))
    w, b = torch.randn((8, 32, 3, 3, 3), device="cuda").half() * 0.05, torch.zeros(8, device="cuda").half()
    call = lambda: ww.corr_cost_stem3d(left, right, w, b, 16, num_groups=32)  # noqa: E731
    want = call()
    torch.cuda.synchronize()
    got = _in_thread(call)
    torch.cuda.synchronize()
    assert torch.equal(want, got)
