"""Host threads that call the same form with different sizes at the same time."""
import threading

import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def env():
    import torch
    import whirlwind_trt_plugins_b200 as ww
    return torch, ww


@pytest.mark.parametrize("form", ["tiles", "token", "gradient"])
def test_two_threads(env, form):
    """One call keeps a long range of bias positions in shared memory, the other a short one: each
    thread repeats its own call through the C ABI, where the threads run side by side."""
    torch, ww = env
    from whirlwind_trt_plugins_b200 import attention as at
    Lq, H, D = 2 if form == "token" else 90, 2, 64
    name = "ww_cross_attention_backward" if form == "gradient" else "ww_cross_attention"
    fn, need = getattr(ww.lib(), name), getattr(ww.lib(), name + "_workspace")
    hold = []

    def call(Lk, distance):
        g = torch.Generator(device="cuda").manual_seed(Lk)
        q = torch.randn((1, Lq, H, D), generator=g, device="cuda").half()
        k = torch.randn((1, Lk, H, D), generator=g, device="cuda").half()
        table = torch.randn((H, 16), generator=g, device="cuda").half()
        out, lse = ww.cross_attention(q, k, k, bias_table=table, max_distance=distance, return_lse=True)
        if form == "gradient":
            want = ww.cross_attention_backward(q, q, k, k, out, lse, bias_table=table, max_distance=distance)
            into = [torch.empty_like(x) for x in want]
            ptrs = [q, k, k, out, lse, None, None, table, q, *into]
        else:
            want = [out, lse]
            into = [torch.empty_like(x) for x in want]
            ptrs = [q, k, k, *into, None, None, table] + [None] * 5
        st = [q.stride()[:3], k.stride()[:3], k.stride()[:3], q.stride()[:3]]
        a = at._ATTN.pack(*[at._ptr(x) for x in ptrs], 0, 0, *[s for x in st for s in x], 1, 1, Lq, Lk, H, H, D, 16,
                          distance, 1, 0, D ** -0.5)
        n = need(a)
        ws = torch.empty(max(n, 1), dtype=torch.uint8, device="cuda")
        a = a[:at._ATTN_WS] + at._WS.pack(ws.data_ptr() if n else 0, n) + a[at._ATTN_WS + 16:]
        hold.extend([ptrs, ws])
        return a, want, into

    calls = [call(2500, 1024), call(40, 16)]
    torch.cuda.synchronize()
    wrong = []
    start = threading.Barrier(2)

    def work(a, want, into):
        try:
            torch.cuda.synchronize()
            stream = torch.cuda.Stream()
            start.wait(30)
            for i in range(20000):
                status = fn(a, stream.cuda_stream)
                if status != 0:
                    wrong.append(f"call {i}: status {status}")
                    break
            stream.synchronize()
            if not all(torch.equal(x, y) for x, y in zip(into, want)):
                wrong.append("results differ")
        except Exception as e:  # noqa: BLE001 -- whatever ended the thread is the finding
            wrong.append(repr(e))

    threads = [threading.Thread(target=work, args=c) for c in calls]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert wrong == []
    assert ww.device_error() == 0
