"""The gradient of ww_cross_attention through the C ABI with a workspace that
holds anything: results do not depend on it, and without queries the gradients
of keys and values are zeros."""
import pytest

pytestmark = pytest.mark.gpu

TYPES = {"f16": 1, "bf16": 7}


@pytest.fixture(scope="module")
def env():
    import torch
    import whirlwind_trt_plugins_b200 as ww
    return torch, ww


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("byte", [0x00, 0x7E, 0x7F, 0xFF])
@pytest.mark.parametrize("buckets", [0, 8])
def test_no_queries(env, dt, byte, buckets):
    torch, ww = env
    from whirlwind_trt_plugins_b200 import attention as at
    t = torch.float16 if dt == "f16" else torch.bfloat16
    B, Lk, Hq, Hk, D = 2, 130, 4, 2, 64
    k, v = (torch.randn((B, Lk, Hk, D), device="cuda").to(t) for _ in range(2))
    dk, dv = torch.full_like(k, float("nan")), torch.full_like(v, float("nan"))
    table = torch.randn((Hq, 8), device="cuda").to(t)
    dtable = torch.full_like(table, float("nan"))
    st = k.stride()[:3]
    a = at._ATTN.pack(0, k.data_ptr(), v.data_ptr(), 0, 0, 0, 0, table.data_ptr() if buckets else 0, 0, 0, dk.data_ptr(),
                      dv.data_ptr(), dtable.data_ptr() if buckets else 0, 0, 0, 0, 0, 0, *st, *st, 0, 0, 0,
                      TYPES[dt], B, 0, Lk, Hq, Hk, D, buckets, 32, 1, 0, 0.125)
    n = ww.lib().ww_cross_attention_backward_workspace(a)
    ws = torch.full((max(n, 1),), byte, dtype=torch.uint8, device="cuda")
    a = a[:at._ATTN_WS] + at._WS.pack(ws.data_ptr(), n) + a[at._ATTN_WS + 16:]
    assert ww.lib().ww_cross_attention_backward(a, torch.cuda.current_stream().cuda_stream) == 0
    assert bool((dk == 0).all()) and bool((dv == 0).all())
    assert not buckets or bool((dtable == 0).all())
    assert ww.device_error() == 0


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("shape", [(3, 90, 130, 4, 2, 64), (40, 160, 160, 3, 3, 32), (1, 600, 700, 4, 4, 128)])
def test_same_bits_over_any_workspace(env, dt, shape):
    """A workspace of another call's size, place and leavings, calls one after the other without a
    gap: every call gives the bits of the first."""
    torch, ww = env
    from whirlwind_trt_plugins_b200 import attention as at
    t = torch.float16 if dt == "f16" else torch.bfloat16
    B, Lq, Lk, Hq, Hk, D = shape
    q, dout = (torch.randn((B, Lq, Hq, D), device="cuda").to(t) for _ in range(2))
    k, v = (torch.randn((B, Lk, Hk, D), device="cuda").to(t) for _ in range(2))
    table = torch.randn((Hq, 16), device="cuda").to(t)
    out, lse = ww.cross_attention(q, k, v, bias_table=table, return_lse=True)
    want = ww.cross_attention_backward(dout, q, k, v, out, lse, bias_table=table)
    sq, sk = q.stride()[:3], k.stride()[:3]

    def packed(into):
        return at._ATTN.pack(*[at._ptr(x) for x in (q, k, v, out, lse, None, None, table, dout, *into)], 0, 0, *sq, *sk,
                             *sk, *sq, TYPES[dt], B, Lq, Lk, Hq, Hk, D, 16, 128, 1, 0, D ** -0.5)

    n = ww.lib().ww_cross_attention_backward_workspace(packed(want))
    got = []
    for byte in (0x00, 0x01, 0x7F, 0xFF):
        ws = torch.full((n + 64,), byte, dtype=torch.uint8, device="cuda")
        for shift in (0, 16, 64):
            into = [torch.full_like(x, float("nan")) for x in want]
            a = packed(into)
            a = a[:at._ATTN_WS] + at._WS.pack(ws.data_ptr() + shift, n) + a[at._ATTN_WS + 16:]
            assert ww.lib().ww_cross_attention_backward(a, torch.cuda.current_stream().cuda_stream) == 0
            got.append((into, ws))
    for into, _ in got:
        assert all(torch.equal(x, y) for x, y in zip(into, want))
    assert ww.device_error() == 0
