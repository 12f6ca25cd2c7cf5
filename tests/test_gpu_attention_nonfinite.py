"""Non-finite values in valid keys: a NaN or +inf score makes its row NaN, a
-inf score is a weight of exactly 0, whatever column of a tile it stands in and
whichever form of the operator runs; and the accuracy of the exponentials that
are computed by a polynomial."""
import math

import pytest
from test_gpu_attention import E, TINY, U, _attention_ref, _randn, _type, _within

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def env():
    import torch
    import whirlwind_trt_plugins_b200 as ww
    return torch, ww


# (Lq, Lk, Hq, Hk, D): tiles of one query block at each head width, of two, and single tokens
FORMS = [(130, 192, 2, 2, 32), (130, 192, 2, 1, 64), (130, 128, 1, 1, 128), (2100, 128, 1, 1, 64), (3, 320, 4, 2, 64),
         (1, 128, 8, 1, 128)]
FIRST = 72  # items 0 to 7 have their value in key FIRST + item, item 8 has none


def _inputs(torch, form, dt, lq=None):
    Lq, Lk, Hq, Hk, D = form
    Lq = lq or Lq
    t = _type(torch, dt)
    a = {"q": _randn(torch, (9, Lq, Hq, D), 1, t), "k": _randn(torch, (9, Lk, Hk, D), 2, t),
         "v": _randn(torch, (9, Lk, Hk, D), 3, t), "dout": _randn(torch, (9, Lq, Hq, D), 4, t)}
    return a, torch.ones((9, Lk), dtype=torch.bool, device="cuda")


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("bias", [False, True])
def test_nan_in_a_valid_key(env, form, dt, bias):
    torch, ww = env
    a, keep = _inputs(torch, form, dt)
    for b in range(8):
        a["k"][b, FIRST + b, :, b] = math.nan
    kw = {"bias_table": _randn(torch, (form[2], 8), 5, a["q"].dtype), "max_distance": 16} if bias else {}
    out, lse = ww.cross_attention(a["q"], a["k"], a["v"], return_lse=True, **kw)
    grads = ww.cross_attention_backward(a["dout"], a["q"], a["k"], a["v"], out, lse, **kw)
    assert bool(out[:8].isnan().all()) and bool(lse[:8].isnan().all())
    for x in grads[:3]:
        assert bool(x[:8].isnan().all()) and bool(x[8].isfinite().all())
    assert bool(out[8].isfinite().all())


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("dt", ["f16", "bf16"])
def test_infinite_scores(env, form, dt):
    """Channel 0 of one key is +inf: rows with q0 > 0 have a score of +inf and are NaN, rows with
    q0 < 0 one of -inf and are what they are without that key."""
    torch, ww = env
    a, keep = _inputs(torch, form, dt)
    a["q"][..., 0] = torch.where(a["q"][..., 0] < 0, -1.0, 1.0)
    for b in range(8):
        a["k"][b, FIRST + b, :, 0] = math.inf
        keep[b, FIRST + b] = False
    scale = 1 / math.sqrt(form[4])
    out, lse = ww.cross_attention(a["q"], a["k"], a["v"], return_lse=True)
    ref, bounds = _attention_ref(torch, ww, a, {}, keep, scale)
    bound = bounds(U[dt], TINY[dt])["out"]
    nan = a["q"][..., 0] > 0
    nan[8] = False
    assert bool(out[nan].isnan().all()) and not bool(lse.transpose(1, 2)[nan].isfinite().any())
    _within(out[~nan], ref["out"][~nan], bound[~nan], "out")
    l, want = lse.transpose(1, 2)[~nan].double(), ref["lse"].transpose(1, 2)[~nan]
    assert bool(((l - want).abs() <= E * (1 + want.abs())).all())


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("dt", ["f16", "bf16"])
def test_scores_of_minus_infinity(env, form, dt):
    """All queries have q0 < 0: the key at +inf has weight 0, and so have its gradients; where every
    key is at +inf a row is empty."""
    torch, ww = env
    a, keep = _inputs(torch, form, dt, 2112 if form[0] > 2048 else 128)
    a["q"][..., 0] = -1.0
    for b in range(8):
        a["k"][b, FIRST + b, :, 0] = math.inf
        keep[b, FIRST + b] = False
    scale = 1 / math.sqrt(form[4])
    out, lse = ww.cross_attention(a["q"], a["k"], a["v"], return_lse=True)
    dq, dk, dv, _ = ww.cross_attention_backward(a["dout"], a["q"], a["k"], a["v"], out, lse)
    ref, bounds = _attention_ref(torch, ww, a, {}, keep, scale)
    bound = bounds(U[dt], TINY[dt])
    for n, x in (("out", out), ("dk", dk), ("dv", dv)):
        _within(x, ref[n], bound[n], n)
    _within(dq[..., 1:], ref["dq"][..., 1:], bound["dq"][..., 1:], "dq")  # channel 0: 0 times inf
    assert bool((dk[~keep] == 0).all()) and bool((dv[~keep] == 0).all())
    for lq in (1, 128, a["q"].shape[1]):
        empty = ww.cross_attention(a["q"][:, :lq], a["k"].clone().index_fill_(3, torch.tensor([0], device="cuda"), math.inf),
                                   a["v"], return_lse=True)
        assert bool((empty[0] == 0).all()) and bool((empty[1] == -math.inf).all())


@pytest.mark.parametrize("column", range(8))
@pytest.mark.parametrize("D,Lq", [(32, 600), (64, 600), (128, 600), (64, 2300)])
def test_exponential(env, column, D, Lq):
    """lse = log(1 + e^x) from two keys that count, x in [-3, 0]: an exponential's relative error is
    2.6e-6 by the polynomial (2^-22 by the unit), plus that of its fp32 argument."""
    torch, ww = env
    q = torch.zeros((1, Lq, 1, D), device="cuda", dtype=torch.float16)
    q[0, :, 0, 0] = -torch.linspace(0, 3, Lq, device="cuda").half()
    q[..., 1] = 1
    k = torch.zeros((1, 64, 1, D), device="cuda", dtype=torch.float16)
    k[..., 1] = -1000
    k[0, 48 + column, 0, :2] = torch.tensor([1.0, 0.0], device="cuda")
    k[0, 20, 0, 1] = 0
    _, lse = ww.cross_attention(q, k, k, 1.0, return_lse=True)
    x = q[0, :, 0, 0].double()
    p = x.exp()
    # argument: a rounded product and sum of up to 3 log2(e) < 8 and log2(e) itself; lse: log2, sum and product
    bound = p / (1 + p) * (2.6e-6 + 3 * 8 * 2.0 ** -24) + 3 * 2.0 ** -23
    assert bool(((lse[0, 0].double() - torch.log1p(p)).abs() <= bound).all())
