"""fp16 gradients whose scores' gradients dS are large or far apart: dS is rounded
to fp16 under a power of two that keeps its largest possible value in range."""
import math

import pytest
from test_gpu_attention import TINY, U, _attention_ref, _randn, _within

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def env():
    import torch
    import whirlwind_trt_plugins_b200 as ww
    return torch, ww


def _check(torch, ww, a, kw=None, keep=None, dt="f16"):
    """Every batch item against 64 bits.  |dS| <= M = 2 max|dO row| max|v row| over its valid keys;
    dS is kept with 2^14 <= (its factor) M, so half of fp16's smallest step, 2^-25, is 2^-39 M of dS."""
    kw = kw or {}
    B, Lk, D = a["q"].shape[0], a["k"].shape[1], a["q"].shape[3]
    if keep is None:
        keep = torch.ones((B, Lk), dtype=torch.bool, device="cuda")
    scale = 1 / math.sqrt(D)
    out, lse = ww.cross_attention(a["q"], a["k"], a["v"], return_lse=True, **kw)
    dq, dk, dv, dtable = ww.cross_attention_backward(a["dout"], a["q"], a["k"], a["v"], out, lse, **kw)
    got = {"out": out, "dq": dq, "dk": dk, "dv": dv}
    total = bound_of_table = 0
    full = {"bidirectional": True, "q_offset": 0, **{n: x for n, x in kw.items() if n not in ("key_mask", "k_lens")}}
    for b in range(B):
        one = {n: x[b:b + 1] for n, x in a.items()}
        ref, bounds = _attention_ref(torch, ww, one, full if "bias_table" in kw else {}, keep[b:b + 1], scale)
        v = a["v"][b][keep[b]].double()
        M = 2 * a["dout"][b].double().norm(dim=-1).max().item() * (v.norm(dim=-1).max().item() if v.numel() else 0)
        bound = bounds(U[dt], max(TINY[dt], 2.0 ** -39 * M / 2))
        for n, x in got.items():
            _within(x[b:b + 1], ref[n], bound[n], f"{n} of item {b}")
        if dtable is not None:
            total, bound_of_table = total + ref["dtable"], bound_of_table + bound["dtable"]
    if dtable is not None:
        _within(dtable, total, bound_of_table, "dtable")


def test_two_opposed_keys(env):
    """V = +32 and -32 at equal scores: dS = +-1024 with dO = 1."""
    torch, ww = env
    for D in (32, 64, 128):
        q = _randn(torch, (2, 70, 2, D), 1, torch.float16)
        k = _randn(torch, (2, 1, 2, D), 2, torch.float16).expand(2, 2, 2, D).contiguous()
        v = torch.full_like(k, 32)
        v[:, 1] = -32
        _check(torch, ww, {"q": q, "k": k, "v": v, "dout": torch.ones_like(q)})


@pytest.mark.parametrize("shape", [(2, 70, 2, 2, 2, 64), (3, 130, 200, 4, 2, 32), (2, 65, 129, 2, 2, 128), (2, 3, 500, 4, 1, 64)])
@pytest.mark.parametrize("size", [16.0, 32.0, 1000.0, 30000.0])
@pytest.mark.parametrize("kind", ["random", "constant", "channel"])
@pytest.mark.parametrize("bias", [False, True])
def test_large_values(env, shape, size, kind, bias):
    """V of this size: random, of one sign along each key's channels, or in one channel only; masked
    places hold what would be larger still."""
    torch, ww = env
    B, Lq, Lk, Hq, Hk, D = shape
    q, k = _randn(torch, (B, Lq, Hq, D), 1, torch.float16), _randn(torch, (B, Lk, Hk, D), 2, torch.float16)
    v = _randn(torch, (B, Lk, Hk, D), 3, torch.float16)
    sign = torch.where(_randn(torch, (B, Lk, Hk, 1), 4, torch.float32) < 0, -size, size)
    if kind == "random":
        v = (v.float() * size).clamp(-60000, 60000).half()
    elif kind == "constant":
        v = sign.expand(B, Lk, Hk, D).half().contiguous()
    else:
        v[..., D // 2] = sign[..., 0].half()
    # the true gradients stay far inside fp16's range
    dout = (_randn(torch, (B, Lq, Hq, D), 5, torch.float32) * (8 / size) if kind == "random"
            else torch.full((B, Lq, Hq, D), 8 / size, device="cuda")).half()
    keep = torch.rand((B, Lk), generator=torch.Generator(device="cuda").manual_seed(6), device="cuda") < 0.7
    keep[:, 0] = True
    for n, bad in enumerate((math.nan, math.inf, -math.inf, 65504.0)):
        k[:, n::4][~keep[:, n::4]] = bad
        v[:, n::4][~keep[:, n::4]] = bad
    kw = {"key_mask": keep}
    if bias:
        kw.update(bias_table=_randn(torch, (Hq, 8), 7, torch.float16), max_distance=24)
    _check(torch, ww, {"q": q, "k": k, "v": v, "dout": dout}, kw, keep)


@pytest.mark.parametrize("D", [32, 64, 128])
def test_incoming_gradients_far_apart(env, D):
    """One row of dO ten thousand times the others, and one batch item's a millionth of another's."""
    torch, ww = env
    a = {n: _randn(torch, (3, L, 2, D), i, torch.float16) for i, (n, L) in enumerate((("q", 100), ("k", 150), ("v", 150)))}
    dout = _randn(torch, (3, 100, 2, D), 9, torch.float32)
    dout[0] *= 1e-2
    dout[0, 41] *= 1e4
    dout[2] *= 1e-6
    _check(torch, ww, {**a, "dout": dout.half()})
    lens = torch.tensor([150, 0, 77], device="cuda", dtype=torch.int32)
    keep = torch.arange(150, device="cuda")[None] < lens[:, None]
    for x in (a["k"], a["v"]):
        x[~keep] = math.inf
    _check(torch, ww, {**a, "dout": dout.half()}, {"k_lens": lens}, keep)


def test_rows_far_apart(env):
    """The queries' gradient keeps rows of dO that are 2^-20 of the largest (dq against its own row's bound)."""
    torch, ww = env
    a = {n: _randn(torch, (1, L, 1, 64), i, torch.float16) for i, (n, L) in enumerate((("q", 128), ("k", 256), ("v", 256)))}
    base = _randn(torch, (1, 128, 1, 64), 9, torch.float32)
    up = torch.where(torch.arange(128, device="cuda") % 2 == 0, 2.0 ** 8, 2.0 ** -12)[None, :, None, None]
    dout = (base * up).half()
    out, lse = ww.cross_attention(a["q"], a["k"], a["v"], return_lse=True)
    dq = ww.cross_attention_backward(dout, a["q"], a["k"], a["v"], out, lse)[0]
    keep = torch.ones((1, 256), dtype=torch.bool, device="cuda")
    for rows in (slice(0, None, 2), slice(1, None, 2)):
        one = {"q": a["q"][:, rows], "k": a["k"], "v": a["v"], "dout": dout[:, rows]}
        ref, bounds = _attention_ref(torch, ww, one, {}, keep, 1 / 8)
        M = 2 * one["dout"].double().norm(dim=-1).max().item() * a["v"].double().norm(dim=-1).max().item()
        # of a result, half a step of fp16 where it is below the normal range
        bound = bounds(U["f16"], 2.0 ** -39 * M / 2)["dq"] + TINY["f16"]
        _within(dq[:, rows], ref["dq"], bound, f"rows {rows}")
