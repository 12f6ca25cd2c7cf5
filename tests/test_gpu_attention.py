"""ww_qk_norm_rope and ww_cross_attention with their gradients on the GPU
against plain implementations in 64 bits (the reference library has no such
ops; their formulas are the specification).

Tolerances, per value, from the roundings the kernels make; u = 2^-11 (fp16),
2^-8 (bf16), 2^-24 (fp32) is a type's unit roundoff:

* norm and rotation: one rounding of the result (u |y|) and fp32 arithmetic
  (2^-20 of the sum of the magnitudes that enter a value);
* attention: out = P v with P rounded once and out rounded once:
  (2 u + e) sum P |v|;  dv the same with |dout|;  dq, dk: dS rounded once, the
  result once, and delta = sum dout * out from the rounded out:
  scale sum ((2 u + e) |dS| + P (u + e) (|dout| . |out| + |dout| . |v|)) |k|;
  dtable: the same without the product with k, and no rounding of dS;
  e = 2^-12 covers fp32 scores (|s| < 40 here, 2^-24 relative, amplified by
  exp and by 128 terms), the exponential's 2^-22 and fp32 sums;
* plus half a subnormal step of the 16-bit type where P or a result falls
  below its normal range (fp16: 2^-25 per term)."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8, "f32": 2.0 ** -24}
E = 2.0 ** -12
TINY = {"f16": 2.0 ** -25, "bf16": 0.0, "f32": 0.0}


@pytest.fixture(scope="module")
def env():
    import torch
    import whirlwind_trt_plugins_b200 as ww
    return torch, ww


def _type(torch, name):
    return {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}[name]


def _randn(torch, shape, seed, dt, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dt)


def _within(got, ref, bound, what):
    d = (got.double() - ref).abs() - bound
    assert bool(torch_isfinite(got)), f"{what}: not finite"
    assert got.numel() == 0 or d.max().item() <= 0, f"{what}: {d.max().item():.3e} over its bound"


def torch_isfinite(t):
    import torch
    return torch.isfinite(t).all()


# ---------------------------------------------------------------- norm and rotation

def _rope_ref(torch, x, w, cos, sin, pos, eps, interleaved):
    """64-bit result and the sum of magnitudes behind each value."""
    L, R = x.shape[1], 2 * cos.shape[1]
    pos = torch.arange(L, device=x.device) if pos is None else pos.long()
    pos = pos.clamp(0, cos.shape[0] - 1)
    if pos.dim() == 1:
        pos = pos[None]
    c, s = cos.double()[pos][:, :, None], sin.double()[pos][:, :, None]
    y = x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + eps) * w
    i = torch.arange(R // 2, device=x.device)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + R // 2)
    out, mag = y.clone(), y.detach().abs().clone()
    out[..., a] = y[..., a] * c - y[..., b] * s
    out[..., b] = y[..., b] * c + y[..., a] * s
    mag[..., a] = (y[..., a] * c).abs().detach() + (y[..., b] * s).abs().detach()
    mag[..., b] = (y[..., b] * c).abs().detach() + (y[..., a] * s).abs().detach()
    return out, mag


# (B, Lq, Lk, Hq, Hk, D, R): single tokens, lengths 0, odd lengths and head
# counts, whole and part rotation, head dims of 1 to 32 lanes and non-powers of two
ROPE = [(1, 1, 1, 8, 8, 64, 64), (2, 7, 13, 5, 1, 32, 16), (3, 33, 0, 3, 2, 8, 8), (1, 0, 5, 4, 4, 128, 64),
        (2, 50, 41, 6, 3, 96, 96), (1, 70, 9, 1, 7, 40, 24), (2, 17, 300, 9, 2, 256, 128), (1, 5, 6, 2, 2, 80, 0)]


@pytest.mark.parametrize("shape", ROPE)
@pytest.mark.parametrize("dt", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("interleaved", [False, True])
def test_norm_rope_and_gradient(env, shape, dt, interleaved):
    torch, ww = env
    B, Lq, Lk, Hq, Hk, D, R = shape
    t, u = _type(torch, dt), U[dt]
    q, k = _randn(torch, (B, Lq, Hq, D), 1, t, 2.0), _randn(torch, (B, Lk, Hk, D), 2, t)
    wq, wk = _randn(torch, (D,), 3, t) + 1, _randn(torch, (D,), 4, t) + 1
    P = 350
    ang = torch.arange(P, device="cuda").double()[:, None] * 100.0 ** (-torch.arange(R // 2, device="cuda") / max(R, 1))
    cos, sin = ang.cos().float(), ang.sin().float()
    qpos = torch.randint(0, P, (B, Lq), device="cuda", dtype=torch.int32)
    kpos = torch.arange(Lk, device="cuda", dtype=torch.int32).flip(0).contiguous()
    gq, gk = _randn(torch, q.shape, 5, t), _randn(torch, k.shape, 6, t)
    eps = 1e-5
    got = ww.qk_norm_rope(q, k, wq, wk, cos, sin, qpos, kpos, eps, interleaved)
    back = ww.qk_norm_rope_backward(gq, gk, q, k, wq, wk, cos, sin, qpos, kpos, eps, interleaved)
    again = ww.qk_norm_rope_backward(gq, gk, q, k, wq, wk, cos, sin, qpos, kpos, eps, interleaved)
    assert all(torch.equal(a, b) for a, b in zip(back, again))  # sums in a fixed order
    f = 2.0 ** -20
    for n, (x, w, pos, g) in enumerate(((q, wq, qpos, gq), (k, wk, kpos, gk))):
        xd, wd = x.double().requires_grad_(True), w.double().requires_grad_(True)
        y, mag = _rope_ref(torch, xd, wd, cos, sin, pos, eps, interleaved)
        _within(got[n], y.detach(), u * y.detach().abs() + f * mag + TINY[dt], f"out {n}")
        dx, dw = torch.autograd.grad(y, (xd, wd), g.double())
        # what enters dx: |g'| w and |x| r mean |g' w xh|, g' the gradient turned back
        r = torch.rsqrt(x.double().pow(2).mean(-1, keepdim=True) + eps)
        ga = _turned_magnitude(torch, g.double(), cos, sin, pos, interleaved)
        xh = (x.double() * r).abs()
        mag = r * (ga * wd.detach().abs() + xh * (ga * wd.detach().abs() * xh).mean(-1, keepdim=True))
        _within(back[n], dx, u * dx.abs() + f * mag + TINY[dt], f"dx {n}")
        _within(back[2 + n], dw, u * dw.abs() + f * (ga * xh).sum((0, 1, 2)) + TINY[dt], f"dw {n}")


def _turned_magnitude(torch, g, cos, sin, pos, interleaved):
    R = 2 * cos.shape[1]
    p = pos.long().clamp(0, cos.shape[0] - 1)
    p = p[None] if p.dim() == 1 else p
    c, s = cos.double()[p][:, :, None].abs(), sin.double()[p][:, :, None].abs()
    i = torch.arange(R // 2, device=g.device)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + R // 2)
    m, g = g.abs().clone(), g.abs()
    m[..., a] = g[..., a] * c + g[..., b] * s
    m[..., b] = g[..., b] * c + g[..., a] * s
    return m


def test_norm_rope_strides_positions_and_zero_rows(env):
    """Slices of one packed projection, a broadcast batch, positions beyond the
    tables (clamped) and all-zero vectors (no division by zero)."""
    torch, ww = env
    B, L, H, D = 3, 21, 4, 64
    packed = _randn(torch, (B, L, 3 * H, D), 7, torch.float16)
    packed[1, 4] = 0
    q, k = packed[:, :, :H], packed[:1, :, H:2 * H].expand(B, L, H, D)
    w = torch.ones(D, device="cuda", dtype=torch.float16)
    ang = torch.arange(16, device="cuda").float()[:, None] * torch.rand(32, device="cuda")
    pos = torch.arange(L, device="cuda", dtype=torch.int32) - 2
    a = ww.qk_norm_rope(q, k, w, w, ang.cos(), ang.sin(), pos, pos)
    b = ww.qk_norm_rope(q.contiguous(), k.contiguous(), w, w, ang.cos(), ang.sin(), pos.clamp(0, 15), pos.clamp(0, 15))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    assert a[0].is_contiguous() and bool((a[0][1, 4] == 0).all()) and bool(torch_isfinite(a[0]))


def test_norm_rope_gradient_against_differences(env):
    """Directional derivative of the fp32 operator against central differences
    (step 1e-3, third derivatives of order 1: 1e-5 relative to the direction's size)."""
    torch, ww = env
    q, k = _randn(torch, (2, 5, 3, 32), 8, torch.float32), _randn(torch, (2, 4, 3, 32), 9, torch.float32)
    w = _randn(torch, (32,), 10, torch.float32) + 1
    ang = torch.arange(8, device="cuda").float()[:, None] * torch.rand(16, device="cuda")
    gq, gk = _randn(torch, q.shape, 11, torch.float32), _randn(torch, k.shape, 12, torch.float32)
    tq, tk, tw = (_randn(torch, x.shape, 13 + n, torch.float32) for n, x in enumerate((q, k, w)))

    def loss(h):
        a, b = ww.qk_norm_rope(q + h * tq, k + h * tk, w + h * tw, w + h * tw, ang.cos(), ang.sin())
        return ((a * gq).double().sum() + (b * gk).double().sum()).item()

    d = ww.qk_norm_rope_backward(gq, gk, q, k, w, w, ang.cos(), ang.sin())
    want = ((d[0] * tq).double().sum() + (d[1] * tk).double().sum() + ((d[2] + d[3]) * tw).double().sum()).item()
    got = (loss(1e-2) - loss(-1e-2)) / 2e-2
    size = math.sqrt(sum(x.double().pow(2).sum().item() for x in (gq, gk)))
    # truncation h^2 / 6 f''' with f''' <= 30 of the direction's size; rounding 2^-22 sum / h
    assert abs(got - want) <= (1e-4 / 6 * 30 + 2.0 ** -22 / 1e-2) * size * math.sqrt(q.numel())


# ---------------------------------------------------------------- attention

def _buckets_ref(torch, ww, Lq, Lk, n, dist, bi, off):
    rel = np.arange(-(Lq - 1) - off, Lk - off)
    row = torch.tensor([ww.relative_position_bucket(int(r), n, dist, bi) for r in rel], device="cuda")
    at = torch.arange(Lk, device="cuda")[None, :] - torch.arange(Lq, device="cuda")[:, None] + (Lq - 1)
    return row[at]


def _attention_case(torch, ww, B, Lq, Lk, Hq, Hk, D, dt, mask, bias, seed=0, garbage=True):
    t = _type(torch, dt)
    a = {"q": _randn(torch, (B, Lq, Hq, D), seed + 1, t), "k": _randn(torch, (B, Lk, Hk, D), seed + 2, t),
         "v": _randn(torch, (B, Lk, Hk, D), seed + 3, t), "dout": _randn(torch, (B, Lq, Hq, D), seed + 4, t)}
    keep = torch.ones((B, Lk), dtype=torch.bool, device="cuda")
    kw = {}
    if "lens" in mask:
        lens = [Lk, 0, 1, max(0, Lk - 3)][:B] if B > 1 else [max(0, Lk - 1)]
        lens += [Lk // 2] * (B - len(lens))
        kw["k_lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        keep &= torch.arange(Lk, device="cuda")[None] < kw["k_lens"][:, None]
    if "keys" in mask:
        g = torch.Generator(device="cuda").manual_seed(seed + 5)
        m = torch.rand((B, Lk), generator=g, device="cuda") < 0.6
        m[-1] = False  # an item without a key
        kw["key_mask"] = m
        keep &= m
    if garbage:  # what masked places hold does not matter
        bad = torch.tensor([float("nan"), float("inf"), -float("inf"), 6e4], device="cuda").to(t)
        for x in (a["k"], a["v"]):
            n = int((~keep).sum())
            x[~keep] = bad[torch.arange(n, device="cuda") % 4][:, None, None]
    if bias is not None:
        n, dist, bi, off = bias
        kw.update(bias_table=_randn(torch, (Hq, n), seed + 6, t), max_distance=dist, bidirectional=bi, q_offset=off)
    return a, kw, keep


def _attention_ref(torch, ww, a, kw, keep, scale):
    """64-bit results and error bounds (in units where u and e multiply)."""
    q, k, v, do = (a[n].double() for n in ("q", "k", "v", "dout"))
    B, Lq, Hq, D = q.shape
    Lk, Hk = k.shape[1], k.shape[2]
    G = Hq // Hk
    zero = ~keep[:, :, None, None]
    k, v = k.masked_fill(zero, 0.0), v.masked_fill(zero, 0.0)
    q, do = q.transpose(1, 2), do.transpose(1, 2)                    # [B, Hq, Lq, D]
    k, v = (x.transpose(1, 2).repeat_interleave(G, 1) for x in (k, v))
    s = scale * q @ k.transpose(2, 3)
    buckets = None
    if "bias_table" in kw:
        buckets = _buckets_ref(torch, ww, Lq, Lk, kw["bias_table"].shape[1], kw["max_distance"], kw["bidirectional"],
                               kw["q_offset"])
        table = kw["bias_table"].double()
        table = torch.where(table <= torch.finfo(kw["bias_table"].dtype).min, -math.inf, table)
        s = s + table[:, buckets]
    s = s.masked_fill(~keep[:, None, None, :], -math.inf)
    lse = torch.logsumexp(s, -1) if Lk else torch.full(s.shape[:3], -math.inf, dtype=torch.float64, device="cuda")
    p = torch.exp(s - torch.where(lse == -math.inf, 0.0, lse)[..., None])
    p = torch.where((lse == -math.inf)[..., None], 0.0, p)
    out = p @ v
    dp = do @ v.transpose(2, 3)
    delta = (do * out).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    # |dout| . |out| + |dout| . |v| behind dP - delta
    behind = p * ((do.abs() * out.abs()).sum(-1, keepdim=True) + do.abs() @ v.abs().transpose(2, 3))
    put = lambda x: x.transpose(1, 2)  # noqa: E731
    share = lambda x: put(x.reshape(B, Hk, G, Lk, D).sum(2))  # noqa: E731
    r = {"out": put(out), "lse": lse, "dq": put(scale * ds @ k), "dk": share(scale * ds.transpose(2, 3) @ q),
         "dv": share(p.transpose(2, 3) @ do)}

    def bounds(u, tiny):
        n2 = 2 * u + E
        loose = n2 * ds.abs() + (u + E) * behind + 2 * tiny
        b = {"out": n2 * put(p @ v.abs()) + 300 * tiny * put((p > 0).double() @ v.abs()) + tiny,
             "dq": scale * put(loose @ k.abs()) + tiny, "dk": share(scale * loose.transpose(2, 3) @ q.abs()) + tiny,
             "dv": share((n2 * p + 2 * tiny * (p > 0)).transpose(2, 3) @ do.abs()) + tiny}
        if buckets is not None:
            b["dtable"] = _by_bucket(torch, E * ds.abs() + (u + E) * behind, buckets, table) \
                + u * r["dtable"].abs() + tiny
        return b

    if buckets is not None:
        r["dtable"] = _by_bucket(torch, ds, buckets, table)
    return r, bounds


def _by_bucket(torch, x, buckets, table):
    flat = x.sum(0).flatten(1)
    return torch.zeros_like(table).index_add_(1, buckets.flatten(), flat)


# (B, Lq, Lk, Hq, Hk, D): one token, tiles that end early, lengths around the
# tile sizes 64, 128 and 256, shared heads, head dims that are not powers of two
SHAPES = [(1, 1, 1, 1, 1, 8), (2, 1, 77, 4, 2, 64), (4, 1, 700, 16, 4, 128), (2, 5, 129, 4, 1, 40),
          (3, 128, 128, 2, 2, 32), (1, 129, 257, 6, 3, 64), (2, 200, 63, 4, 4, 128), (1, 300, 640, 2, 1, 80),
          (4, 16, 1000, 8, 8, 64), (5, 65, 191, 3, 3, 24), (2, 256, 256, 2, 2, 128), (1, 9, 2500, 2, 2, 96),
          (2, 1000, 3, 2, 1, 64)]
BIASES = [None, (32, 128, True, 0), (8, 20, False, -3), (128, 500, True, 60)]


def _run_case(env, shape, dt, mask, bias, seed=0, garbage=True):
    torch, ww = env
    a, kw, keep = _attention_case(torch, ww, *shape, dt, mask, bias, seed, garbage)
    scale = 1.3 / math.sqrt(shape[-1])
    out, lse = ww.cross_attention(a["q"], a["k"], a["v"], scale, return_lse=True, **kw)
    only = ww.cross_attention(a["q"], a["k"], a["v"], scale, **kw)
    dq, dk, dv, dtable = ww.cross_attention_backward(a["dout"], a["q"], a["k"], a["v"], out, lse, scale, **kw)
    again = ww.cross_attention_backward(a["dout"], a["q"], a["k"], a["v"], out, lse, scale, **kw)
    assert torch.equal(only, out)
    ref, bounds = _attention_ref(torch, ww, a, kw, keep, scale)
    bound = bounds(U[dt], TINY[dt])
    got = {"out": out, "dq": dq, "dk": dk, "dv": dv}
    if bias is not None:
        got["dtable"] = dtable
    else:
        assert dtable is None
    for n, x in got.items():
        _within(x, ref[n], bound[n], n)
    empty = ref["lse"] == -math.inf
    assert torch.equal(lse == -math.inf, empty)
    assert bool(((lse.double() - ref["lse"])[~empty].abs() <= E * (1 + ref["lse"][~empty].abs())).all())
    assert bool((dk[~keep] == 0).all()) and bool((dv[~keep] == 0).all())
    for x, y in zip((dq, dk, dv, dtable), again):
        assert x is None or torch.equal(x, y)  # the same call gives the same bits
    assert ww.device_error() == 0


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("bias", BIASES)
@pytest.mark.parametrize("mask", ["", "lens", "keys", "lens keys"])
def test_attention_and_gradients(env, shape, mask, bias):
    _run_case(env, shape, "f16" if (SHAPES.index(shape) + BIASES.index(bias)) % 2 else "bf16", mask, bias)


@pytest.mark.parametrize("dt", ["f16", "bf16"])
def test_rows_of_a_stereo_pair(env, dt):
    _run_case(env, (40, 160, 160, 5, 5, 64), dt, "keys", (32, 128, True, 0), 3)


@pytest.mark.parametrize("shape", [(1, 1, 20001, 8, 2, 128), (2, 3, 9000, 4, 4, 64), (1, 140, 5000, 2, 2, 32),
                                   (1, 6000, 70, 2, 1, 64)])
def test_long_axes(env, shape):
    """Few rows against long ones: the work is split over the long axis and joined."""
    _run_case(env, shape, "bf16", "", (32, 300, False, shape[2] - shape[1]), 4)
    _run_case(env, shape, "f16", "keys", None, 5)


# Both sides of each rule that picks how a call runs: single tokens of many heads that
# do not share keys, more and fewer than 2048 queries, several query blocks per CTA,
# last rounds that are split over the streamed axis and ones that are not.
@pytest.mark.parametrize("shape", [(40, 1, 100, 4, 4, 64), (25, 30, 70, 6, 6, 24), (38, 2, 90, 4, 2, 128),
                                   (1, 2300, 300, 2, 2, 32), (1, 2100, 200, 3, 1, 64), (1, 2300, 300, 1, 1, 128),
                                   (100, 300, 140, 3, 3, 32), (1, 300, 1500, 16, 16, 64), (2, 300, 1500, 16, 8, 128)])
@pytest.mark.parametrize("mask,bias", [("", None), ("lens keys", (16, 100, True, 5))])
def test_forms(env, shape, mask, bias):
    _run_case(env, shape, "f16" if shape[1] % 4 else "bf16", mask, bias, 6)


@pytest.mark.parametrize("shape", [(700, 51, 43, 6, 3, 80), (150, 160, 160, 5, 5, 64), (400, 130, 300, 3, 3, 32),
                                   (300, 7, 20, 5, 5, 40), (90, 257, 65, 7, 7, 128)])
@pytest.mark.parametrize("mask,bias", [("", None), ("keys", None), ("", (32, 40, False, 3)), ("keys", (8, 300, True, 0))])
def test_many_short_rows(env, shape, mask, bias):
    """Query blocks of several batch items one after the other in a CTA."""
    _run_case(env, shape, "bf16" if shape[0] % 4 else "f16", mask, bias, 7)


@pytest.mark.parametrize("shape", [(1, 200, 2600, 1, 1, 128), (1, 2600, 200, 2, 1, 128), (1, 150, 2600, 2, 2, 64),
                                   (1, 2600, 150, 1, 1, 32), (1, 4, 2600, 4, 1, 128)])
def test_widest_tables(env, shape):
    """The most buckets and the longest distance, every position of a range in use."""
    _run_case(env, shape, "bf16", "keys", (128, 1024, True, (shape[2] - shape[1]) // 2), 8)


@pytest.mark.parametrize("Lq,Lk,B", [(0, 5, 2), (5, 0, 2), (0, 0, 1), (3, 4, 0)])
def test_lengths_of_zero(env, Lq, Lk, B):
    torch, ww = env
    q = torch.randn((B, Lq, 4, 64), device="cuda").half()
    k = torch.randn((B, Lk, 2, 64), device="cuda").half()
    table = torch.randn((4, 8), device="cuda").half()
    out, lse = ww.cross_attention(q, k, k, bias_table=table, max_distance=32, return_lse=True)
    assert out.shape == q.shape and bool((out == 0).all()) == (Lk == 0 or out.numel() == 0)
    got = ww.cross_attention_backward(q, q, k, k, out, lse, bias_table=table, max_distance=32)
    if Lk == 0 or Lq == 0 or B == 0:
        assert all(bool((x == 0).all()) for x in got)


def test_strides_and_broadcast_inputs(env):
    """Queries, keys and values as slices of packed projections, and states
    shared by a batch and by heads through stride 0, against contiguous copies."""
    torch, ww = env
    B, L, H, D = 3, 150, 4, 64
    pk = _randn(torch, (B, L, 3, H, D), 21, torch.bfloat16)
    q, k, v = pk[:, :, 0], pk[:, :, 1], pk[:, :, 2]
    kb, vb = k[:1].expand(B, L, H, D), v[:, :, :1].expand(B, L, H, D)
    qt = q.transpose(1, 2).contiguous().transpose(1, 2)  # heads outside of tokens
    for a in ((q, k, v), (q, kb, vb), (qt, k, v), (q[:, :1], kb, vb), (q[:, 3:90], k[:, 5:, 1:3], v[:, 5:, 1:3])):
        c = [x.contiguous() for x in a]
        out, lse = ww.cross_attention(*a, return_lse=True)
        ref, lref = ww.cross_attention(*c, return_lse=True)
        assert torch.equal(out, ref) and torch.equal(lse, lref)
        do = _randn(torch, (B, out.shape[1], D, H), 22, torch.bfloat16).contiguous().transpose(2, 3).contiguous()
        got = ww.cross_attention_backward(do, *a, out, lse)
        want = ww.cross_attention_backward(do, *c, out, lse)
        assert all(torch.equal(x, y) for x, y in zip(got[:3], want[:3]))


def test_forbidden_biases_and_large_scores(env):
    """Table values of -inf and of the type's lowest forbid their pairs (a row
    of them alone is empty); scores of thousands leave a finite one-hot softmax."""
    torch, ww = env
    for dt in (torch.float16, torch.bfloat16):
        q, k, v = (_randn(torch, (2, 70, 2, 64), 30 + n, dt) for n in range(3))
        table = _randn(torch, (2, 8), 33, dt)
        table[:, 5] = torch.finfo(dt).min
        table[:, 6] = -math.inf
        table[1] = torch.finfo(dt).min
        kw = {"bias_table": table, "max_distance": 16}
        do = _randn(torch, q.shape, 34, dt)
        keep = torch.ones((2, 70), dtype=torch.bool, device="cuda")
        out, lse = ww.cross_attention(q, k, v, return_lse=True, **kw)
        grads = ww.cross_attention_backward(do, q, k, v, out, lse, **kw)
        full = dict(kw, bidirectional=True, q_offset=0)
        ref, bounds = _attention_ref(torch, ww, {"q": q, "k": k, "v": v, "dout": do}, full, keep, 1 / 8)
        name = "f16" if dt == torch.float16 else "bf16"
        b = bounds(U[name], TINY[name])
        _within(out, ref["out"], b["out"], "out")
        for n, x in zip(("dq", "dk", "dv", "dtable"), grads):
            _within(x, ref[n], b[n], n)
        assert bool((out[:, :, 1] == 0).all()) and bool((lse[:, 1] == -math.inf).all())
        assert bool((grads[3][:, 5:7] == 0).all()) and bool((grads[3][1] == 0).all())
        q30, k30 = q * 30, k * 30
        big = ww.cross_attention(q30, k30, v)
        s = q30.double().transpose(1, 2) @ k30.double().permute(0, 2, 3, 1) / 8
        top = torch.softmax(s, -1) @ v.double().transpose(1, 2)
        # fp32 scores of up to 2^12 are within 2^-9: P within 2^-8 of its value
        lim = (2 * U[name] + 2.0 ** -7) * (torch.softmax(s, -1) @ v.double().abs().transpose(1, 2)) + 1e-6
        _within(big, top.transpose(1, 2), lim.transpose(1, 2), "large scores")


def test_attention_gradient_against_differences(env):
    """Directional derivative of a 64-bit restatement by central differences
    against the kernel's gradients, bf16 roundings at their summed bound."""
    torch, ww = env
    shape, bias = (2, 33, 50, 4, 2, 32), (8, 24, True, 2)
    a, kw, keep = _attention_case(torch, ww, *shape, "f16", "keys", bias, 40, garbage=False)
    scale = 0.2
    out, lse = ww.cross_attention(a["q"], a["k"], a["v"], scale, return_lse=True, **kw)
    got = ww.cross_attention_backward(a["dout"], a["q"], a["k"], a["v"], out, lse, scale, **kw)
    _, bounds = _attention_ref(torch, ww, a, kw, keep, scale)
    b = bounds(U["f16"], TINY["f16"])
    for n, (name, where) in enumerate((("dq", "q"), ("dk", "k"), ("dv", "v"), ("dtable", "bias_table"))):
        src = a[where] if where in a else kw[where]
        t = _randn(torch, src.shape, 50 + n, torch.float64)

        def loss(h):
            moved, more = dict(a), dict(kw)
            x = src.double() + h * t
            if where in a:
                moved[where] = x
            else:
                more[where] = x
            r, _ = _attention_ref(torch, ww, moved, more, keep, scale)
            return (r["out"] * a["dout"].double()).sum().item()

        want = (loss(1e-4) - loss(-1e-4)) / 2e-4
        have = (got[n].double() * t).sum().item()
        assert abs(have - want) <= (b[name] * t.abs()).sum().item() + 1e-5 * abs(want) + 1e-6


def test_autograd_and_streams(env):
    """The differentiable forms, with an expanded gradient and shared encoder
    states, give the functions' gradients; a side stream gives the same bits."""
    torch, ww = env
    q = _randn(torch, (3, 40, 4, 64), 60, torch.bfloat16).requires_grad_(True)
    k = _randn(torch, (1, 90, 2, 64), 61, torch.bfloat16).requires_grad_(True)
    v = _randn(torch, (1, 90, 2, 64), 62, torch.bfloat16).requires_grad_(True)
    w = torch.ones(64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    table = _randn(torch, (4, 16), 63, torch.bfloat16).requires_grad_(True)
    ang = torch.arange(90, device="cuda").float()[:, None] * torch.rand(32, device="cuda")
    cos, sin = ang.cos(), ang.sin()
    qr, kr = ww.qk_norm_rope_autograd(q, k.expand(3, 90, 2, 64), w, w, cos, sin)
    out = ww.cross_attention_autograd(qr, kr, v.expand(3, 90, 2, 64), table, max_distance=64)
    out.sum(dim=(0, 2, 3)).mean().backward()
    assert q.grad.shape == q.shape and k.grad.shape == k.shape and v.grad.shape == v.shape
    assert w.grad is not None and table.grad.shape == table.shape
    # the same by hand: shared states get the sum over the batch
    with torch.no_grad():
        ke, ve = k.expand(3, 90, 2, 64), v.expand(3, 90, 2, 64)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        qr2, kr2 = ww.qk_norm_rope(q, ke, w, w, cos, sin, stream=side)
        o2, lse = ww.cross_attention(qr2, kr2, ve, bias_table=table, max_distance=64, return_lse=True, stream=side)
        with torch.cuda.stream(side):
            do = torch.full(o2.shape, 1 / 40, device="cuda", dtype=torch.bfloat16)
        g = ww.cross_attention_backward(do, qr2, kr2, ve, o2, lse, bias_table=table, max_distance=64,
                                        stream=side.cuda_stream)
        n = ww.qk_norm_rope_backward(g[0], g[1], q, ke, w, w, cos, sin, stream=side)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(out, o2) and torch.equal(table.grad, g[3]) and torch.equal(q.grad, n[0])
        assert torch.allclose(v.grad.float(), g[2].float().sum(0, keepdim=True), rtol=2 ** -6, atol=1e-3)


def test_refusals(env):
    torch, ww = env
    q = torch.zeros((2, 4, 4, 64), device="cuda", dtype=torch.float16)
    k = torch.zeros((2, 6, 2, 64), device="cuda", dtype=torch.float16)
    with pytest.raises(TypeError):
        ww.cross_attention(q.float(), k.float(), k.float())
    with pytest.raises(TypeError):
        ww.cross_attention(q.cpu(), k, k)
    with pytest.raises(TypeError):
        ww.cross_attention(q, k.bfloat16(), k)
    with pytest.raises(ValueError):
        ww.cross_attention(q, k[:1], k)
    with pytest.raises(ValueError):
        ww.cross_attention(q, k, k[:, :5])
    with pytest.raises(ValueError):  # 4 heads over 3
        ww.cross_attention(q, torch.zeros((2, 6, 3, 64), device="cuda").half(), torch.zeros((2, 6, 3, 64), device="cuda").half())
    with pytest.raises(ValueError):  # strides of 65 elements
        ww.cross_attention(torch.zeros((2, 4, 4, 65), device="cuda").half()[..., :64], k, k)
    with pytest.raises(ValueError):
        ww.cross_attention(q, k, k, out=torch.empty((2, 4, 4, 32), device="cuda").half())
    with pytest.raises(ValueError):
        ww.cross_attention(q, k, k, key_mask=torch.ones((2, 5), device="cuda", dtype=torch.bool))
    with pytest.raises(TypeError):
        ww.cross_attention(q, k, k, k_lens=torch.ones(2, device="cuda", dtype=torch.int64))
    with pytest.raises(ValueError):
        ww.cross_attention(q, k, k, bias_table=torch.zeros((2, 8), device="cuda").half())
    for table, dist in ((9, 32), (8, 2)):  # odd and bidirectional; no room for the logarithm
        with pytest.raises(ww.WWError) as e:
            ww.cross_attention(q, k, k, bias_table=torch.zeros((4, table), device="cuda").half(), max_distance=dist)
        assert e.value.status == 2
    for wide in (12, 136):
        x = torch.zeros((1, 2, 2, wide), device="cuda").half()
        with pytest.raises((ww.WWError, ValueError)):
            ww.cross_attention(x, x, x)
    with pytest.raises(ww.WWError) as e:  # a base off the 16-byte grid
        buf = torch.zeros(8 * 64 + 1, device="cuda").half()[1:].view(1, 2, 4, 64)
        ww.cross_attention(buf, buf, buf)
    assert e.value.status == 6
    cos = torch.zeros((8, 32), device="cuda")
    w = torch.ones(64, device="cuda").half()
    with pytest.raises(ValueError):
        ww.qk_norm_rope(q, k, w[:32], w, cos, cos)
    with pytest.raises(ValueError):
        ww.qk_norm_rope(q, k, w, w, torch.zeros((8, 40), device="cuda"), torch.zeros((8, 40), device="cuda"))
    with pytest.raises(TypeError):
        ww.qk_norm_rope(q, k, w, w, cos.half(), cos.half())
    with pytest.raises(ValueError):
        ww.qk_norm_rope(q, k, w, w, cos, cos, q_pos=torch.zeros(3, device="cuda", dtype=torch.int32))
    with pytest.raises(ww.WWError):  # 12 rotated dims
        ww.qk_norm_rope(q, k, w, w, cos[:, :6].contiguous(), cos[:, :6].contiguous())


def test_plugin_enqueue_and_calls_without_workspace(env):
    """The plugins give the functions' bits; without a workspace the keys are not
    split, which rounds differently but stays within the bounds."""
    torch, ww = env
    from whirlwind_trt_plugins_b200 import plugins as pl
    T = pl.TensorDesc.of
    a, kw, keep = _attention_case(torch, ww, 2, 3, 900, 8, 2, 64, "bf16", "lens keys", (32, 64, True, 5), 70)
    p = pl.get_plugin_creator("CrossAttention").create_plugin(
        {"use_lens": 1, "use_mask": 1, "use_bias": 1, "max_distance": 64, "q_offset": 5})
    ins = [a["q"], a["k"], a["v"], kw["k_lens"], kw["key_mask"], kw["bias_table"]]
    want = ww.cross_attention(a["q"], a["k"], a["v"], **kw)
    ws = torch.empty(p.get_workspace_size(), dtype=torch.uint8, device="cuda")
    out, plain = torch.empty_like(want), torch.empty_like(want)
    assert p.enqueue([T(x) for x in ins], ins, [out], ws) == 0
    assert p.enqueue([T(x) for x in ins], ins, [plain]) == 0
    assert torch.equal(out, want)
    ref, bounds = _attention_ref(torch, ww, a, kw, keep, 1 / 8)
    _within(plain, ref["out"], bounds(U["bf16"], 0.0)["out"], "without workspace")
    w = torch.ones(64, device="cuda", dtype=torch.bfloat16)
    ang = torch.arange(900, device="cuda").float()[:, None] * torch.rand(32, device="cuda")
    cos, sin = ang.cos(), ang.sin()
    pos = torch.arange(3, device="cuda", dtype=torch.int32) + 5, torch.arange(900, device="cuda", dtype=torch.int32)
    k = torch.randn((2, 900, 2, 64), device="cuda").bfloat16()
    want = ww.qk_norm_rope(a["q"], k, w, w, cos, sin, *pos, eps=1e-6)
    r = pl.get_plugin_creator("QkNormRope").create_plugin({"use_positions": 1})
    ins = [a["q"], k, w, w, cos, sin, *pos]
    outs = [torch.empty_like(x) for x in want]
    assert r.enqueue([T(x) for x in ins], ins, outs) == 0
    assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])


def test_example_trains_and_matches():
    """The matching layer of examples/: training lowers its loss, its features
    give the rows' disparities through the volume and the regression."""
    import importlib.util
    import os

    from conftest import ROOT
    spec = importlib.util.spec_from_file_location("example", os.path.join(ROOT, "examples", "stereo_cross_attention.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    losses, error = m.main(steps=60, verbose=False)
    assert all(map(math.isfinite, losses))
    assert sum(losses[-5:]) < 0.9 * sum(losses[:5])
    assert error < 2.0
