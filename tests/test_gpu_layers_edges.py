"""The 8-bit layer operators at the edges of what they take, on the GPU against plain
implementations in 64 bits; tolerances count roundings as in test_gpu_layers.py."""
import math

import pytest
from test_gpu_layers import F, TINY, U, _attention_reference, _caches, _randn, _type, _weights, _within, env  # noqa: F401

pytestmark = pytest.mark.gpu

# every form of the norm: 4 to 32 lanes a row, 2 to 4 pieces a lane, blocks, single values, pairs, rows beyond a block's
# registers, all with a length whose reciprocal is rounded
NORM_LENGTHS = [24, 40, 120, 250, 264, 328, 504, 712, 1000, 1048, 1337, 3, 100, 5001, 4104, 40001]


def _one_value_rows(torch, t, n, rows):
    """Rows of one value each."""
    values = torch.tensor([3.0, 1000.0, 30000.0, -0.1, 1000.1, 2.0 ** -14, 7.0], device="cuda").to(t)
    return values.repeat(rows // 7 + 1)[:rows, None].repeat(1, n)


@pytest.mark.parametrize("n", NORM_LENGTHS)
@pytest.mark.parametrize("dt", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("residual", [False, True])
def test_layer_norm_of_rows_of_one_value(env, n, dt, residual):  # noqa: F811
    """Their deviations are 0, whatever rounding the mean has met: the result is the bias, in 8 bits 0, and the mean the value."""
    torch, ww = env
    t = _type(torch, dt)
    x = _one_value_rows(torch, t, n, 40)
    r = torch.full_like(x, 0.5) if residual else None
    h = x + r if residual else x
    b = _randn(torch, (n,), 1, t)
    y, *more = ww.layer_norm(x, residual=r, return_stats=True)
    assert not y.any()
    assert torch.equal(more[-2], h[:, 0].float())
    assert ((more[-1].double() * math.sqrt(1e-5) - 1).abs() <= F).all()
    assert torch.equal(ww.layer_norm(x, torch.ones_like(b), b, residual=r)[0 if residual else slice(None)], b.expand(40, n))
    q, scale, *_ = ww.layer_norm_int8(x, residual=r)
    assert not q.any() and not scale.any()


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_layer_norm_of_many_sums_of_one_value(env, dt):  # noqa: F811
    """The same through the ring of long rows with a residual."""
    torch, ww = env
    t = _type(torch, dt)
    x = _one_value_rows(torch, t, 4104, 1200)
    r = torch.full_like(x, 0.5)
    y, h, mean, rstd = ww.layer_norm(x, residual=r, return_stats=True)
    assert not y.any() and torch.equal(mean, h[:, 0].float()) and ((rstd.double() * math.sqrt(1e-5) - 1).abs() <= F).all()
    q, scale, _ = ww.layer_norm_int8(x, residual=r)
    assert not q.any() and not scale.any()
    assert ww.device_error() == 0


@pytest.mark.parametrize("n", NORM_LENGTHS)
@pytest.mark.parametrize("size", [100.0, 4096.0, 1e6])
def test_layer_norm_far_from_zero(env, n, size):  # noqa: F811
    """Deviations of about 1 around a mean far above them: x less the fp32 mean is exact (neighbours of one another), what is
    left of the mean is found to 2^-18 of the mean deviation, and so the result keeps its digits.  Rows between them that are
    not far from zero have the bits that they have by themselves."""
    torch, ww = env
    x = _randn(torch, (23, n), 1, torch.float32)
    near = torch.arange(23, device="cuda") % 3 == 1
    x[~near] += size
    y, mean, rstd = ww.layer_norm(x, return_stats=True)
    d = x.double() - x.double().mean(-1, keepdim=True)
    rs = 1 / torch.sqrt(d.pow(2).mean(-1, keepdim=True) + 1e-5)
    mag = (d.abs() + d.abs().mean(-1, keepdim=True)) * rs
    bound = 2.0 ** -18 * mag
    bound[near] += F * (x.double().abs().mean(-1, keepdim=True) * rs)[near]
    _within(y, d * rs, bound, "y")
    _within(mean, x.double().mean(-1), F * x.double().abs().mean(-1), "mean")
    _within(rstd, rs[:, 0], 2.0 ** -18 * rs[:, 0], "rstd")
    alone = x.clone()
    alone[~near] = x[near][0]
    assert torch.equal(ww.layer_norm(alone)[near], y[near])


# ---------------------------------------------------------------- products

@pytest.mark.parametrize("shape", [(13090, 256, 288), (9600, 256, 416), (4300, 256, 1056)])
@pytest.mark.parametrize("dt", ["f16", "f32"])
def test_products_of_tiles_in_part_outside(env, shape, dt):  # noqa: F811
    """Several narrow tiles a block, between them some whose second half lies outside the result and is not stored: what is
    staged for the next one does not reach a store that is still under way."""
    torch, ww = env
    M, K, N = shape
    t, u = _type(torch, dt), U[dt]
    w, ws = _weights(torch, ww, N, K, 1)
    x = _randn(torch, (M, K), 2, t)
    xq, xs = ww.quantize_tokens(x)
    one = (xq.double() @ w.double().t()) * xs.double()[:, None] * ws.double()
    for _ in range(5):
        _within(ww.int8_matmul(xq, xs, w, ws, dtype=t), one, u * one.abs() + 2.0 ** -22 * one.abs() + TINY[dt], "out")
    assert ww.device_error() == 0


# ---------------------------------------------------------------- attention by 16-bit copies

# (B, Lq, Lk, Hq, Hk, D): more rows a key head than are read from the 8-bit form, and fewer that are faster by copies in fp16
MANY = [(2, 70, 300, 6, 3, 64), (3, 150, 333, 4, 4, 32), (2, 200, 1000, 2, 2, 128), (3, 45, 77, 12, 2, 48), (64, 1, 100, 160, 8, 64), (40, 48, 130, 8, 8, 32),
        (8, 100, 1100, 8, 8, 64)]
# factors of the keys' scales and of the values', and how far scores lie from one another
SIZES = [(0.05, 0.05, 3.0), (2.0 ** -20, 2.0 ** -12, 3.0), (2.0 ** 10, 0.05, 3.0), (2.0 ** 60, 2.0 ** -20, 3.0), (2.0 ** -90, 2.0 ** 11, 0.5)]


@pytest.mark.parametrize("shape", MANY)
@pytest.mark.parametrize("sizes", SIZES)
@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("form", ["plain", "masked", "biased"])
def test_attention_by_copies(env, shape, sizes, dt, form):  # noqa: F811
    """Keys and values rounded to 16 bits (u each) against 64 bits, whatever the sizes of their scales.  A score is off by u scale sum |q k|,
    e for the row's largest, and its weight by exp(2 e) - 1; values by u; P by u and 2^-12 for fp32; the result by u.  In fp16 elements
    below its normal range are off by 2^-25 where the head's largest is 2^-10 or more: 2^-15 of that; and P, whose largest is 1 or more, by
    2^-25 a key."""
    torch, ww = env
    B, Lq, Lk, Hq, Hk, D = shape
    t, u = _type(torch, dt), U[dt]
    q = _randn(torch, (B, Lq, Hq, D), 1, t)
    kept = _caches(torch, B, Lk, Hk, D, 2)
    kept[2], kept[3] = kept[2] * 20 * sizes[0], kept[3] * 20 * sizes[1]
    scale = sizes[2] / (sizes[0] * 42 * math.sqrt(D))
    keep = torch.ones((B, Lk), device="cuda", dtype=torch.bool)
    lens = mask = table = None
    if form != "plain":
        lens = torch.tensor([(Lk, Lk // 3, 0, 1, Lk + 5)[b % 5] for b in range(B)], device="cuda", dtype=torch.int32)
        g = torch.Generator(device="cuda").manual_seed(3)
        mask = torch.rand((B, Lk), generator=g, device="cuda") >= 0.3
        keep = mask & (torch.arange(Lk, device="cuda")[None] < lens[:, None])
        other = torch.where(torch.rand((B, 1, Lk), generator=g, device="cuda") < 0.5, math.nan, 1e30)
        for i in range(2):  # what masked places hold does not matter
            kept[2 + i] = torch.where(keep[:, None, :], kept[2 + i], other)
    if form == "biased":
        table = _randn(torch, (Hq, 32), 4, t)
    more = dict(k_lens=lens, key_mask=mask, bias_table=table, max_distance=64, q_offset=3)
    out, lse = ww.cross_attention_int8(q, *kept, scale=scale, return_lse=True, **more)
    assert torch.equal(out, ww.cross_attention_int8(q, *kept, scale=scale, **more))
    clean = kept[:2] + [torch.where(keep[:, None, :], c, 0.0) for c in kept[2:]]
    ref, rl, sums, most = _attention_reference(torch, ww, q, clean, keep, table, 64, True, 3, scale)
    size = [(clean[i].double() * clean[2 + i].double().transpose(1, 2)[..., None]).abs() for i in range(2)]
    size = [x.repeat_interleave(Hq // Hk, 2) for x in size]
    tiny = 2.0 ** -15 if dt == "f16" else 0.0
    top_k, top_v = (x.amax((1, 3)) for x in size)  # of each head
    e = scale * (u * torch.einsum("bihd,bjhd->bhij", q.double().abs(), size[0]).amax(-1) + tiny * q.double().abs().sum(-1).transpose(1, 2) * top_k[:, :, None])
    e = e.transpose(1, 2)[..., None]
    bound = (torch.expm1(2 * e) + 3 * u + 2.0 ** -12) * (1 + 4 * u) * sums + Lk * 2.0 ** -24 * most + tiny * top_v[:, None, :, None] + TINY[dt]
    if dt == "f16":  # a result of 65520 or more, half a step above the largest, is an infinity of fp16 (an item of one key: its value, up to 127 x 2048)
        beyond = (ref.abs() + bound >= 65520) & (out == torch.sign(ref) * math.inf)
        out = torch.where(beyond, ref, out.double())
    _within(out, ref, bound, "out")
    empty = torch.isinf(rl)
    assert torch.equal(torch.isinf(lse), empty) and not out.transpose(1, 2)[empty].any()
    if (~empty).any():
        assert ((lse.double() - rl).abs() - e[..., 0].transpose(1, 2))[~empty].max().item() <= 2.0 ** -11
    assert ww.device_error() == 0


def test_attention_by_copies_keeps_nonfinite_rows_apart(env):  # noqa: F811
    """A NaN scale in a valid place reaches its head's rows, and no others; scales that are large there do not change the others' bits."""
    torch, ww = env
    q = _randn(torch, (2, 140, 4, 64), 1, torch.float16)
    kept = _caches(torch, 2, 300, 2, 64, 2)
    plain = ww.cross_attention_int8(q, *kept)
    for which in (2, 3):
        changed = [c.clone() for c in kept]
        changed[which][0, 1, 77] = math.nan
        changed[which][1, 0, 5] = 3000.0 if which == 2 else 600.0
        out = ww.cross_attention_int8(q, *changed)
        assert out[0, :, 2:].isnan().all() and torch.isfinite(out[1]).all()
        assert torch.equal(out[0, :, :2], plain[0, :, :2]) and torch.equal(out[1, :, 2:], plain[1, :, 2:])


def test_attention_by_copies_with_the_least_memory(env):  # noqa: F811
    """A workspace of the copies alone: the same bits where fp16 holds the values."""
    torch, ww = env
    from whirlwind_trt_plugins_b200 import attention, layers
    q = _randn(torch, (1, 140, 4, 64), 1, torch.float16)
    kept = _caches(torch, 1, 900, 2, 64, 2)
    ref = ww.cross_attention_int8(q, *kept)
    n, st, out = 2 * 900 * 128 * 2, [900 * 128, 128, 64], torch.empty_like(q)
    ws = torch.empty(n, device="cuda", dtype=torch.uint8)
    a = attention._ATTN.pack(q.data_ptr(), kept[0].data_ptr(), kept[1].data_ptr(), out.data_ptr(), *[0] * 9, ws.data_ptr(), n, 140 * 256, 256, 64, *st, *st,
                             0, 0, 0, 1, 1, 140, 900, 4, 2, 64, 0, 128, 1, 0, 0.125)
    a += layers._SCALES.pack(kept[2].data_ptr(), kept[3].data_ptr(), 1800, 900, 1800, 900)
    assert layers._lib.ww_cross_attention_int8(a, torch.cuda.current_stream().cuda_stream) == 0
    # keys in other parts: either result is within P's and its own rounding (u each) and 2^-12 of the values' largest
    most = (kept[1].double() * kept[3].double().transpose(1, 2)[..., None]).abs().max()
    assert (out.double() - ref.double()).abs().max() <= 2 * (2 * U["f16"] + 2.0 ** -12) * most


# ---------------------------------------------------------------- together

def test_dispatch_modes_see_the_outputs(env):  # noqa: F811
    """A mode that watches torch's calls (a memory counter, say) sees the tensors that the operators allocate, and the bits are the same."""
    from torch.utils._python_dispatch import TorchDispatchMode
    torch, ww = env
    x, w = _randn(torch, (8, 64), 1, torch.float16), _randn(torch, (64,), 2, torch.float16)
    q = _randn(torch, (1, 4, 2, 64), 3, torch.float16)
    kv = _randn(torch, (1, 300, 2, 64), 4, torch.float16)
    wq, ws = ww.quantize_tokens(_randn(torch, (32, 64), 5, torch.float16))
    kept = [torch.empty((1, 300, 2, 64), device="cuda", dtype=torch.int8) for _ in range(2)] + [torch.empty((1, 2, 300), device="cuda") for _ in range(2)]
    ww.quantize_kv(kv, kv, *kept)
    angle = torch.rand((300, 32), device="cuda")
    calls = [lambda: ww.layer_norm(x, w, return_stats=True), lambda: ww.layer_norm_int8(x, w), lambda: (ww.int8_linear(x, wq, ws),),
             lambda: ww.cross_attention(q, kv, kv, return_lse=True), lambda: ww.cross_attention_int8(q, *kept, return_lse=True),
             lambda: ww.qk_norm_rope(q, kv, w, w, angle.cos(), angle.sin()), lambda: ww.dequantize_kv(*kept)]

    class Watch(TorchDispatchMode):
        def __init__(self):
            super().__init__()
            self.seen = []

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            out = func(*args, **(kwargs or {}))
            if isinstance(out, torch.Tensor):
                self.seen.append(out)  # alive, so that no other one is in its place
            return out

    for call in calls:
        plain = call()
        with Watch() as watch:
            got = call()
        places = {t.untyped_storage().data_ptr() for t in watch.seen}
        assert all(t.untyped_storage().data_ptr() in places for t in got)
        assert all(torch.equal(a, b) for a, b in zip(got, plain))


def test_copies_and_far_rows_captured(env):  # noqa: F811
    """Attention by copies (three kernels behind one another) and a norm whose rows turn far from zero, captured twice and replayed at once on
    two streams on changed inputs: the bits of eager calls."""
    torch, ww = env
    x = [_randn(torch, (700, 264), s, torch.float16) for s in (1, 2)]
    q = [_randn(torch, (2, 140, 4, 64), s, torch.float16) for s in (3, 4)]
    kept = [_caches(torch, 2, n, 2, 64, n) for n in (900, 3000)]
    lens = torch.tensor([900, 333], device="cuda", dtype=torch.int32)
    step = lambda i: (ww.layer_norm(x[i]), ww.cross_attention_int8(q[i], *kept[i], k_lens=lens))  # noqa: E731
    for i in (0, 1):
        step(i)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for i in (0, 1):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(i))
        graphs.append(g)
    x[0][::3] = 7.0
    kept[0][2][1] *= 2.0 ** 20
    kept[1][3][0] *= 2.0 ** -30
    lens.copy_(torch.tensor([17, 900], dtype=torch.int32))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(3):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for i in (0, 1):
        assert all(torch.equal(a, b) for a, b in zip(outs[i], step(i)))
    assert not outs[0][0][::3].any() and all(torch.isfinite(o[1]).all() for o in outs)
    assert ww.device_error() == 0
