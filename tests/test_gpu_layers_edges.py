"""The 8-bit layer operators at the edges of what they take, on the GPU against plain
implementations in 64 bits; tolerances count roundings as in test_gpu_layers.py."""
import math

import pytest
from test_gpu_layers import F, TINY, U, _randn, _type, _weights, _within, env  # noqa: F401

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
