"""ww_layer_norm with its gradient, ww_int8_matmul, the caches in 8 bits and
ww_cross_attention_int8 on the GPU against plain implementations in 64 bits (the
reference library has no such ops; their formulas are the specification).

Tolerances, per value; u = 2^-11 (fp16), 2^-8 (bf16), 2^-24 (fp32) is a type's unit
roundoff:

* layer norm: one rounding of the result (u |y|) and fp32 arithmetic, 2^-20 of the
  magnitudes that enter a value, a normalised value's being (|x| + mean |x|) rstd; sums
  over rows: 2^-18 of the magnitudes (up to 60 additions in a row at 2^-24);
* 8 bits: whole numbers and scales of rows are compared with the same fp32 operations
  on the host, bit for bit; a normalised row is within half a step of its exact value
  and the fp32 term above;
* products: three fp32 roundings and the result's: 2^-22 (|sum xs ws| + |b|) + u |y|;
* attention on 8-bit values: P once to fp16 (2^-11) and the result once to its type,
  2^-12 for fp32 scores and exponentials: (2^-11 + 2^-12 + u) sum P |v|; and where P falls
  below fp16's normal range half a subnormal step, 2^-25, of weights whose largest is
  2^6 or more: 2^-31 of the row's largest P |v| for each key;
* plus half a subnormal step of an fp16 result (2^-25)."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8, "f32": 2.0 ** -24}
TINY = {"f16": 2.0 ** -25, "bf16": 0.0, "f32": 0.0}
F = 2.0 ** -20


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
    import torch
    assert bool(torch.isfinite(got).all()), f"{what}: not finite"
    d = (got.double() - ref).abs() - bound
    assert got.numel() == 0 or d.max().item() <= 0, f"{what}: {d.max().item():.3e} over its bound"


# ---------------------------------------------------------------- layer norm

# every form: 4 to 32 lanes a row and 1 to 4 pieces a lane, blocks of 2 and 4 pieces, rows of single values (odd
# widths), rows beyond a block's registers; one row and one value
NORMS = [(1, 8), (3, 32), (1000, 64), (77, 128), (513, 256), (40, 320), (33, 512), (9, 704), (2000, 1024), (5, 1032), (6, 4096),
         (4, 8192), (3, 9000), (2, 20000), (3, 32776), (1, 1), (7, 2), (50, 17), (300, 129), (6, 511), (129, 1337), (3, 5001),
         (2, 16389), (1, 40001), (0, 64), (3001, 33), (1999, 251), (700, 505), (2500, 1001), (900, 2047), (301, 8191)]


def _norm_reference(torch, h, w, b, eps):
    hd = h.double()
    mean = hd.mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt((hd - mean).pow(2).mean(-1, keepdim=True) + eps)
    xh = (hd - mean) * rstd
    mag = (hd.abs() + hd.abs().mean(-1, keepdim=True)) * rstd
    y = xh if w is None else xh * w.double() + (0 if b is None else b.double())
    bound = mag if w is None else mag * w.double().abs() + (0 if b is None else b.double().abs())
    return y, bound, mean, rstd, xh, mag


@pytest.mark.parametrize("shape", NORMS)
@pytest.mark.parametrize("dt", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("form", ["plain", "affine", "residual"])
def test_layer_norm_and_gradient(env, shape, dt, form):
    torch, ww = env
    t, u, (rows, n) = _type(torch, dt), U[dt], shape
    x = _randn(torch, shape, 1, t, 2.0) + _randn(torch, (n,), 2, t)
    w = b = r = None
    if form != "plain":
        w, b = _randn(torch, (n,), 3, t) + 1, _randn(torch, (n,), 4, t)
    if form == "residual":
        r = _randn(torch, shape, 5, t)
    eps = 1e-5
    y, *more = ww.layer_norm(x, w, b, eps, residual=r, return_stats=True)
    mean, rstd = more[-2:]
    h = x
    if r is not None:
        h = more[0]
        assert torch.equal(h, x + r)
    ref, mag, m, rs, xh, xa = _norm_reference(torch, h, w, b, eps)
    _within(y, ref, u * ref.abs() + F * mag + TINY[dt], "y")
    _within(mean, m[:, 0], F * h.double().abs().mean(-1), "mean")
    _within(rstd, rs[:, 0], F * rs[:, 0] * (1 + h.double().abs().mean(-1) * rs[:, 0]), "rstd")
    dy = _randn(torch, shape, 6, t)
    ds = _randn(torch, shape, 7, t) if r is not None else None
    got = ww.layer_norm_backward(dy, h, w, mean, rstd, dsum=ds)
    again = ww.layer_norm_backward(dy, h, w, mean, rstd, dsum=ds)
    assert all(a is None or torch.equal(a, c) for a, c in zip(got, again))  # sums in a fixed order
    g = dy.double() if w is None else dy.double() * w.double()
    dx = rs * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True))
    mag = rs * (g.abs() + g.abs().mean(-1, keepdim=True) + xa * (g.abs() * xa).mean(-1, keepdim=True))
    if ds is not None:
        dx, mag = dx + ds.double(), mag + ds.double().abs()
    _within(got[0], dx, u * dx.abs() + F * mag + TINY[dt], "dx")
    if w is None:
        assert got[1] is None and got[2] is None
        return
    dw, db = (dy.double() * xh).sum(0), dy.double().sum(0)
    _within(got[1], dw, u * dw.abs() + 4 * F * (dy.double().abs() * xa).sum(0) + TINY[dt], "dweight")
    _within(got[2], db, u * db.abs() + 4 * F * dy.double().abs().sum(0) + TINY[dt], "dbias")


def test_layer_norm_gradient_is_the_differences(env):
    """fp32 gradients against central differences of the 64-bit formula."""
    torch, ww = env
    x, w, b = _randn(torch, (3, 12), 1, torch.float32), _randn(torch, (12,), 2, torch.float32), _randn(torch, (12,), 3, torch.float32)
    dy = _randn(torch, (3, 12), 4, torch.float32)
    _, mean, rstd = ww.layer_norm(x, w, b, return_stats=True)
    got = ww.layer_norm_backward(dy, x, w, mean, rstd)
    loss = lambda x, w, b: (torch.nn.functional.layer_norm(x, (12,), w, b, 1e-5) * dy.double()).sum()  # noqa: E731
    args, step = [t.double() for t in (x, w, b)], 1e-5
    for k in range(3):
        for i in range(args[k].numel()):
            moved = []
            for s in (step, -step):
                a = [t.clone() for t in args]
                a[k].view(-1)[i] += s
                moved.append(loss(*a))
            assert abs((moved[0] - moved[1]).item() / (2 * step) - got[k].view(-1)[i].item()) < 1e-5


@pytest.mark.parametrize("n", [256, 255])
def test_layer_norm_strides_and_empty_sums(env, n):
    torch, ww = env
    wide = _randn(torch, (6, 5, 2 * n), 1, torch.bfloat16)
    x, w, b = wide[..., n:], _randn(torch, (n,), 2, torch.bfloat16), _randn(torch, (n,), 3, torch.bfloat16)
    y, mean, rstd = ww.layer_norm(x, w, b, return_stats=True)
    assert torch.equal(y, ww.layer_norm(x.contiguous(), w, b)) and mean.shape == (6, 5)
    dy = _randn(torch, (30, n), 4, torch.bfloat16)[:1].expand(30, n).view(6, 5, n)  # one row for all
    got = ww.layer_norm_backward(dy, x, w, mean, rstd)
    ref = ww.layer_norm_backward(dy.contiguous(), x.contiguous(), w, mean, rstd)
    assert all(torch.equal(a, c) for a, c in zip(got, ref))
    none = x[:0].contiguous()
    dx, dw, db = ww.layer_norm_backward(none, none, w, mean[:0].contiguous(), rstd[:0].contiguous())
    assert dx.shape == none.shape and not dw.any() and not db.any()
    assert ww.layer_norm(none, w, b).shape == none.shape


@pytest.mark.parametrize("off", [1, 3, 8])
@pytest.mark.parametrize("n", [100, 600, 1336])
def test_layer_norm_rows_that_begin_anywhere(env, n, off):
    """Rows off 16 bytes by themselves, or all tensors alike, have the bits of the same rows elsewhere."""
    torch, ww = env
    rows = 700
    x, dy, r = (_randn(torch, (rows, n), s, torch.float16) for s in (1, 2, 3))
    w, b = _randn(torch, (n,), 4, torch.float16), _randn(torch, (n,), 5, torch.float16)

    def moved(t):
        m = torch.empty(t.numel() + off, device="cuda", dtype=t.dtype)[off:].view(t.shape)
        return m.copy_(t)

    y, h, mean, rstd = ww.layer_norm(x, w, b, residual=r, return_stats=True)
    got = ww.layer_norm(moved(x), moved(w), moved(b), residual=moved(r), return_stats=True)
    assert torch.equal(got[1], h)
    ref, mag, *_ = _norm_reference(torch, h, w, b, 1e-5)
    _within(got[0], ref, U["f16"] * ref.abs() + F * mag + TINY["f16"], "y")
    one = ww.layer_norm_backward(dy, h, w, mean, rstd, dsum=r)
    two = ww.layer_norm_backward(moved(dy), moved(h), moved(w), mean, rstd, dsum=moved(r))
    for a, c in zip(one, two):  # in another order of the sums
        assert (a.float() - c.float()).abs().max() <= 2.0 ** -8 * a.float().abs().max()


def test_layer_norm_large_mean_and_nonfinite(env):
    """A mean of thousands of deviations costs no digits of the variance; a NaN or an infinity stays in its row."""
    torch, ww = env
    x = (_randn(torch, (16, 1000), 1, torch.float32) + 4096).contiguous()
    ref, mag, *_ = _norm_reference(torch, x, None, None, 1e-5)
    _within(ww.layer_norm(x), ref, F * mag, "y")
    x = _randn(torch, (16, 256), 2, torch.float16)
    x[3, 17], x[5, 0] = math.nan, math.inf
    y = ww.layer_norm(x)
    bad = torch.tensor([i in (3, 5) for i in range(16)], device="cuda")
    assert torch.equal(y.isnan().all(-1), bad) and torch.equal(y.isnan().any(-1), bad)
    q, scale = ww.layer_norm_int8(x)
    assert torch.equal(scale.isnan(), bad)
    y = ww.layer_norm(torch.full((4, 64), 3.0, device="cuda"))  # rows of one value: 0 / sqrt(eps)
    assert not y.any()


def test_layer_norm_autograd(env):
    torch, ww = env
    x, r = (_randn(torch, (4, 9, 64), s, torch.float32).requires_grad_(True) for s in (1, 2))
    w, b = (_randn(torch, (64,), s, torch.float32).requires_grad_(True) for s in (3, 4))
    y, h = ww.layer_norm_autograd(x, w, b, 1e-5, r)
    loss = (y * y).sum() + (h * h * h).sum()
    got = torch.autograd.grad(loss, (x, r, w, b))
    leaves = [t.detach().double().requires_grad_(True) for t in (x, r, w, b)]
    hd = leaves[0] + leaves[1]
    yd = torch.nn.functional.layer_norm(hd, (64,), leaves[2], leaves[3], 1e-5)
    ref = torch.autograd.grad((yd * yd).sum() + (hd * hd * hd).sum(), leaves)
    for g, e in zip(got, ref):
        assert (g.double() - e).abs().max() <= 1e-4 * e.abs().max()
    # only the sum, or only the result, is used; transposed incoming gradients; a second derivative raises
    y, h = ww.layer_norm_autograd(x, w, b, 1e-5, r)
    assert torch.equal(torch.autograd.grad(h.sum(), x)[0], torch.ones_like(x))
    y = ww.layer_norm_autograd(x, w)
    torch.autograd.grad(y.transpose(0, 1).contiguous().sum(), x)
    g, = torch.autograd.grad((ww.layer_norm_autograd(x, w) ** 2).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), x)


def test_layer_norm_autograd_of_one_result(env):
    """Gradients where only the sum or only the normed rows are used: zeros for what does not reach the loss."""
    torch, ww = env
    x, r = (_randn(torch, (5, 40), s, torch.float32).requires_grad_(True) for s in (1, 2))
    w, b = (_randn(torch, (40,), s, torch.float32).requires_grad_(True) for s in (3, 4))
    e = _randn(torch, (5, 40), 5, torch.float32)
    got = torch.autograd.grad((ww.layer_norm_autograd(x, w, b, 1e-5, r)[1] * e).sum(), (x, r, w, b))
    assert torch.equal(got[0], e) and torch.equal(got[1], e) and not got[2].any() and not got[3].any()
    y, h = ww.layer_norm_autograd(x, w, b, 1e-5, r)
    got = torch.autograd.grad((y * e).sum(), (x, r, w, b))
    _, mean, rstd = ww.layer_norm(h.detach(), w.detach(), b.detach(), return_stats=True)
    ref = ww.layer_norm_backward(e, h.detach(), w.detach(), mean, rstd)
    assert all(torch.equal(g, f) for g, f in zip(got, (ref[0], *ref)))


@pytest.mark.parametrize("shape", [(15000, 320), (4000, 504), (13001, 712), (9000, 1024), (9001, 1048), (2500, 4096), (1500, 8192)])
@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("dsum", [False, True])
def test_layer_norm_gradient_of_many_rows(env, shape, dt, dsum):
    """Many rows for each lane and block, of strided inputs: their own sums, and the same bits on every run."""
    torch, ww = env
    rows, n = shape
    t, u = _type(torch, dt), U[dt]
    w, dy = _randn(torch, (n,), 1, t), _randn(torch, (rows, n), 2, t)
    x = _randn(torch, (rows, n + 16), 3, t)[:, :n]
    ds = _randn(torch, (rows, 2 * n), 4, t)[:, n:] if dsum else None
    _, mean, rstd = ww.layer_norm(x, w, return_stats=True)
    got = ww.layer_norm_backward(dy, x, w, mean, rstd, dsum=ds)
    assert all(torch.equal(a, b) for a, b in zip(got, ww.layer_norm_backward(dy, x, w, mean, rstd, dsum=ds)))
    xh = (x.double() - mean.double()[:, None]) * rstd.double()[:, None]
    g = dy.double() * w.double()
    s2 = (g * xh).mean(-1, keepdim=True)
    ref = rstd.double()[:, None] * (g - g.mean(-1, keepdim=True) - xh * s2)
    mag = rstd.double()[:, None] * (g.abs() + g.abs().mean(-1, keepdim=True) + xh.abs() * (g * xh).abs().mean(-1, keepdim=True))
    if dsum:
        ref, mag = ref + ds.double(), mag + ds.double().abs()
    _within(got[0], ref, u * ref.abs() + 2.0 ** -18 * mag, "dx")
    for a, terms in ((got[1], dy.double() * xh), (got[2], dy.double())):
        _within(a, terms.sum(0), u * terms.sum(0).abs() + 2.0 ** -18 * terms.abs().sum(0), "sums")
    assert ww.device_error() == 0


@pytest.mark.parametrize("shape", [(9001, 1048), (2500, 4096), (1500, 8200), (700, 16384)])
@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("affine", [False, True])
def test_layer_norm_of_many_long_sums(env, shape, dt, affine):
    """Many long rows of strided inputs and their residuals: the sums, the result and its 8-bit form row by row."""
    torch, ww = env
    rows, n = shape
    if dt == "f32" and n > 8192:
        n //= 2
    t, u = _type(torch, dt), U[dt]
    x, r = _randn(torch, (rows, n + 8), 1, t)[:, 8:], _randn(torch, (rows, n), 2, t)
    w, b = (_randn(torch, (n,), 3, t) + 1, _randn(torch, (n,), 4, t)) if affine else (None, None)
    y, h, mean, rstd = ww.layer_norm(x, w, b, residual=r, return_stats=True)
    assert torch.equal(h, x + r)
    ref, mag, m, rs, *_ = _norm_reference(torch, h, w, b, 1e-5)
    _within(y, ref, u * ref.abs() + F * mag, "y")
    _within(mean, m[:, 0], F * h.double().abs().mean(-1), "mean")
    _within(rstd, rs[:, 0], F * rs[:, 0] * (1 + h.double().abs().mean(-1) * rs[:, 0]), "rstd")
    q, scale, total = ww.layer_norm_int8(x, w, b, residual=r)
    assert torch.equal(total, h)
    _within(q.double() * scale.double()[:, None], ref, 0.5 * scale.double()[:, None] * (1 + F) + 2 * F * mag.amax(-1, keepdim=True), "8 bits")
    few = ww.layer_norm(x[:40], w, b, residual=r[:40])
    assert (few[0].double() - y[:40].double()).abs().max() <= 2 * u * y[:40].double().abs().max()
    assert ww.device_error() == 0


@pytest.mark.parametrize("n", [2049, 2050, 5001, 8191, 10239, 10240])
@pytest.mark.parametrize("off", [0, 1])
@pytest.mark.parametrize("dt", ["f16", "bf16", "f32"])
def test_layer_norm_of_many_long_odd_rows(env, n, off, dt):
    """Rows in pairs: every other one begins off their grid, all with `off`; several rows a block; what lies next to them counts for nothing."""
    torch, ww = env
    t, u, rows = _type(torch, dt), U[dt], 700

    def make(seed, pitch=n):  # rows `off` values behind 16 bytes, NaN around them
        flat = torch.full((rows * pitch + 16,), math.nan, device="cuda", dtype=t)
        x = flat[off:off + rows * pitch].view(rows, pitch)[:, :n]
        return x.copy_(_randn(torch, (rows, n), seed, t))

    x, dy, ds, w, b = make(1), make(2), make(3, n + 2 * (n % 3)), _randn(torch, (n + 1,), 4, t)[1:], _randn(torch, (n + 1,), 5, t)[1:]
    y = torch.full((rows * n + 16,), 7.0, device="cuda", dtype=t)
    out = y[off:off + rows * n].view(rows, n)
    got, mean, rstd = ww.layer_norm(x, w, b, return_stats=True, out=out)
    ref, mag, m, rs, xh, xa = _norm_reference(torch, x, w, b, 1e-5)
    _within(got, ref, u * ref.abs() + F * mag + TINY[dt], "y")
    assert torch.equal(y[:off], torch.full_like(y[:off], 7)) and torch.equal(y[off + rows * n:], torch.full_like(y[off + rows * n:], 7))
    q, scale = ww.layer_norm_int8(x, w, b)
    _within(q.double() * scale.double()[:, None], ref, 0.5 * scale.double()[:, None] * (1 + F) + 2 * F * mag.amax(-1, keepdim=True), "8 bits")
    qx, sx = ww.quantize_tokens(x)
    hq, hs, _ = _int8_host(x)
    assert np.array_equal(qx.cpu().numpy(), hq) and np.array_equal(sx.cpu().numpy(), hs)
    dx, dw, db = ww.layer_norm_backward(dy, x, w, mean, rstd, dsum=ds)
    g = dy.double() * w.double()
    dref = rs * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True)) + ds.double()
    dmag = rs * (g.abs() + g.abs().mean(-1, keepdim=True) + xa * (g.abs() * xa).mean(-1, keepdim=True)) + ds.double().abs()
    _within(dx, dref, u * dref.abs() + F * dmag + TINY[dt], "dx")
    for a, terms, size in ((dw, dy.double() * xh, dy.double().abs() * xa), (db, dy.double(), dy.double().abs())):
        _within(a, terms.sum(0), u * terms.sum(0).abs() + 4 * F * size.sum(0) + TINY[dt], "sums")
    again = ww.layer_norm_backward(dy, x, w, mean, rstd, dsum=ds)
    assert all(torch.equal(p, r) for p, r in zip((dx, dw, db), again))


@pytest.mark.parametrize("n", [24, 40, 60])
@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_layer_norm_gradient_of_large_equal_values(env, n, dt):
    """Rows of one large value: xh is 0 although mean rstd passes fp32's range, and so it is in lanes beyond a row."""
    torch, ww = env
    t = _type(torch, dt)
    x, w, dy = torch.full((9, n), 2.0 ** 122, device="cuda", dtype=t), _randn(torch, (n,), 1, t), _randn(torch, (9, n), 2, t)
    mean, rstd = torch.full((9,), 2.0 ** 122, device="cuda"), torch.full((9,), 316.0, device="cuda")
    dx, dw, db = ww.layer_norm_backward(dy, x, w, mean, rstd)
    g = dy.double() * w.double()
    ref = 316 * (g - g.mean(-1, keepdim=True))
    _within(dx, ref, U[dt] * ref.abs() + 316 * 2.0 ** -18 * (g.abs() + g.abs().mean(-1, keepdim=True)), "dx")
    assert not dw.any()
    _within(db, dy.double().sum(0), U[dt] * dy.double().sum(0).abs() + 2.0 ** -18 * dy.double().abs().sum(0), "dbias")


def test_outputs_apart_from_inputs(env):
    torch, ww = env
    x = torch.zeros((8, 64), device="cuda", dtype=torch.float16)
    wq, ws = ww.quantize_tokens(torch.ones((64, 64), device="cuda"))
    kept = [torch.zeros((1, 4, 2, 32), device="cuda", dtype=torch.int8)] * 2 + [torch.zeros((1, 2, 4), device="cuda")] * 2
    q = x.view(1, 8, 2, 32)
    both = torch.zeros((16, 64), device="cuda", dtype=torch.float16)
    for call in (lambda: ww.layer_norm(x, out=x), lambda: ww.layer_norm(both[:8], residual=both[4:12], out=both[8:]),
                 lambda: ww.int8_linear(x, wq, ws, out=x), lambda: ww.cross_attention_int8(q, *kept, out=q)):
        with pytest.raises(ValueError, match="shares memory"):
            call()
    assert ww.layer_norm(both[:8], out=both[8:]).data_ptr() == both[8:].data_ptr()


# ---------------------------------------------------------------- 8 bits

def _int8_host(x):
    """Whole numbers and scales of rows by the same fp32 operations on the host."""
    x = x.float().cpu().numpy()
    top = np.abs(x).max(-1, keepdims=True).astype(np.float32)
    with np.errstate(all="ignore"):
        small, bad = top < np.float32(2.0 ** -119), ~np.isfinite(top)
        inv = np.where(small | bad, np.float32(0), np.float32(1) / top * np.float32(127)).astype(np.float32)
        q = np.rint((np.where(np.isfinite(x), x, 0) * inv).astype(np.float32)).astype(np.int8)
        scale = np.where(small, np.float32(0), np.where(bad, np.float32(np.nan), top / np.float32(127)))
    return q, scale[..., 0].astype(np.float32), bad[..., 0]


@pytest.mark.parametrize("shape", [(1, 1), (5, 16), (3, 4, 48), (1000, 256), (7, 1000), (2, 1337), (1, 9001), (3, 40000), (2, 40001)])
@pytest.mark.parametrize("dt", ["f16", "bf16", "f32"])
def test_quantize_tokens(env, shape, dt):
    torch, ww = env
    x = _randn(torch, shape, 1, _type(torch, dt), 3.0)
    x.view(-1, shape[-1])[0] *= 2.0 ** -10
    q, scale = ww.quantize_tokens(x)
    hq, hs, _ = _int8_host(x)
    assert q.shape == x.shape and q.stride(-2 if len(shape) > 1 else 0) % 16 == 0
    assert np.array_equal(q.cpu().numpy(), hq) and np.array_equal(scale.cpu().numpy(), hs)


def test_quantize_tokens_extremes(env):
    torch, ww = env
    x = torch.zeros((9, 40), device="cuda")
    x[1], x[2, 3], x[3, 5], x[4, 7] = 2.0 ** -119, 2.0 ** -130, math.inf, math.nan
    x[5, 1], x[6, :2] = 3e38, torch.tensor([1.0, -1.0])
    x[7, :3] = torch.tensor([127.0, 0.5, 1.5])  # ties go to the even number
    x[8] = 2.0 ** -120
    q, scale = ww.quantize_tokens(x)
    hq, hs, bad = _int8_host(x)
    good = ~bad
    assert np.array_equal(q.cpu().numpy()[good], hq[good])
    assert np.array_equal(scale.cpu().numpy(), hs, equal_nan=True)
    assert q[7, :3].tolist() == [127, 0, 2] and scale[2] == 0 and scale[8] == 0 and scale[3].isnan()


@pytest.mark.parametrize("shape", [(1, 64), (9, 1024), (300, 320), (5, 1337), (3, 6000), (2, 40001)])
@pytest.mark.parametrize("dt", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("residual", [False, True])
def test_layer_norm_int8(env, shape, dt, residual):
    torch, ww = env
    t = _type(torch, dt)
    x, w, b = _randn(torch, shape, 1, t), _randn(torch, shape[-1:], 2, t) + 1, _randn(torch, shape[-1:], 3, t)
    r = _randn(torch, shape, 4, t) if residual else None
    q, scale, *more = ww.layer_norm_int8(x, w, b, residual=r)
    h = more[0] if residual else x
    assert not residual or torch.equal(h, x + r)
    ref, mag, *_ = _norm_reference(torch, h, w, b, 1e-5)
    top = ref.abs().amax(-1)
    err = F * mag.amax(-1)
    assert ((scale.double() * 127 - top).abs() <= err + 2.0 ** -22 * top).all()
    assert (q.abs().amax(-1) == 127).all()
    _within(q.double() * scale.double()[..., None], ref, (0.5 + 2.0 ** -12) * scale.double()[..., None] + 2 * F * mag.amax(-1, keepdim=True), "q")


# (M, K, N): few tokens (to 16, within shared memory and beyond), tiles of 64, 128 and 256 channels, partial tiles in every
# direction, K below and off a stage, rows of the output off 16 bytes, several tiles a block
PRODUCTS = [(1, 1, 1), (1, 64, 16), (1, 4096, 100), (3, 100, 33), (8, 1000, 257), (9, 130, 48), (16, 4096, 64), (16, 8192, 40), (17, 64, 8), (2, 9000, 700), (5, 20000, 30), (12, 4096, 1000), (30, 1000, 4099), (64, 512, 520), (65, 3000, 128), (128, 8192, 264), (20, 131, 20000), (9, 20000, 136),
            (1, 64, 70001), (4, 33, 70000), (1, 16, 263000), (20, 128, 64), (24, 640, 100), (32, 1025, 72), (33, 384, 96), (40, 900, 130),
            (100, 33, 200), (128, 128, 64), (129, 129, 65), (300, 1000, 1111), (1000, 256, 768), (2500, 300, 520), (5000, 144, 513),
            (4096, 512, 1024), (700, 2048, 4104), (0, 64, 64), (5, 64, 0)]


def _weights(torch, ww, n, k, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    pitch = (k + 15) // 16 * 16
    w = torch.randint(-128, 128, (n, pitch), generator=g, device="cuda", dtype=torch.int8)[:, :k]  # what lies behind a row does not matter
    return w, torch.rand((n,), generator=g, device="cuda") * 0.01 + 1e-4


@pytest.mark.parametrize("shape", PRODUCTS)
@pytest.mark.parametrize("dt", ["f16", "bf16", "f32"])
def test_products(env, shape, dt):
    torch, ww = env
    M, K, N = shape
    t, u = _type(torch, dt), U[dt]
    w, ws = _weights(torch, ww, N, K, 1)
    x = _randn(torch, (M, K), 2, t)
    bias = _randn(torch, (N,), 3, t) if N % 2 == 0 else None
    xq, xs = ww.quantize_tokens(x)
    got = ww.int8_matmul(xq, xs, w, ws, bias, dtype=t)
    acc = xq.double() @ w.double().t()
    one = acc * xs.double()[:, None] * ws.double()
    ref = one if bias is None else one + bias.double()
    mag = one.abs() + (0 if bias is None else bias.double().abs())
    _within(got, ref, u * ref.abs() + 2.0 ** -22 * mag + TINY[dt], "out")
    assert torch.equal(ww.int8_linear(x, w, ws, bias), got)  # brought to 8 bits inside the call: the same numbers
    assert ww.device_error() == 0


def test_products_of_the_largest_numbers(env):
    """Sums of equal products at the largest magnitudes stay exact; -128 too."""
    torch, ww = env
    for M, K, N in ((2, 131071, 16), (200, 131071, 72)):
        xq = torch.full((M, (K + 15) // 16 * 16), -128, device="cuda", dtype=torch.int8)[:, :K]
        w = torch.full((N, (K + 15) // 16 * 16), -128, device="cuda", dtype=torch.int8)[:, :K]
        got = ww.int8_matmul(xq, torch.ones(M, device="cuda"), w, torch.ones(N, device="cuda"), dtype=torch.float32)
        assert (got == float(np.float32(K * 16384))).all()


def test_products_layouts_and_nonfinite(env):
    torch, ww = env
    w, ws = _weights(torch, ww, 96, 80, 1)
    wide = _randn(torch, (2, 50, 200), 2, torch.bfloat16)
    for x in (wide[..., 16:96], wide[..., 3:83], wide[:, :1, :80].expand(2, 1, 80)):  # on and off 16 bytes
        assert torch.equal(ww.int8_linear(x, w, ws), ww.int8_linear(x.contiguous(), w, ws))
    x = _randn(torch, (300, 80), 3, torch.float16)
    x[7, 3], x[200, 0], x[201] = math.nan, math.inf, 0
    y = ww.int8_linear(x, w, ws)
    assert torch.equal(y.isnan().all(-1), torch.tensor([i in (7, 200) for i in range(300)], device="cuda"))
    assert not y[201].any() and torch.equal(y.isnan().any(-1), y.isnan().all(-1))
    out = torch.full((300, 97), 5.0, device="cuda", dtype=torch.float16)
    with pytest.raises(ValueError):
        ww.int8_linear(x, w, ws, out=out[:, :96])


# ---------------------------------------------------------------- keys and values in 8 bits

def _caches(torch, B, places, H, D, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    c = [torch.randint(-127, 128, (B, places, H, D), generator=g, device="cuda", dtype=torch.int8) for _ in range(2)]
    return c + [torch.rand((B, H, places), generator=g, device="cuda") * 0.05 for _ in range(2)]


@pytest.mark.parametrize("shape", [(1, 1, 1, 1, 16), (2, 7, 20, 3, 48), (3, 33, 33, 5, 64), (2, 100, 77, 8, 128), (1, 1000, 2000, 2, 32),
                                   (4, 0, 9, 2, 32), (2, 5, 300, 1, 112)])
@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("ragged", [False, True])
def test_cache_written_and_read(env, shape, dt, ragged):
    torch, ww = env
    B, L, places, H, D = shape
    t = _type(torch, dt)
    k, v = _randn(torch, (B, L, H, D), 1, t), _randn(torch, (B, L, H, D), 2, t, 30.0)
    start = lens = None
    if ragged:  # items that begin before the cache, within it, and end behind it
        start = torch.tensor([(-2, places - 3, 0, 5)[b % 4] for b in range(B)], device="cuda", dtype=torch.int32)
        lens = torch.tensor([(L, L + 9, 0, -1)[b % 4] for b in range(B)], device="cuda", dtype=torch.int32)
    kept = _caches(torch, B, places, H, D, 3)
    want = [c.clone() for c in kept]
    for i, x in enumerate((k, v)):
        q, scale, _ = _int8_host(x) if L else (None, None, None)
        for b in range(B):
            at = 0 if start is None else int(start[b])
            n = L if lens is None else min(L, int(lens[b]))
            for row in range(max(0, n)):
                if 0 <= at + row < places:
                    want[i][b, at + row] = torch.from_numpy(q[b, row]).cuda()
                    want[2 + i][b, :, at + row] = torch.from_numpy(scale[b, row]).cuda()
    ww.quantize_kv(k, v, *kept, start=start, lens=lens)
    assert all(torch.equal(a, c) for a, c in zip(kept, want))
    valid = torch.tensor([(places, 0, 3, -4)[b % 4] for b in range(B)], device="cuda", dtype=torch.int32) if ragged else None
    got = ww.dequantize_kv(*kept, lens=valid, dtype=t)
    for i in range(2):
        ref = (kept[i].float() * kept[2 + i].transpose(1, 2)[..., None]).to(t)
        if valid is not None:
            ref[torch.arange(places, device="cuda")[None] >= valid[:, None]] = 0
        assert torch.equal(got[i], ref)


def test_cache_layouts(env):
    """Slices of one projection in, views of larger caches out, broadcast reads, places beyond 2^32 bytes."""
    torch, ww = env
    B, L, H, D = 2, 9, 4, 64
    qkv = _randn(torch, (B, L, 3, H, D), 1, torch.bfloat16)
    k, v = qkv[:, :, 1], qkv[:, :, 2]
    kept = _caches(torch, B, L, H, D, 2)
    ww.quantize_kv(k.contiguous(), v.contiguous(), *kept)
    big = _caches(torch, B + 1, 40, 2 * H, D, 3)
    views = [c[1:, 5:14, H:] for c in big[:2]] + [c[1:, H:, 5:14] for c in big[2:]]
    before = [c.clone() for c in big]
    ww.quantize_kv(k, v, *views)
    assert all(torch.equal(a, c) for a, c in zip(views, kept))
    for a, c in zip(big, before):  # nothing else was written
        same = a == c
        (same[1:, 5:14, H:] if a.dim() == 4 else same[1:, H:, 5:14]).fill_(True)
        assert same.all()
    one = [c[:1].expand(3, *c.shape[1:]) for c in kept]
    for a, c in zip(ww.dequantize_kv(*one), ww.dequantize_kv(*[c.contiguous() for c in one])):
        assert torch.equal(a, c)
    far = torch.empty(2 ** 32 + 2 ** 21, device="cuda", dtype=torch.int8)
    step = 2 ** 32 // 64  # place 64 starts 2^32 bytes behind place 0
    kc, vc = (far[o:].as_strided((1, 65, 1, 64), (0, step, 64, 1)) for o in (0, 1 << 20))
    scales = [torch.zeros((1, 1, 65), device="cuda") for _ in range(2)]
    x, y = _randn(torch, (1, 65, 1, 64), 5, torch.float16), _randn(torch, (1, 65, 1, 64), 6, torch.float16)
    near = _caches(torch, 1, 65, 1, 64, 7)
    ww.quantize_kv(x, y, kc, vc, *scales)
    ww.quantize_kv(x, y, *near)
    assert torch.equal(kc, near[0]) and torch.equal(vc, near[1])
    assert all(torch.equal(a, c) for a, c in zip(ww.dequantize_kv(kc, vc, *scales), ww.dequantize_kv(*near)))
    q = _randn(torch, (1, 1, 1, 64), 8, torch.float16)
    assert torch.equal(ww.cross_attention_int8(q, kc, vc, *scales), ww.cross_attention_int8(q, *near))


# ---------------------------------------------------------------- attention over them

def _buckets(ww, torch, Lq, Lk, offset, num, dist, bi):
    row = torch.tensor([ww.relative_position_bucket(r, num, dist, bi) for r in range(-(Lq - 1) - offset, Lk - offset)], device="cuda")
    return row[torch.arange(Lk, device="cuda")[None, :] - torch.arange(Lq, device="cuda")[:, None] + Lq - 1]


def _attention_reference(torch, ww, q, kept, keep, table, dist, bi, offset, scale):
    """out, lse, sum P |v| and the largest P |v| of each row, in 64 bits."""
    kd, vd = (kept[i].double() * kept[2 + i].double().transpose(1, 2)[..., None] for i in range(2))
    kd, vd = (torch.where(keep[:, :, None, None], x, 0.0) for x in (kd, vd))
    B, Lq, Hq, D = q.shape
    Hk, Lk = kd.shape[2], kd.shape[1]
    kd, vd = (x.repeat_interleave(Hq // Hk, 2) for x in (kd, vd))
    s = torch.einsum("bihd,bjhd->bhij", q.double(), kd) * scale
    if table is not None:
        t = table.double()
        t = torch.where(t <= float(torch.finfo(table.dtype).min), -math.inf, t)
        s = s + t[:, _buckets(ww, torch, Lq, Lk, offset, table.shape[1], dist, bi)]
    s = s.masked_fill(~keep[:, None, None, :], -math.inf)
    lse = torch.logsumexp(s, -1) if Lk else torch.full((B, Hq, Lq), -math.inf, device="cuda", dtype=torch.float64)
    p = torch.exp(s - torch.where(torch.isinf(lse), 0.0, lse)[..., None])
    out = torch.einsum("bhij,bjhd->bihd", p, vd)
    sums = torch.einsum("bhij,bjhd->bihd", p, vd.abs())
    most = torch.zeros((B, Lq, Hq, 1), device="cuda", dtype=torch.float64)
    if Lk:
        most = (p * vd.abs().amax(-1).transpose(1, 2)[:, :, None, :]).amax(-1).transpose(1, 2)[..., None]
    return out, lse, sums, most


# (B, Lq, Lk, Hq, Hk, D): single tokens, shared heads to 128 rows a key head, odd lengths, every head width, no keys
FEW = [(1, 1, 1, 1, 1, 16), (1, 1, 40, 8, 8, 32), (3, 1, 1500, 16, 4, 64), (2, 1, 9001, 32, 8, 128), (2, 5, 333, 6, 3, 48), (1, 3, 700, 12, 2, 80),
       (2, 2, 65, 32, 4, 128), (1, 1, 5000, 40, 2, 64), (1, 9, 515, 16, 2, 112), (2, 17, 100, 3, 1, 32), (1, 1, 257, 128, 1, 128),
       (200, 1, 70, 4, 4, 32), (1, 4, 0, 4, 2, 64), (2, 0, 8, 4, 2, 64), (1, 1, 30000, 2, 1, 64)]


@pytest.mark.parametrize("shape", FEW)
@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("form", ["plain", "masked", "biased"])
def test_attention_few_rows(env, shape, dt, form):
    torch, ww = env
    B, Lq, Lk, Hq, Hk, D = shape
    t, u = _type(torch, dt), U[dt]
    q = _randn(torch, (B, Lq, Hq, D), 1, t)
    kept = _caches(torch, B, Lk, Hk, D, 2)
    keep = torch.ones((B, Lk), device="cuda", dtype=torch.bool)
    lens = mask = table = None
    dist, bi, offset = 64, D % 32 == 0, Lk // 2
    if form != "plain":
        lens = torch.tensor([(Lk, Lk // 2, 0, 1, Lk + 5, -1)[b % 6] for b in range(B)], device="cuda", dtype=torch.int32)
        g = torch.Generator(device="cuda").manual_seed(3)
        mask = torch.rand((B, Lk), generator=g, device="cuda") >= 0.4
        mask[-1] = B == 1  # an item without keys
        keep = mask & (torch.arange(Lk, device="cuda")[None] < lens[:, None])
        for i in range(2):  # what masked places hold does not matter
            kept[2 + i].masked_fill_(~keep[:, None, :], math.nan)
    if form == "biased":
        table = _randn(torch, (Hq, 32), 4, t)
        table[:, 3] = float(torch.finfo(t).min)
    more = dict(k_lens=lens, key_mask=mask, bias_table=table, max_distance=dist, bidirectional=bi, q_offset=offset)
    out, lse = ww.cross_attention_int8(q, *kept, return_lse=True, **more)
    assert torch.equal(out, ww.cross_attention_int8(q, *kept, **more))
    clean = kept[:2] + [torch.nan_to_num(c) for c in kept[2:]]
    ref, rl, sums, most = _attention_reference(torch, ww, q, clean, keep, table, dist, bi, offset, 1 / math.sqrt(D))
    _within(out, ref, (2.0 ** -11 + 2.0 ** -12 + u) * sums + Lk * 2.0 ** -31 * most + TINY[dt], "out")
    empty = torch.isinf(rl)
    assert torch.equal(torch.isinf(lse), empty) and not out.transpose(1, 2)[empty].any()
    assert (lse.double() - rl)[~empty].abs().max().item() <= 2.0 ** -12 if (~empty).any() else True
    assert ww.device_error() == 0


@pytest.mark.parametrize("shape", [(2, 70, 300, 6, 3, 64), (1, 200, 1000, 8, 8, 128), (2, 33, 65, 8, 2, 32), (1, 500, 77, 2, 2, 48), (2, 130, 0, 1, 1, 64)])
@pytest.mark.parametrize("dt", ["f16", "bf16"])
def test_attention_many_rows(env, shape, dt):
    """More rows than 128 a key head: the attention of the keys and values read back, bit for bit."""
    torch, ww = env
    B, Lq, Lk, Hq, Hk, D = shape
    t = _type(torch, dt)
    q = _randn(torch, (B, Lq, Hq, D), 1, t)
    kept = _caches(torch, B, Lk, Hk, D, 2)
    lens = torch.tensor([(Lk, Lk // 3)[b % 2] for b in range(B)], device="cuda", dtype=torch.int32)
    mask = torch.rand((B, Lk), device="cuda") >= 0.2
    table = _randn(torch, (Hq, 16), 4, t)
    for more in ({}, dict(k_lens=lens, key_mask=mask, bias_table=table, q_offset=3)):
        got = ww.cross_attention_int8(q, *kept, return_lse=True, **more)
        ref = ww.cross_attention(q, *ww.dequantize_kv(*kept, dtype=t), return_lse=True, **more)
        assert all(torch.equal(a, c) for a, c in zip(got, ref))


def test_attention_scales_of_all_sizes(env):
    """Values' scales from 2^-60 to 2^40 next to one another, zeros among them: each row keeps its own precision."""
    torch, ww = env
    B, Lk, H, D = 4, 999, 2, 64
    q = _randn(torch, (B, 1, H, D), 1, torch.bfloat16)
    kept = _caches(torch, B, Lk, H, D, 2)
    g = torch.Generator(device="cuda").manual_seed(3)
    kept[3] = torch.exp2(torch.rand(kept[3].shape, generator=g, device="cuda") * 100 - 60)
    kept[3][1] = 0
    kept[3][2, :, ::2] = 0
    kept[3][3] = 2.0 ** -60  # one large value far from the others in score
    kept[2][3] = 0.05
    keep = torch.ones((B, Lk), device="cuda", dtype=torch.bool)
    ref, _, sums, most = _attention_reference(torch, ww, q, kept, keep, None, 0, True, 0, 0.125)
    out = ww.cross_attention_int8(q, *kept)
    _within(out, ref, (2.0 ** -11 + 2.0 ** -12 + 2.0 ** -8) * sums + Lk * 2.0 ** -31 * most, "out")
    assert not out[1].any() and out[3].any()


@pytest.mark.parametrize("factor", [2.0 ** -90, 2.0 ** -20, 2.0 ** 60])
def test_attention_queries_of_all_sizes(env, factor):
    """bf16 queries far outside fp16's range, with scales that bring the scores back."""
    torch, ww = env
    q = _randn(torch, (1, 1, 4, 64), 1, torch.float32)
    kept = _caches(torch, 1, 500, 2, 64, 2)
    keep = torch.ones((1, 500), device="cuda", dtype=torch.bool)
    qb = (q * factor).to(torch.bfloat16)
    ref, _, sums, most = _attention_reference(torch, ww, qb, kept, keep, None, 0, True, 0, 0.125 / factor)
    out = ww.cross_attention_int8(qb, *kept, scale=0.125 / factor)
    _within(out, ref, (2.0 ** -11 + 2.0 ** -12 + 2.0 ** -8) * sums + 500 * 2.0 ** -31 * most, "out")


@pytest.mark.parametrize("where", ["k_scale", "v_scale", "q"])
def test_attention_nonfinite(env, where):
    """A NaN in a valid place reaches its rows in every column, and no others."""
    torch, ww = env
    q = _randn(torch, (2, 1, 4, 64), 1, torch.float16)
    kept = _caches(torch, 2, 300, 2, 64, 2)
    if where == "q":
        q[1, 0, 2, 5] = math.nan
        bad = [(1, 2)]
    else:
        kept[2 if where == "k_scale" else 3][0, 1, 77] = math.nan
        bad = [(0, 2), (0, 3)]
    out = ww.cross_attention_int8(q, *kept)
    want = torch.zeros((2, 4), device="cuda", dtype=torch.bool)
    for b, h in bad:
        want[b, h] = True
    assert torch.equal(out[:, 0].isnan().all(-1), want) and torch.equal(out[:, 0].isnan().any(-1), want)


def test_attention_layouts(env):
    torch, ww = env
    qkv = _randn(torch, (2, 3, 3, 8, 64), 1, torch.float16)
    kept = _caches(torch, 3, 400, 8, 64, 2)
    q = qkv[:, :, 1]
    views = [c[1:, 100:365, 4:6] for c in kept[:2]] + [c[1:, 4:6, 100:365] for c in kept[2:]]
    assert torch.equal(ww.cross_attention_int8(q, *views), ww.cross_attention_int8(q.contiguous(), *[c.contiguous() for c in views]))
    one = [c[:1, :, :1].expand(2, 400, 2, 64) for c in kept[:2]] + [c[:1, :1].expand(2, 2, 400) for c in kept[2:]]
    assert torch.equal(ww.cross_attention_int8(q, *one), ww.cross_attention_int8(q, *[c.contiguous() for c in one]))
    many = _randn(torch, (2, 100, 8, 64), 3, torch.float16)
    assert torch.equal(ww.cross_attention_int8(many, *one), ww.cross_attention_int8(many, *[c.contiguous() for c in one]))


# ---------------------------------------------------------------- together, streams, graphs

def _layer(torch, ww, dt, seed=0):
    """Weights of a decoder's layer in 8 bits: C channels, 4 heads of 32."""
    C = 128
    make = lambda n, s: ww.quantize_tokens(_randn(torch, (n, C), seed + s, dt, C ** -0.5))  # noqa: E731
    return {"C": C, "q": make(C, 1), "kv": make(2 * C, 2), "out": make(C, 3), "w": _randn(torch, (C,), seed + 4, dt, 0.1) + 1,
            "b": _randn(torch, (C,), seed + 5, dt, 0.1)}


def _step(torch, ww, p, x, residual, kept, lens):
    """Norm in 8 bits, projection, attention over the cache, projection."""
    xq, xs, h = ww.layer_norm_int8(x, p["w"], p["b"], residual=residual)
    q = ww.int8_matmul(xq, xs, *p["q"], dtype=x.dtype).view(*x.shape[:2], 4, 32)
    a = ww.cross_attention_int8(q, *kept, k_lens=lens)
    return h, ww.int8_linear(a.view(x.shape), *p["out"])


def _cache_of(torch, ww, p, states):
    B, L, C = states.shape
    kv = ww.int8_linear(states, *p["kv"]).view(B, L, 2, 4, 32)
    kept = [torch.zeros((B, L, 4, 32), device="cuda", dtype=torch.int8) for _ in range(2)]
    kept += [torch.zeros((B, 4, L), device="cuda") for _ in range(2)]
    ww.quantize_kv(kv[:, :, 0], kv[:, :, 1], *kept)
    return kept


@pytest.mark.parametrize("dt", ["f16", "bf16"])
def test_a_layer_in_8_bits(env, dt):
    """The operators as a decoder's layer runs them against the same steps in 64 bits on the same 8-bit numbers: each step
    is given the previous one's result, and the whole stays within 5 % of a layer without 8 bits."""
    torch, ww = env
    t = _type(torch, dt)
    p = _layer(torch, ww, t)
    B, L = 3, 200
    states = _randn(torch, (B, L, p["C"]), 11, t)
    lens = torch.tensor([200, 55, 0], device="cuda", dtype=torch.int32)
    kept = _cache_of(torch, ww, p, states)
    x, r = _randn(torch, (B, 1, p["C"]), 12, t), _randn(torch, (B, 1, p["C"]), 13, t)
    h, y = _step(torch, ww, p, x, r, kept, lens)
    assert torch.equal(h, x + r) and not y[2].any()
    full = {n: p[n][0].double() * p[n][1].double()[:, None] for n in ("q", "kv", "out")}
    xd = torch.nn.functional.layer_norm(h.double(), (p["C"],), p["w"].double(), p["b"].double(), 1e-5)
    q = (xd @ full["q"].t()).view(B, 1, 4, 32)
    kv = (states.double() @ full["kv"].t()).view(B, L, 2, 4, 32)
    s = torch.einsum("bihd,bjhd->bhij", q, kv[:, :, 0]) / math.sqrt(32)
    s = s.masked_fill(torch.arange(L, device="cuda")[None, None, None] >= lens[:, None, None, None], -math.inf)
    pr = torch.nan_to_num(torch.softmax(s, -1))
    ref = torch.einsum("bhij,bjhd->bihd", pr, kv[:, :, 1]).reshape(B, 1, -1) @ full["out"].t()
    assert (y.double() - ref).norm() <= 0.05 * ref.norm()
    assert ww.device_error() == 0


def test_streams_and_graphs(env):
    """A captured step replays on new inputs; two captured graphs with their own workspaces run at once; a call on
    another stream belongs to it."""
    torch, ww = env
    p = _layer(torch, ww, torch.float16)
    C = p["C"]
    kept = _cache_of(torch, ww, p, _randn(torch, (2, 3000, C), 1, torch.float16))
    lens = torch.tensor([3000, 1234], device="cuda", dtype=torch.int32)
    ins = [(_randn(torch, (2, n, C), 10 + n, torch.float16), _randn(torch, (2, n, C), 20 + n, torch.float16)) for n in (1, 30)]
    eager = [_step(torch, ww, p, *i, kept, lens) for i in ins]
    graphs, outs = [], []
    torch.cuda.synchronize()
    for i in ins:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(_step(torch, ww, p, *i, kept, lens))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(3):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for a, b in zip(outs, eager):
        assert all(torch.equal(x, y) for x, y in zip(a, b))
    for (x, r), s in zip(ins, streams):
        x.copy_(x.flip(0))
        torch.cuda.synchronize()
    lens.copy_(lens.flip(0))
    torch.cuda.synchronize()
    for g in graphs:
        g.replay()
    torch.cuda.synchronize()
    for i, a in zip(ins, outs):
        assert all(torch.equal(x, y) for x, y in zip(a, _step(torch, ww, p, *i, kept, lens)))
    s = torch.cuda.Stream()
    x, r = ins[1]
    got = ww.int8_linear(x, *p["q"], stream=s), ww.layer_norm(x, p["w"], p["b"], stream=s)
    s.synchronize()
    assert torch.equal(got[0], ww.int8_linear(x, *p["q"])) and torch.equal(got[1], ww.layer_norm(x, p["w"], p["b"]))


def test_backward_captured(env):
    """The norm's gradient captured into a graph and replayed on new incoming gradients."""
    torch, ww = env
    x, w, b = _randn(torch, (3000, 320), 1, torch.bfloat16), _randn(torch, (320,), 2, torch.bfloat16), _randn(torch, (320,), 3, torch.bfloat16)
    _, mean, rstd = ww.layer_norm(x, w, b, return_stats=True)
    dy = _randn(torch, (3000, 320), 4, torch.bfloat16)
    ww.layer_norm_backward(dy, x, w, mean, rstd)
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        out = ww.layer_norm_backward(dy, x, w, mean, rstd)
    dy.copy_(_randn(torch, (3000, 320), 5, torch.bfloat16))
    g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(out, ww.layer_norm_backward(dy, x, w, mean, rstd)))


def test_refusals(env):
    torch, ww = env
    f16, f32 = torch.float16, torch.float32
    x, w = torch.zeros((4, 64), device="cuda", dtype=f16), torch.zeros(64, device="cuda", dtype=f16)
    stats = [torch.zeros(4, device="cuda") for _ in range(2)]
    i8, s4, s8 = torch.zeros((8, 64), device="cuda", dtype=torch.int8), torch.zeros(4, device="cuda"), torch.zeros(8, device="cuda")
    k = torch.zeros((2, 5, 4, 32), device="cuda", dtype=f16)
    kept = _caches(torch, 2, 9, 4, 32, 1)
    for error, call in [
            (TypeError, lambda: ww.layer_norm(x.double())), (TypeError, lambda: ww.layer_norm(x, w.float())),
            (ValueError, lambda: ww.layer_norm(x, w[:32])), (ValueError, lambda: ww.layer_norm(x, None, w)),
            (ValueError, lambda: ww.layer_norm(x.t())), (ValueError, lambda: ww.layer_norm(x[:, :0])),
            (ValueError, lambda: ww.layer_norm(x, residual=x[:2])), (ValueError, lambda: ww.layer_norm(x.view(2, 2, 64).transpose(0, 1))),
            (ww.WWError, lambda: ww.layer_norm(x, eps=-1.0)), (ValueError, lambda: ww.layer_norm(x, out=x[:2])),
            (ValueError, lambda: ww.layer_norm_backward(x[:2], x, w, *stats)), (TypeError, lambda: ww.layer_norm_backward(x, x, w, w, w)),
            (ValueError, lambda: ww.layer_norm_backward(x, x, w, s8, s8)),
            (ValueError, lambda: ww.int8_linear(x, i8[:, :32], s8)), (TypeError, lambda: ww.int8_linear(x, x, s8)),
            (ValueError, lambda: ww.int8_linear(x, i8, s4)), (TypeError, lambda: ww.int8_linear(x, i8, s8, s8)),
            (ValueError, lambda: ww.int8_linear(x[:, :63].contiguous(), torch.zeros((8, 63), device="cuda", dtype=torch.int8), s8)),
            (TypeError, lambda: ww.int8_matmul(x, s4, i8, s8)), (TypeError, lambda: ww.int8_matmul(i8[:4], s4, i8, s8, dtype=torch.int8)),
            (ww.WWError, lambda: ww.int8_linear(x, torch.zeros(513, device="cuda", dtype=torch.int8)[1:].view(8, 64), s8)),
            (ValueError, lambda: ww.quantize_kv(k, k[:, :3], *kept)), (TypeError, lambda: ww.quantize_kv(k.float(), k.float(), *kept)),
            (ValueError, lambda: ww.quantize_kv(k[:1], k[:1], *kept)), (TypeError, lambda: ww.quantize_kv(k, k, *kept, start=s4.int()[:2].long())),
            (ValueError, lambda: ww.quantize_kv(k, k, *kept, lens=s4.int())), (ValueError, lambda: ww.quantize_kv(k, k, *kept[:2], s4, s4)),
            (ww.WWError, lambda: ww.quantize_kv(k, k, *[c[:1].expand(2, *c.shape[1:]) for c in kept])),
            (TypeError, lambda: ww.dequantize_kv(*kept, dtype=f32)), (TypeError, lambda: ww.dequantize_kv(kept[0].short(), *kept[1:])),
            (ValueError, lambda: ww.cross_attention_int8(k[..., :16].contiguous(), *kept)), (TypeError, lambda: ww.cross_attention_int8(k.float(), *kept)),
            (ValueError, lambda: ww.cross_attention_int8(k[:, :, :3].contiguous(), *kept)), (ValueError, lambda: ww.cross_attention_int8(k, *kept, key_mask=s4)),
            (ValueError, lambda: ww.cross_attention_int8(k, *kept, bias_table=w[None]))]:
        with pytest.raises(error):
            call()


def test_plugins_give_the_functions_bits(env):
    torch, ww = env
    from whirlwind_trt_plugins_b200 import plugins as pl
    T = pl.TensorDesc.of

    def run(p, ins, outs, *ws):
        assert p.enqueue([T(t) for t in ins], ins, outs, *ws) == 0
        return outs

    like = torch.empty_like
    x, r = _randn(torch, (3, 40, 64), 1, torch.float16), _randn(torch, (3, 40, 64), 2, torch.float16)
    w, b = _randn(torch, (64,), 3, torch.float16), _randn(torch, (64,), 4, torch.float16)
    got = run(pl.LayerNormPlugin(use_residual=1, eps_nano=2000), [x, w, b, r], [like(x), like(x)])
    assert all(torch.equal(a, c) for a, c in zip(got, ww.layer_norm(x, w, b, 2e-6, residual=r)))
    assert torch.equal(run(pl.LayerNormPlugin(), [x, w, b], [like(x)])[0], ww.layer_norm(x, w, b))
    wq, ws = ww.quantize_tokens(_randn(torch, (128, 64), 5, torch.float16))
    bias = _randn(torch, (128,), 6, torch.float16)
    for rows in (x, x[:, :1].contiguous()):
        p = pl.Int8LinearPlugin(use_bias=1)
        ins = [rows, wq, ws, bias]
        scratch = torch.empty(max(16, p.get_workspace_size([T(t) for t in ins])), device="cuda", dtype=torch.uint8)
        out = torch.empty((*rows.shape[:2], 128), device="cuda", dtype=torch.float16)
        assert torch.equal(run(p, ins, [out], scratch)[0], ww.int8_linear(*ins))
    k, v = _randn(torch, (2, 900, 2, 64), 7, torch.bfloat16), _randn(torch, (2, 900, 2, 64), 8, torch.bfloat16)
    kept = [torch.empty(k.shape, device="cuda", dtype=torch.int8) for _ in range(2)] + [torch.empty((2, 2, 900), device="cuda") for _ in range(2)]
    want = [like(c) for c in kept]
    run(pl.QuantizeKvPlugin(), [k, v], kept)
    ww.quantize_kv(k, v, *want)
    assert all(torch.equal(a, c) for a, c in zip(kept, want))
    lens, table = torch.tensor([900, 333], device="cuda", dtype=torch.int32), _randn(torch, (8, 32), 9, torch.bfloat16)
    mask = torch.rand((2, 900), device="cuda") >= 0.1
    for Lq in (1, 3, 50):
        q = _randn(torch, (2, Lq, 8, 64), 10, torch.bfloat16)
        p = pl.CrossAttentionInt8Plugin(1, 1, 1, max_distance=64, q_offset=5)
        ins = [q, *kept, lens, mask, table]
        scratch = torch.empty(p.get_workspace_size([T(t) for t in ins]), device="cuda", dtype=torch.uint8)
        ref = ww.cross_attention_int8(q, *kept, k_lens=lens, key_mask=mask, bias_table=table, max_distance=64, q_offset=5)
        assert torch.equal(run(p, ins, [like(q)], scratch)[0], ref)
        if Lq < 50:  # few rows also without a workspace: in other parts, so not to the bit
            plain = run(p, ins, [like(q)])[0]
            assert (plain.float() - ref.float()).abs().max() <= 2.0 ** -7 * ref.float().abs().max()
    assert ww.device_error() == 0


def test_example_layer_in_8_bits(env):
    """The example's layer in 8 bits beside itself: 8-bit steps of 1/254 of a row's largest value."""
    import importlib.util
    import os

    from conftest import ROOT
    torch, ww = env
    spec = importlib.util.spec_from_file_location("example", os.path.join(ROOT, "examples", "stereo_cross_attention.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    torch.manual_seed(0)
    layer = m.RowCrossAttention(64, heads=2).cuda().bfloat16()
    left, right, _, valid = m.pair(1, 64, 6, 160, 24, torch.Generator(device="cuda").manual_seed(0))
    with torch.no_grad():
        full = layer(left.bfloat16(), right.bfloat16(), valid).float()
    got = m.Int8RowCrossAttention(layer)(left.bfloat16(), right.bfloat16(), valid).float()
    assert torch.isfinite(got).all() and (got - full).norm() <= 0.05 * full.norm()


def test_long_rows_without_workspace(env):
    """Up to 128 rows a key head run without scratch memory through the C call."""
    torch, ww = env
    from whirlwind_trt_plugins_b200 import attention, layers
    q = _randn(torch, (1, 1, 4, 64), 1, torch.float16)
    kept = _caches(torch, 1, 9000, 2, 64, 2)
    ref = ww.cross_attention_int8(q, *kept)
    out = torch.empty_like(q)
    st = [9000 * 128, 128, 64]
    a = attention._ATTN.pack(q.data_ptr(), kept[0].data_ptr(), kept[1].data_ptr(), out.data_ptr(), *[0] * 10, 0, 256, 256, 64, *st, *st, 0, 0, 0,
                             1, 1, 1, 9000, 4, 2, 64, 0, 128, 1, 0, 0.125) + layers._SCALES.pack(kept[2].data_ptr(), kept[3].data_ptr(), 18000, 9000, 18000, 9000)
    assert layers._lib.ww_cross_attention_int8_workspace(a) > 0
    assert layers._lib.ww_cross_attention_int8(a, torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    assert (out.float() - ref.float()).abs().max() <= 2.0 ** -9 * ref.float().abs().max()
