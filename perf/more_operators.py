"""Measured cases of the operators of an 8-bit matching layer around the attention operators: layer norm (with
a residual sum, with an 8-bit result for a projection) and its gradient, products in 8-bit integers with a scale for each token
and channel, keys and values kept in 8 bits, and attention that reads them.

Sizes are those of stereo matching with the configurations of this repository (the tokens of 16 pairs of 94 x 312
features of 256 channels, 120 x 160 maps of 320 channels), of a decoder that attends to an encoder's states one
token at a time, and generic ones.  Inputs are seeded and made on the GPU.
"""
import math

import torch

own = False

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
EPS = 1e-5
SMALL = 2.0 ** -119  # a row whose largest magnitude is below this has the scale 0 in 8 bits


def _norm(name, rows, n, dtype, residual=False, out=0, backward=False):
    return {"name": name, "op": "norm", "rows": rows, "n": n, "dtype": dtype, "residual": residual, "out": out,
            "backward": backward}


def _linear(name, rows, k, n, dtype, bias=True):
    return {"name": name, "op": "linear", "rows": rows, "k": k, "n": n, "dtype": dtype, "bias": bias}


def _cache(name, B, L, room, H, D, dtype, ragged=False):
    return {"name": name, "op": "cache", "B": B, "L": L, "room": room, "H": H, "D": D, "dtype": dtype,
            "ragged": ragged}


def _attn(name, B, Lq, Lk, Hq, Hk, D, dtype, ragged=False, masked=0.0, buckets=0, distance=128, offset=0):
    return {"name": name, "op": "attn", "B": B, "Lq": Lq, "Lk": Lk, "Hq": Hq, "Hk": Hk, "D": D, "dtype": dtype,
            "ragged": ragged, "masked": masked, "buckets": buckets, "distance": distance, "offset": offset}


def listed():
    return [
        # one token of a decoder: the residual stream updated, normalised into 8 bits, projected: latency only
        _norm("norm_token_int8", 1, 1024, "bf16", residual=True, out=1024),
        # all pixels of 16 stereo pairs (94 x 312 features of 256 channels): bandwidth
        _norm("norm_rows_312", 16 * 94 * 312, 256, "f16"),
        # its gradient in training with the residual stream's
        _norm("norm_grad_rows", 16 * 94 * 312, 256, "bf16", residual=True, backward=True),
        # gradient in full precision, odd rows and an odd width
        _norm("norm_grad_odd_f32", 9001, 1337, "f32", backward=True),
        # one token of a decoder through a wide projection: the weights' bytes are the bound
        _linear("linear_token", 1, 4096, 4096, "f16"),
        # queries, keys and values of the pixels of 16 pairs from 256 channels: bandwidth of the result
        _linear("linear_rows_qkv", 16 * 94 * 312, 256, 768, "f16"),
        # odd sizes in every direction
        _linear("linear_ragged", 1777, 1000, 1111, "bf16"),
        # a wide projection of many tokens: the tensor cores' rate
        _linear("linear_wide", 8192, 8192, 8192, "bf16", bias=False),
        # one new token for each of 8 items written behind their own lengths, the cache read back
        _cache("cache_token", 8, 1, 512, 8, 128, "bf16", ragged=True),
        # an encoder's states written and read back
        _cache("cache_encoder", 2, 40001, 40001, 8, 128, "f16"),
        # one token of a decoder against a short encoder, lengths per item, one of them empty, some keys masked
        _attn("attn_token_ragged", 8, 1, 1500, 16, 4, 64, "bf16", ragged=True, masked=0.05),
        # one token against a long encoder with a relative bias: the cache's bytes are the bound
        _attn("attn_token_long", 2, 1, 40001, 32, 8, 128, "bf16", buckets=32, distance=512, offset=40000),
    ]


def _between(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    dtype = rng.choice(["f16", "bf16"])
    op = rng.choice(["norm", "norm_grad", "linear", "linear", "cache", "attn", "attn"])
    if op.startswith("norm"):
        n = rng.choice([_between(rng, 17, 9000), 8 * _between(rng, 4, 1024)])
        rows = _between(rng, 1, 16 * 94 * 312 * 256 // max(n, 256))
        if rows * n < 6e7:
            dtype = rng.choice([dtype, dtype, "f32"])
        if op == "norm":
            c = _norm("", rows, n, dtype, rng.random() < 0.5)
            if dtype != "f32" and rng.random() < 0.4:
                c["out"] = _between(rng, 16, 1024)
                c["rows"] = min(rows, 16 * 94 * 312 * 256 // (n + c["out"]))
        else:
            c = _norm("", rows, n, dtype, rng.random() < 0.5, backward=True)
    elif op == "linear":
        k, n = (rng.choice([_between(rng, 17, 8192), 64 * _between(rng, 1, 128)]) for _ in range(2))
        dtype = rng.choice([dtype, dtype, dtype, "f32"])
        size = 4 if dtype == "f32" else 2
        most = min(8192 ** 3 // (k * n), 16 * 94 * 312 * 2 * (256 + 768) // (size * (k + n)))
        c = _linear("", rng.choice([_between(rng, 1, 64), _between(rng, 1, most)]), k, n, dtype, rng.random() < 0.7)
    elif op == "cache":
        H, D = rng.choice([1, 2, 4, 5, 8]), rng.choice([32, 48, 64, 80, 128])
        most = 2 * 40001 * 8 * 128 // (H * D)
        B = _between(rng, 1, 32)
        room = _between(rng, 1, most // B)
        c = _cache("", B, rng.choice([1, room, _between(rng, 1, room)]), room, H, D, dtype, rng.random() < 0.5)
    else:
        D, Hk = rng.choice([32, 48, 64, 80, 128]), rng.choice([1, 2, 3, 5, 8])
        Hq = Hk * rng.choice([1, 1, 2, 4, 8])
        if rng.random() < 0.75:
            Lq, Lk = rng.choice([1, 1, 1, 2, 5, 9]), _between(rng, 1, 40001)
            B = max(1, min(_between(rng, 1, 64), 80002 * 1024 // (Lk * Hk * D)))
        else:
            Lq, Lk = _between(rng, 30, 4000), _between(rng, 77, 4000)
            B = max(1, min(8, 4000 * 4000 * 8 * 128 // (Lq * Lk * Hq * D)))
        c = _attn("", B, Lq, Lk, Hq, Hk, D, dtype, B > 1 and rng.random() < 0.4, rng.choice([0.0, 0.0, 0.05, 0.3]),
                  rng.choice([0, 0, 32, 48]), rng.choice([64, 128, 300]), max(0, Lk - Lq))
    del c["name"]
    return c


def _lengths(c):
    """Keys of each batch item: all of them, or spread over (0, Lk] with the last item empty."""
    B, Lk = c["B"], c["Lk"]
    if not c["ragged"]:
        return [Lk] * B
    return [max(1, Lk - (b * 7919) % max(1, (3 * Lk) // 4)) for b in range(B - 1)] + [0]


def prepare(c, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dt = TYPES[c["dtype"]]

    def normal(*shape, dtype=dt):
        return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)

    def spread(t):
        """Rows of different sizes, as activations have: a factor between 1/4 and 4 for each."""
        return t * torch.exp2(4 * torch.rand(t.shape[:-1] + (1,), generator=g, device="cuda") - 2).to(t.dtype)

    s = {"case": c}
    def projection(n, k):
        """Weights in 8 bits, rows starting on 16 bytes, and their scales."""
        w = spread(normal(n, k, dtype=torch.float32)) / math.sqrt(k)
        s["w_scale"] = w.abs().amax(-1) / 127.0
        s["w_q"] = torch.zeros((n, (k + 15) // 16 * 16), device="cuda", dtype=torch.int8)[:, :k]
        s["w_q"].copy_(torch.round(w / s["w_scale"][:, None]))

    if c["op"] == "norm":
        rows, n = c["rows"], c["n"]
        if c["out"]:
            projection(c["out"], n)
        s["x"] = spread(normal(rows, n)) + normal(n)
        s["weight"], s["bias"] = (1 + 0.1 * normal(n, dtype=torch.float32)).to(dt), (0.1 * normal(n)).to(dt)
        s["residual"] = normal(rows, n) if c["residual"] else None  # in the backward pass: the sum's gradient
        if c["backward"]:
            s["dy"] = normal(rows, n)
            x = s["x"].float()  # what the forward pass has saved
            s["mean"] = x.mean(-1)
            s["rstd"] = torch.rsqrt((x - s["mean"][:, None]).square_().mean(-1) + EPS)
    elif c["op"] == "linear":
        rows, k, n = c["rows"], c["k"], c["n"]
        s["x"] = spread(normal(rows, k))
        projection(n, k)
        s["bias"] = (0.1 * normal(n)).to(dt) if c["bias"] else None
    else:
        B, H = c["B"], c["H"] if c["op"] == "cache" else c["Hk"]
        D, L = c["D"], c["L"] if c["op"] == "cache" else c["Lk"]
        k, v = spread(normal(B, L, H, D)), spread(normal(B, L, H, D))
        if c["op"] == "cache":
            room = c["room"]
            s["k"], s["v"] = k, v
            s["start"] = s["lens"] = None
            if c["ragged"]:  # tokens of an item that are there, and where its first one goes
                at = [(b * 7919) % (room - L + 1) for b in range(B)]
                s["start"] = torch.tensor(at, device="cuda", dtype=torch.int32)
                s["lens"] = torch.tensor([max(1, L - b % max(1, L // 2)) for b in range(B)], device="cuda", dtype=torch.int32)
            for x in "kv":
                s[x + "_cache"] = torch.randint(-127, 128, (B, room, H, D), generator=g, device="cuda", dtype=torch.int8)
                s[x + "_scale"] = 0.01 + 0.02 * torch.rand((B, H, room), generator=g, device="cuda")
            return s
        for name, x in (("k", k), ("v", v)):
            scale = x.float().abs().amax(-1) / 127.0
            s[name + "_cache"] = torch.round(x.float() / scale[..., None]).to(torch.int8)
            s[name + "_scale"] = scale.transpose(1, 2).contiguous()
        s["q"] = normal(B, c["Lq"], c["Hq"], D)
        s["k_lens"] = torch.tensor(_lengths(c), device="cuda", dtype=torch.int32) if c["ragged"] else None
        s["key_mask"] = torch.rand((B, L), generator=g, device="cuda") >= c["masked"] if c["masked"] else None
        s["table"] = normal(c["Hq"], c["buckets"]) if c["buckets"] else None
    return s


# ---- the plain forms: elementary operations in 32 bits, one rounding at the end ----

def _quantised(x):
    """Whole numbers in [-127, 127] and the scale of each row."""
    top = x.abs().amax(-1, keepdim=True)
    small = top < SMALL
    q = torch.round(x * (127.0 / torch.where(small, 1.0, top)))
    return torch.where(small, 0.0, q), torch.where(small, 0.0, top / 127.0)


def _plain_norm(s):
    c, dt, n = s["case"], s["x"].dtype, s["case"]["n"]
    x, w = s["x"].float(), s["weight"].float()
    if c["backward"]:
        xh = (x - s["mean"][:, None]) * s["rstd"][:, None]
        dy = s["dy"].float()
        dw, db = (dy * xh).sum(0), dy.sum(0)
        dy = dy * w
        dx = s["rstd"][:, None] * (dy - dy.mean(-1, keepdim=True) - xh * (dy * xh).mean(-1, keepdim=True))
        if s["residual"] is not None:
            dx = dx + s["residual"].float()
        return {"dx": dx.to(dt), "dweight": dw.to(dt), "dbias": db.to(dt)}
    got = {}
    if s["residual"] is not None:
        got["sum"] = s["x"] + s["residual"]  # the residual stream, in its type
        x = got["sum"].float()
    mean = x.sum(-1, keepdim=True) / n
    x = x - mean
    y = x * torch.rsqrt((x * x).sum(-1, keepdim=True) / n + EPS) * w + s["bias"].float()
    if c["out"]:
        q, scale = _quantised(y)
        y = (q @ s["w_q"].float().t()).mul_(scale).mul_(s["w_scale"])
    return {**got, "y": y.to(dt)}


def _plain_linear(s):
    q, scale = _quantised(s["x"].float())
    y = (q @ s["w_q"].float().t()).mul_(scale).mul_(s["w_scale"])
    if s["bias"] is not None:
        y += s["bias"].float()
    return y.to(s["x"].dtype)


def _plain_cache(s):
    c, got = s["case"], {}
    B, L, room = c["B"], c["L"], c["room"]
    start = torch.zeros(B, device="cuda", dtype=torch.int64) if s["start"] is None else s["start"].long()
    at = torch.arange(room, device="cuda")[None, :] - start[:, None]  # the token that goes to each place
    there = (at >= 0) & (at < (L if s["lens"] is None else s["lens"][:, None]))
    at = at.clamp(0, L - 1)
    item = torch.arange(B, device="cuda")[:, None]
    for x in "kv":
        q, scale = _quantised(s[x].float())
        put = there[:, :, None, None]
        cache, old = s[x + "_cache"], s[x + "_scale"]
        cache.copy_(torch.where(put, q[item, at].to(torch.int8), cache))
        old.copy_(torch.where(put[..., 0], scale[item, at][..., 0], old.transpose(1, 2)).transpose(1, 2))
        got[x] = (cache.float() * old.transpose(1, 2)[..., None]).to(s[x].dtype)
        got[x + "_scale"] = old
    return got


def _plain_buckets(c):
    """Bucket of each (query, key), keys behind the query in one: exact for short distances, then logarithmic."""
    i = torch.arange(c["Lq"], device="cuda")[:, None] + c["offset"]
    d = (i - torch.arange(c["Lk"], device="cuda")[None, :]).clamp(min=0)
    n = c["buckets"]
    e = n // 2
    far = torch.log(d.clamp(min=1).double() / e) / math.log(c["distance"] / e) * (n - e)
    return torch.where(d < e, d, (e + torch.floor(far + 1e-9).long()).clamp(max=n - 1))


def _plain_attn(s):
    c, dt = s["case"], s["q"].dtype
    B, Lq, Lk, Hq, Hk, D = (c[n] for n in ("B", "Lq", "Lk", "Hq", "Hk", "D"))
    keep = torch.ones((B, Lk), device="cuda", dtype=torch.bool)
    if s["k_lens"] is not None:
        keep = torch.arange(Lk, device="cuda")[None, :] < s["k_lens"][:, None]
    if s["key_mask"] is not None:
        keep = keep & s["key_mask"]
    q = s["q"].float().transpose(1, 2).reshape(B, Hk, Hq // Hk * Lq, D)
    k = s["k_cache"].transpose(1, 2).float() * s["k_scale"][..., None]
    x = (q @ k.transpose(2, 3)).mul_(1.0 / math.sqrt(D)).view(B, Hk, Hq // Hk, Lq, Lk)
    if s["table"] is not None:
        x += s["table"].float()[:, _plain_buckets(c)].view(Hk, Hq // Hk, Lq, Lk)
    x.masked_fill_(~keep[:, None, None, None, :], -math.inf)
    top = x.amax(-1, keepdim=True)
    p = x.sub_(torch.where(torch.isinf(top), 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    p = p.div_(torch.where(total == 0, 1.0, total)).view(B, Hk, Hq // Hk * Lq, Lk)
    v = s["v_cache"].transpose(1, 2).float() * s["v_scale"][..., None]
    return (p @ v).view(B, Hq, Lq, D).transpose(1, 2).contiguous().to(dt)


def run(s):
    c = s["case"]
    if not own:
        return {"norm": _plain_norm, "linear": _plain_linear, "cache": _plain_cache, "attn": _plain_attn}[c["op"]](s)
    import whirlwind_trt_plugins_b200 as ww
    if c["op"] == "norm":
        if c["backward"]:
            dx, dw, db = ww.layer_norm_backward(s["dy"], s["x"], s["weight"], s["mean"], s["rstd"], dsum=s["residual"])
            return {"dx": dx, "dweight": dw, "dbias": db}
        if not c["out"]:
            got = ww.layer_norm(s["x"], s["weight"], s["bias"], EPS, residual=s["residual"])
            return {"y": got} if s["residual"] is None else {"y": got[0], "sum": got[1]}
        q, scale, *more = ww.layer_norm_int8(s["x"], s["weight"], s["bias"], EPS, residual=s["residual"])
        got = {"y": ww.int8_matmul(q, scale, s["w_q"], s["w_scale"], dtype=s["x"].dtype)}
        return {**got, "sum": more[0]} if more else got
    if c["op"] == "linear":
        return ww.int8_linear(s["x"], s["w_q"], s["w_scale"], s["bias"])
    kept = s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"]
    if c["op"] == "cache":
        ww.quantize_kv(s["k"], s["v"], *kept, start=s["start"], lens=s["lens"])
        k, v = ww.dequantize_kv(*kept, dtype=s["k"].dtype)
        return {"k": k, "v": v, "k_scale": s["k_scale"], "v_scale": s["v_scale"]}
    return ww.cross_attention_int8(s["q"], *kept, k_lens=s["k_lens"], key_mask=s["key_mask"], bias_table=s["table"],
                                   max_distance=c["distance"], bidirectional=False, q_offset=c["offset"])


# ---- the definitions in 64 bits ----

def _exact_int8(x):
    """Nearest multiples of each row's step, and the step."""
    x = x.double()
    step = x.abs().max(-1, keepdim=True).values / 127
    step = torch.where(step * 127 < SMALL, torch.zeros_like(step), step)
    return torch.where(step == 0, torch.zeros_like(x), torch.round(x / step)), step


def _exact_norm(c, s):
    n, grads = c["n"], c["backward"]
    w, b = s["weight"].double().requires_grad_(grads), s["bias"].double().requires_grad_(grads)
    got = {}
    matrix = (s["w_q"].double() * s["w_scale"].double()[:, None]).t() if c["out"] else None

    def put(name, t):
        got.setdefault(name, []).append(t)

    for r in range(0, c["rows"], 1 + (1 << 25) // n):
        at = slice(r, r + 1 + (1 << 25) // n)
        x = s["x"][at]
        if s["residual"] is not None and not grads:
            x = (x.double() + s["residual"][at].double()).to(x.dtype)  # rounded once, then normalised as it is kept
            put("sum", x.double())
        x = x.double().requires_grad_(grads)
        var, mean = torch.var_mean(x, -1, correction=0, keepdim=True)
        y = (x - mean) / torch.sqrt(var + EPS) * w + b
        if grads:
            dx, dw, db = torch.autograd.grad(y, (x, w, b), s["dy"][at].double())
            put("dx", dx if s["residual"] is None else dx + s["residual"][at].double())
            put("dweight", dw)
            put("dbias", db)
        elif c["out"]:
            q, step = _exact_int8(y)
            put("y", (q * step) @ matrix)
        else:
            put("y", y)
    return {k: torch.stack(v).sum(0) if k in ("dweight", "dbias") else torch.cat(v) for k, v in got.items()}


def _exact_linear(c, s):
    w = (s["w_q"].double() * s["w_scale"].double()[:, None]).t().contiguous()
    out = []
    for r in range(0, c["rows"], 65536):
        q, step = _exact_int8(s["x"][r:r + 65536])
        y = (q * step) @ w
        out.append(y if s["bias"] is None else y + s["bias"].double())
    return torch.cat(out)


def _exact_cache(c, s):
    got = {}
    for x in "kv":
        value = s[x + "_cache"].double() * s[x + "_scale"].double().transpose(1, 2)[..., None]
        scale = s[x + "_scale"].double()
        for b in range(c["B"]):
            n = c["L"] if s["lens"] is None else int(s["lens"][b])
            at = 0 if s["start"] is None else int(s["start"][b])
            q, step = _exact_int8(s[x][b, :n])
            value[b, at:at + n] = q * step
            scale[b, :, at:at + n] = step[..., 0].t()
        got[x], got[x + "_scale"] = value, scale
    return got


def _exact_bias(c, table):
    """Bias of each distance back from the query, by whole-number comparison: a distance d is in logarithmic bucket
    t or above where (d / e)^(n - e) >= (distance / e)^t."""
    n, top = c["buckets"], c["distance"]
    e = n // 2
    m = n - e
    edges = []
    for t in range(1, m):
        d = e
        while d ** m < e ** (m - t) * top ** t:
            d += 1
        edges.append(d)
    near = torch.tensor([d if d < e else e + sum(d >= x for x in edges) for d in range(top + 1)], device="cuda")
    i = torch.arange(c["Lq"], device="cuda")[:, None] + c["offset"]
    back = (i - torch.arange(c["Lk"], device="cuda")[None, :]).clamp(0, top)
    return table.double()[near[back]]


def _exact_attn(c, s):
    B, Lq, Hq, Hk, D = (c[n] for n in ("B", "Lq", "Hq", "Hk", "D"))
    if B * Hq > 2500:
        return None
    out = torch.zeros((B, Lq, Hq, D), dtype=torch.float64, device="cuda")
    lens = _lengths(c)
    for h in range(Hq):
        g = h // (Hq // Hk)
        bias = None if s["table"] is None else _exact_bias(c, s["table"][h])
        for b in range(B):
            keys = torch.arange(lens[b], device="cuda")
            if s["key_mask"] is not None:
                keys = keys[s["key_mask"][b, :lens[b]]]
            if keys.numel() == 0:
                continue
            k, v = (s[x + "_cache"][b, keys, g].double() * s[x + "_scale"][b, g, keys].double()[:, None] for x in "kv")
            x = s["q"][b, :, h].double() @ k.t() / math.sqrt(D)
            out[b, :, h] = torch.softmax(x if bias is None else x + bias[:, keys], -1) @ v
    return out


def exact(c, seed):
    s = prepare(c, seed)
    return {"norm": _exact_norm, "linear": _exact_linear, "cache": _exact_cache, "attn": _exact_attn}[c["op"]](c, s)


def work(c):
    size = 4 if c["dtype"] == "f32" else 2
    if c["op"] == "norm":
        one, w = c["rows"] * c["n"] * size, 2 * c["n"] * size
        if c["backward"]:
            return {"bytes": (3 + c["residual"]) * one + 8 * c["rows"] + w, "flops": 14 * c["rows"] * c["n"]}
        if c["out"]:
            out, w = c["rows"] * c["out"] * size, w + c["out"] * (c["n"] + 4)
        else:
            out = one
        return {"bytes": (1 + 2 * c["residual"]) * one + out + w, "flops": c["rows"] * c["n"] * (8 + 2 * c["out"])}
    if c["op"] == "linear":
        M, K, N = c["rows"], c["k"], c["n"]
        return {"bytes": M * K * size + N * K + M * N * size + 4 * N, "flops": 2 * M * K * N}
    if c["op"] == "cache":
        vectors, held = 2 * c["B"] * c["L"] * c["H"], 2 * c["B"] * c["room"] * c["H"]
        # tokens read and written in 8 bits, the others' 8 bits read, everything written back in 16
        return {"bytes": vectors * c["D"] * 2 + held * (3 * c["D"] + 4), "flops": 3 * vectors * c["D"] + held * c["D"]}
    keys = sum(_lengths(c))
    q = c["B"] * c["Lq"] * c["Hq"] * c["D"] * 2
    return {"bytes": 2 * q + 2 * keys * c["Hk"] * (c["D"] + 4), "flops": 4 * c["Lq"] * c["Hq"] * keys * c["D"]}
