"""Measured cases of the attention operators: the per-head norm and rotation of
queries and keys, cross attention to an encoder's states of another length with
a learned relative position bias by buckets, and their gradients.

Sizes are those of stereo matching with the configurations of this repository
(image rows of 160, 312 and 320 feature columns attending to the rows of the
other view, coarse maps attending to each other as a whole) and of a decoder
that attends to an encoder's states one token at a time.  Inputs are seeded and
made on the GPU.
"""
import math

import torch

own = False

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
EPS = 1e-6


def _rope(name, B, Lq, Lk, Hq, Hk, D, R, dtype, backward=False, interleaved=False):
    return {"name": name, "op": "rope", "B": B, "Lq": Lq, "Lk": Lk, "Hq": Hq, "Hk": Hk, "D": D, "R": R,
            "dtype": dtype, "backward": backward, "interleaved": interleaved}


def _attn(name, B, Lq, Lk, Hq, Hk, D, dtype, backward=False, ragged=False, masked=0.0, buckets=0, distance=128,
          bidirectional=True, offset=0):
    return {"name": name, "op": "attn", "B": B, "Lq": Lq, "Lk": Lk, "Hq": Hq, "Hk": Hk, "D": D, "dtype": dtype,
            "backward": backward, "ragged": ragged, "masked": masked, "buckets": buckets, "distance": distance,
            "bidirectional": bidirectional, "offset": offset}


def listed():
    return [
        # one new token of a decoder: its query and the key it adds; latency only
        _rope("rope_one_token", 1, 1, 1, 8, 8, 64, 64, "f16"),
        # queries and keys of all image rows of 16 stereo pairs (94 x 312 features of 256 channels): bandwidth
        _rope("rope_rows_312", 16 * 94, 312, 312, 8, 8, 32, 32, "f16"),
        # its gradient in training, shared key heads, half of each head rotated, an odd encoder length
        _rope("rope_grad_gqa", 8, 1200, 1777, 16, 4, 128, 64, "bf16", backward=True),
        # gradient in full precision over the rows of one 120 x 160 pair, neighbouring pairs rotated
        _rope("rope_grad_f32", 120, 160, 160, 5, 5, 64, 64, "f32", backward=True, interleaved=True),
        # one token of a decoder against a short encoder, lengths per item, one of them empty
        _attn("token_ragged", 8, 1, 1500, 16, 4, 64, "bf16", ragged=True),
        # one token against a long encoder: the cache's bytes are the bound
        _attn("token_long", 2, 1, 40001, 32, 8, 128, "bf16", buckets=32, distance=512, bidirectional=False,
              offset=40000),
        # rows of one 120 x 160 pair, left columns attending to right columns, relative bias
        _attn("rows_160", 120, 160, 160, 5, 5, 64, "f16", buckets=32),
        # rows of 16 pairs of 94 x 312 with invalid pixels masked, relative bias: the batched case
        _attn("rows_312_masked", 16 * 94, 312, 312, 8, 8, 32, "f16", masked=0.05, buckets=32, distance=192),
        # every pixel of one 120 x 160 map to every pixel of the other view: long on both sides
        _attn("map_19200", 1, 19200, 19200, 5, 5, 64, "f16"),
        # training on rows: forward and all gradients with the bias table's
        _attn("train_rows_320", 2 * 180, 320, 320, 3, 3, 32, "f16", backward=True, masked=0.05, buckets=32,
              bidirectional=False),
        # training a decoder on encoders of another, ragged length with shared heads
        _attn("train_ragged_gqa", 4, 1200, 1777, 16, 4, 64, "bf16", backward=True, ragged=True),
        # training on a whole 60 x 80 map, wide heads, relative bias
        _attn("train_map_4800", 1, 4800, 4800, 8, 8, 128, "bf16", backward=True, buckets=64, distance=640),
    ]


def _between(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    dtype = rng.choice(["f16", "bf16"])
    if rng.random() < 0.4:  # norm and rotation
        D = rng.choice([32, 64, 96, 128])
        Hk = rng.choice([1, 2, 4, 5, 8])
        Hq = Hk * rng.choice([1, 1, 2, 4])
        tokens = _between(rng, 1, 400000 * 256 // (D * (Hq + Hk)))
        B = min(_between(rng, 1, 1504), tokens)
        L = max(1, tokens // B)
        c = _rope("", B, L, _between(rng, max(1, L // 2), L), Hq, Hk, D, rng.choice([D, D // 2]),
                  rng.choice([dtype, dtype, "f32"]), rng.random() < 0.5, rng.random() < 0.3)
    else:
        D = rng.choice([32, 40, 64, 80, 128])
        Hk = rng.choice([1, 2, 3, 5, 8])
        Hq = Hk * rng.choice([1, 1, 2, 4])
        buckets = rng.choice([0, 0, 32, 48])
        backward = False
        shape = rng.choice(["token", "rows", "map"])
        if shape == "token":
            B, Lq, Lk = _between(rng, 1, 32), rng.choice([1, 1, 1, 2, 5]), _between(rng, 1, 40001)
            B = max(1, min(B, 80002 * 1024 // (Lk * Hk * D)))
            offset = Lk - 1
        elif shape == "rows":
            Lq = _between(rng, 40, 400)
            Lk = _between(rng, max(1, Lq // 2), Lq)
            B = _between(rng, 4, max(4, 1504 * 312 * 312 * 8 // (Lq * Lk * Hq * 2)))
            B = min(B, 1504 * 312 * 256 // (Lq * Hq * D) + 1)
            backward, offset = rng.random() < 0.5, 0
        else:
            Lq, Lk = _between(rng, 300, 6000), _between(rng, 77, 6000)
            B = max(1, min(8, 4800 * 4800 * 8 * 128 // (Lq * Lk * Hq * D * 2)))
            backward, offset = rng.random() < 0.5, 0
        masked = rng.choice([0.0, 0.0, 0.05, 0.3])
        c = _attn("", B, Lq, Lk, Hq, Hk, D, dtype, backward, B > 1 and rng.random() < 0.4, masked, buckets,
                  rng.choice([64, 128, 300]), rng.random() < 0.7, offset)
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

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dt)

    B, Lq, Lk, Hq, Hk, D = (c[n] for n in ("B", "Lq", "Lk", "Hq", "Hk", "D"))
    s = {"case": c, "q": normal(B, Lq, Hq, D), "k": normal(B, Lk, Hk, D)}
    if c["op"] == "rope":
        half = c["R"] // 2
        at = torch.arange(max(Lq, Lk) + 16, device="cuda", dtype=torch.float64)[:, None]
        angle = at * 10000.0 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        s["q_weight"] = (1 + 0.1 * normal(D).float()).to(dt)
        s["k_weight"] = (1 + 0.1 * normal(D).float()).to(dt)
        # a decoder's queries stand at the end of the sequence, the encoder's keys at their own places
        s["q_pos"] = torch.arange(Lq, device="cuda", dtype=torch.int32) + 16
        s["k_pos"] = None
        if c["backward"]:
            s["dq_out"], s["dk_out"] = normal(B, Lq, Hq, D), normal(B, Lk, Hk, D)
        return s
    s["v"] = normal(B, Lk, Hk, D)
    s["k_lens"] = torch.tensor(_lengths(c), device="cuda", dtype=torch.int32) if c["ragged"] else None
    s["key_mask"] = torch.rand((B, Lk), generator=g, device="cuda") >= c["masked"] if c["masked"] else None
    s["table"] = normal(Hq, c["buckets"]) if c["buckets"] else None
    if c["backward"]:
        s["dout"] = normal(B, Lq, Hq, D)
    return s


# ---- the plain forms: elementary operations in 32 bits, one rounding at the end ----

def _rotate(y, cos, sin, R, interleaved):
    if interleaved:
        a, b = y[..., 0:R:2], y[..., 1:R:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    else:
        a, b = y[..., :R // 2], y[..., R // 2:R]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    return torch.cat([turned, y[..., R:]], dim=-1)


def _plain_rope(c, x, w, cos, sin, pos, dout):
    L, R = x.shape[1], c["R"]
    pos = torch.arange(L, device=x.device) if pos is None else pos.long()
    cos, sin = cos[pos][None, :, None, :], sin[pos][None, :, None, :]
    xf, wf = x.float(), w.float()
    inv = torch.rsqrt((xf * xf).mean(-1, keepdim=True) + EPS)
    if dout is None:
        return _rotate(xf * inv * wf, cos, sin, R, c["interleaved"]).to(x.dtype)
    dy = _rotate(dout.float(), cos, -sin, R, c["interleaved"])
    xh = xf * inv
    dw = (dy * xh).sum((0, 1, 2))
    dh = dy * wf
    dx = inv * (dh - xh * (dh * xh).mean(-1, keepdim=True))
    return dx.to(x.dtype), dw.to(w.dtype)


def _plain_buckets(c, device):
    """Bucket of each (query, key): exact for short distances, then logarithmic up to the last."""
    i = torch.arange(c["Lq"], device=device)[:, None] + c["offset"]
    rel = torch.arange(c["Lk"], device=device)[None, :] - i
    n = c["buckets"] // 2 if c["bidirectional"] else c["buckets"]
    first = torch.where(rel > 0, n, 0) if c["bidirectional"] else torch.zeros_like(rel)
    d = rel.abs() if c["bidirectional"] else (-rel).clamp(min=0)
    e = n // 2
    far = torch.log(d.clamp(min=1).double() / e) / math.log(c["distance"] / e) * (n - e)
    far = (e + torch.floor(far + 1e-9).long()).clamp(max=n - 1)
    return first + torch.where(d < e, d, far)


def _plain_attn(s):
    c, dt = s["case"], s["q"].dtype
    B, Lq, Lk, Hq, Hk, D = (c[n] for n in ("B", "Lq", "Lk", "Hq", "Hk", "D"))
    G, scale = Hq // Hk, 1.0 / math.sqrt(D)
    keep = torch.ones((B, Lk), device="cuda", dtype=torch.bool)
    if s["k_lens"] is not None:
        keep = torch.arange(Lk, device="cuda")[None, :] < s["k_lens"][:, None]
    if s["key_mask"] is not None:
        keep = keep & s["key_mask"]
    q = s["q"].float().transpose(1, 2).reshape(B, Hk, G * Lq, D)
    zero = ~keep[:, None, :, None]
    k = s["k"].float().transpose(1, 2).masked_fill(zero, 0.0)
    v = s["v"].float().transpose(1, 2).masked_fill(zero, 0.0)
    x = (q @ k.transpose(2, 3)).mul_(scale).view(B, Hk, G, Lq, Lk)
    if s["table"] is not None:
        bucket = _plain_buckets(c, "cuda")
        x += s["table"].float()[:, bucket].view(Hk, G, Lq, Lk)
    x.masked_fill_(~keep[:, None, None, None, :], -math.inf)
    top = x.amax(-1, keepdim=True)
    top = torch.where(torch.isinf(top), 0.0, top)
    p = x.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    p /= torch.where(total == 0, 1.0, total)
    p = p.view(B, Hk, G * Lq, Lk)
    out = p @ v
    put = lambda y, H: y.reshape(B, H, -1, D).transpose(1, 2).contiguous().to(dt)  # noqa: E731
    if not c["backward"]:
        return {"out": put(out, Hq)}
    do = s["dout"].float().transpose(1, 2).reshape(B, Hk, G * Lq, D)
    dv = p.transpose(2, 3) @ do
    ds = (do @ v.transpose(2, 3)).sub_((do * out).sum(-1, keepdim=True)).mul_(p)
    got = {"out": put(out, Hq), "dq": put((ds @ k) * scale, Hq), "dk": put((ds.transpose(2, 3) @ q) * scale, Hk),
           "dv": put(dv, Hk)}
    if s["table"] is not None:
        flat = ds.view(B, Hq, Lq, Lk).sum(0).view(Hq, Lq * Lk)
        dtable = torch.zeros((Hq, c["buckets"]), device="cuda")
        got["dtable"] = dtable.index_add_(1, bucket.view(-1), flat).to(dt)
    return got


def run(s):
    c = s["case"]
    if c["op"] == "rope":
        names = ("q", "k", "q_weight", "k_weight", "cos", "sin", "q_pos", "k_pos")
        if own:
            import whirlwind_trt_plugins_b200 as ww
            a = [s[n] for n in names]
            if not c["backward"]:
                return ww.qk_norm_rope(*a, eps=EPS, interleaved=c["interleaved"])
            return ww.qk_norm_rope_backward(s["dq_out"], s["dk_out"], *a, eps=EPS, interleaved=c["interleaved"])
        got = [_plain_rope(c, s[x], s[x + "_weight"], s["cos"], s["sin"], s[x + "_pos"], s.get("d" + x + "_out"))
               for x in "qk"]
        return (got[0][0], got[1][0], got[0][1], got[1][1]) if c["backward"] else tuple(got)
    if not own:
        return _plain_attn(s)
    import whirlwind_trt_plugins_b200 as ww
    more = {"k_lens": s["k_lens"], "key_mask": s["key_mask"], "bias_table": s["table"],
            "max_distance": c["distance"], "bidirectional": c["bidirectional"], "q_offset": c["offset"]}
    if not c["backward"]:
        return {"out": ww.cross_attention(s["q"], s["k"], s["v"], **more)}
    out, lse = ww.cross_attention(s["q"], s["k"], s["v"], return_lse=True, **more)
    dq, dk, dv, dtable = ww.cross_attention_backward(s["dout"], s["q"], s["k"], s["v"], out, lse, **more)
    got = {"out": out, "dq": dq, "dk": dk, "dv": dv}
    if dtable is not None:
        got["dtable"] = dtable
    return got


# ---- the definitions in 64 bits, one (batch item, head) or token block at a time, gradients by autograd ----

def _exact_rope(c, x, w, cos, sin, pos, dout):
    B, L, H, D = x.shape
    R = c["R"]
    pos = torch.arange(L, device=x.device) if pos is None else pos.long()
    turn = torch.complex(cos.double()[pos], sin.double()[pos])[:, None, :]
    w = w.double().requires_grad_(dout is not None)
    outs, grads, dw = [], [], torch.zeros(D, dtype=torch.float64, device=x.device)
    for b0 in range(0, B, 64):
        xb = x[b0:b0 + 64].double().requires_grad_(dout is not None)
        y = xb / torch.sqrt(xb.pow(2).sum(-1, keepdim=True) / D + EPS) * w
        if c["interleaved"]:
            z = torch.view_as_complex(y[..., :R].reshape(*y.shape[:3], R // 2, 2).contiguous()) * turn
            t = torch.view_as_real(z).reshape(*y.shape[:3], R)
        else:
            z = torch.complex(y[..., :R // 2], y[..., R // 2:R]) * turn
            t = torch.cat([z.real, z.imag], -1)
        t = torch.cat([t, y[..., R:]], -1)
        if dout is None:
            outs.append(t)
        else:
            gx, gw = torch.autograd.grad(t, (xb, w), dout[b0:b0 + 64].double())
            grads.append(gx)
            dw += gw
    return torch.cat(outs) if dout is None else (torch.cat(grads), dw)


def _exact_bucket_row(c):
    """Bucket of every distance j - i - offset that occurs, from the lowest up, by whole-number comparison:
    a distance d is in logarithmic bucket t or above where (d / e)^(n - e) >= (distance / e)^t."""
    lo, hi = -(c["Lq"] - 1) - c["offset"], c["Lk"] - 1 - c["offset"]
    n = c["buckets"] // 2 if c["bidirectional"] else c["buckets"]
    e = n // 2
    m, top = n - e, c["distance"]
    least = []
    for t in range(1, m):
        d = e
        while d ** m < e ** (m - t) * top ** t:
            d += 1
        least.append(d)
    near = [d if d < e else e + sum(d >= x for x in least) for d in range(top + 1)]
    row = []
    for rel in range(lo, hi + 1):
        d = abs(rel) if c["bidirectional"] else max(0, -rel)
        row.append(near[min(d, top)] + (n if c["bidirectional"] and rel > 0 else 0))
    return torch.tensor(row, device="cuda")


def exact(c, seed):
    s = prepare(c, seed)
    if c["op"] == "rope":
        got = [_exact_rope(c, s[x], s[x + "_weight"], s["cos"], s["sin"], s[x + "_pos"], s.get("d" + x + "_out"))
               for x in "qk"]
        return (got[0][0], got[1][0], got[0][1], got[1][1]) if c["backward"] else tuple(got)
    B, Lq, Lk, Hq, Hk, D = (c[n] for n in ("B", "Lq", "Lk", "Hq", "Hk", "D"))
    if B * Hq > 2500:
        return None
    need = c["backward"]
    out = torch.zeros((B, Lq, Hq, D), dtype=torch.float64, device="cuda")
    dq, dk, dv = torch.zeros_like(out), *(torch.zeros((B, Lk, Hk, D), dtype=torch.float64, device="cuda")
                                          for _ in range(2))
    dtable = torch.zeros((Hq, c["buckets"]), dtype=torch.float64, device="cuda")
    bucket = None
    if c["buckets"]:
        at = torch.arange(Lk, device="cuda")[None, :] - torch.arange(Lq, device="cuda")[:, None] + (Lq - 1)
        bucket = _exact_bucket_row(c)[at]
    lens = _lengths(c)
    for b in range(B):
        keys = torch.arange(lens[b], device="cuda")
        if s["key_mask"] is not None:
            keys = keys[s["key_mask"][b, :lens[b]]]
        if keys.numel() == 0:
            continue
        for h in range(Hq):
            g = h // (Hq // Hk)
            leaves = [s["q"][b, :, h].double(), s["k"][b, keys, g].double(), s["v"][b, keys, g].double()]
            if bucket is not None:
                leaves.append(s["table"][h].double())
            leaves = [x.requires_grad_(need) for x in leaves]
            x = leaves[0] @ leaves[1].t() / math.sqrt(D)
            if bucket is not None:
                x = x + leaves[3][bucket[:, keys]]
            o = torch.softmax(x, -1) @ leaves[2]
            out[b, :, h] = o.detach()
            if need:
                grads = torch.autograd.grad(o, leaves, s["dout"][b, :, h].double())
                dq[b, :, h] = grads[0]
                dk[b, keys, g] += grads[1]
                dv[b, keys, g] += grads[2]
                if bucket is not None:
                    dtable[h] += grads[3]
    got = {"out": out}
    if need:
        got.update(dq=dq, dk=dk, dv=dv)
        if bucket is not None:
            got["dtable"] = dtable
    return got


def work(c):
    B, Lq, Lk, Hq, Hk, D = (c[n] for n in ("B", "Lq", "Lk", "Hq", "Hk", "D"))
    size = 4 if c["dtype"] == "f32" else 2
    q, k = B * Lq * Hq * D * size, B * Lk * Hk * D * size
    if c["op"] == "rope":
        tables = 4 * c["R"] * max(Lq, Lk) + 2 * D * size
        per = 12 if c["backward"] else 6
        return {"bytes": (q + k) * (3 if c["backward"] else 2) + tables, "flops": per * (q + k) // size}
    keys = sum(_lengths(c))
    pairs = Lq * Hq * keys
    kv = 2 * keys * Hk * D * size
    if not c["backward"]:
        return {"bytes": 2 * q + kv, "flops": 4 * pairs * D}
    # forward and backward: q, k, v, dout read, out, dq, dk, dv written; two products forward, five backward
    return {"bytes": 4 * q + kv + 2 * k, "flops": 14 * pairs * D}
