"""A matching layer on stereo features: every left pixel attends to the pixels
of its row in the right view, then the refined features go into the correlation
volume and the disparity regression.

    python examples/stereo_cross_attention.py [--steps 150]

The layer runs ``qk_norm_rope`` (norm and column rotation of queries and keys),
``cross_attention`` with a learned bias by column distance and invalid right
pixels masked, and in training their gradients.  The trained layer also runs in 8
bits (``int8_linear``, ``quantize_kv``, ``cross_attention_int8``).  The data are
synthetic: random left rows and right rows shifted by a per-row disparity, with noise.
"""
from __future__ import annotations

import argparse
import os
import sys

import torch
from torch import nn

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import whirlwind_trt_plugins_b200 as ww  # noqa: E402


class RowCrossAttention(nn.Module):
    """Left features [B, C, H, W] attend to the right view's, row by row."""

    def __init__(self, channels: int, heads: int, buckets: int = 32, max_distance: int = 64, max_width: int = 512):
        super().__init__()
        d = channels // heads
        self.heads, self.max_distance = heads, max_distance
        self.to_q = nn.Linear(channels, channels, bias=False)
        self.to_kv = nn.Linear(channels, 2 * channels, bias=False)
        self.q_weight, self.k_weight = nn.Parameter(torch.ones(d)), nn.Parameter(torch.ones(d))
        self.bias_table = nn.Parameter(torch.zeros(heads, buckets))
        angle = torch.arange(max_width)[:, None] * 100.0 ** (-torch.arange(d // 4) / (d // 4))
        self.register_buffer("cos", angle.cos().float(), persistent=False)  # half of each head is rotated
        self.register_buffer("sin", angle.sin().float(), persistent=False)

    def _apply(self, fn, recurse=True):
        super()._apply(fn, recurse)
        self.cos, self.sin = self.cos.float(), self.sin.float()  # the tables stay fp32
        return self

    def forward(self, left, right, right_valid=None):
        B, C, H, W = left.shape
        rows = lambda x: x.permute(0, 2, 3, 1).reshape(B * H, W, C)  # noqa: E731
        q = self.to_q(rows(left)).view(B * H, W, self.heads, -1)
        kv = self.to_kv(rows(right)).view(B * H, W, 2, self.heads, -1)
        k, v = kv[:, :, 0], kv[:, :, 1]  # slices of one projection
        mask = None if right_valid is None else right_valid.reshape(B * H, W)
        if torch.is_grad_enabled():
            q, k = ww.qk_norm_rope_autograd(q, k, self.q_weight, self.k_weight, self.cos, self.sin)
            out = ww.cross_attention_autograd(q, k, v, self.bias_table, key_mask=mask, max_distance=self.max_distance)
        else:
            q, k = ww.qk_norm_rope(q, k, self.q_weight, self.k_weight, self.cos, self.sin)
            out = ww.cross_attention(q, k, v, bias_table=self.bias_table, key_mask=mask,
                                     max_distance=self.max_distance)
        return out.reshape(B, H, W, C).permute(0, 3, 1, 2)


class Int8RowCrossAttention:
    """A trained layer for inference in 8 bits: weights with a scale for each channel, tokens
    with one each, keys and values with one for each token and head."""

    def __init__(self, layer: RowCrossAttention):
        self.layer = layer
        self.to_q, self.to_kv = ww.quantize_tokens(layer.to_q.weight.detach()), ww.quantize_tokens(layer.to_kv.weight.detach())

    @torch.no_grad()
    def __call__(self, left, right, right_valid=None):
        n, (B, C, H, W) = self.layer, left.shape
        rows = lambda x: x.permute(0, 2, 3, 1).reshape(B * H, W, C).contiguous()  # noqa: E731
        q = ww.int8_linear(rows(left), *self.to_q).view(B * H, W, n.heads, -1)
        kv = ww.int8_linear(rows(right), *self.to_kv).view(B * H, W, 2, n.heads, -1)
        q, k = ww.qk_norm_rope(q, kv[:, :, 0], n.q_weight, n.k_weight, n.cos, n.sin)
        kept = [torch.empty(k.shape, device=k.device, dtype=torch.int8) for _ in range(2)]
        kept += [torch.empty((B * H, n.heads, W), device=k.device) for _ in range(2)]
        ww.quantize_kv(k, kv[:, :, 1], *kept)
        mask = None if right_valid is None else right_valid.reshape(B * H, W)
        out = ww.cross_attention_int8(q, *kept, bias_table=n.bias_table, key_mask=mask, max_distance=n.max_distance)
        return out.reshape(B, H, W, C).permute(0, 3, 1, 2)


def pair(B, C, H, W, max_disp, generator):
    """Left and right features, the disparity of each row and the valid right pixels."""
    wide = torch.randn((B, C, H, W + max_disp), generator=generator, device="cuda")
    disp = torch.randint(0, max_disp, (B, H), generator=generator, device="cuda")
    at = torch.arange(W, device="cuda")
    left = wide[..., :W]
    index = (at[None, None] + disp[..., None])[:, None].expand(B, C, H, W)
    right = torch.gather(wide, 3, index)  # right[x] = left[x + d]: left x matches right x - d
    right = right + 0.1 * torch.randn(right.shape, generator=generator, device="cuda")
    valid = torch.rand((B, H, W), generator=generator, device="cuda") >= 0.05
    return left, right, disp, valid


def main(steps: int = 150, verbose: bool = True):
    torch.manual_seed(0)
    g = torch.Generator(device="cuda").manual_seed(0)
    B, C, H, W, D = 2, 64, 30, 160, 24
    layer = RowCrossAttention(C, heads=2).cuda().bfloat16()
    master = [p.detach().float().clone().requires_grad_(True) for p in layer.parameters()]
    opt = torch.optim.Adam(master, lr=3e-3)
    losses = []
    for step in range(steps):
        left, right, _, valid = pair(B, C, H, W, D, g)
        out = layer(left.bfloat16(), right.bfloat16(), valid)
        # pixels whose match lies inside the image should fetch it: the left features without the noise
        loss = (out.float() - left)[..., D:].square().mean()
        layer.zero_grad(set_to_none=True)
        loss.backward()
        for m, p in zip(master, layer.parameters()):
            m.grad = p.grad.float()
        opt.step()
        with torch.no_grad():
            for m, p in zip(master, layer.parameters()):
                p.copy_(m)
        losses.append(loss.item())
        if verbose and step % 25 == 0:
            print(f"step {step:4d}  loss {losses[-1]:.4f}")
    with torch.no_grad():
        left, right, disp, valid = pair(B, C, H, W, D, g)
        fetched = layer(left.bfloat16(), right.bfloat16(), valid)
        in_8_bits = Int8RowCrossAttention(layer)(left.bfloat16(), right.bfloat16(), valid)
        apart = (in_8_bits.float() - fetched.float()).norm() / fetched.float().norm()
        volume = ww.corr_volume((left + fetched.float()).half().contiguous(), right.half().contiguous(), D)
        estimate = ww.disparity_regression(volume * 16, ww.DISP_SOFTARGMAX, dtype=torch.float32)[:, 0]
        error = (estimate - disp[..., None]).abs()[..., D:].mean().item()
    if verbose:
        print(f"loss {losses[0]:.4f} -> {losses[-1]:.4f}; mean disparity error {error:.3f} of {D}; "
              f"features in 8 bits {apart:.3f} apart")
    assert ww.device_error() == 0
    return losses, error


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--steps", type=int, default=150)
    main(ap.parse_args().steps)
