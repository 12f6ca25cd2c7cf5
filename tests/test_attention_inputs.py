"""What the attention wrappers take as input, without a GPU."""


def test_incoming_gradients_in_any_layout():
    """What autograd may hand over: broadcast, transposed, with odd strides, or a contiguous view
    that starts off the 16-byte grid (the gradient of a concatenation)."""
    import torch
    from whirlwind_trt_plugins_b200 import attention
    shape, n = (2, 3, 4, 8), 2 * 3 * 4 * 8
    x = torch.arange(n, dtype=torch.float16).view(shape)
    buf = torch.cat([torch.zeros(1, dtype=torch.float16), x.flatten()])
    off = buf[1:].view(shape)
    assert off.is_contiguous() and off.data_ptr() % 16 != 0
    wide = torch.zeros((2, 3, 4, 9), dtype=torch.float16)
    wide[..., :8] = x
    for g in (x, off, x[:1].expand(shape), x[:, :1].expand(shape), x.transpose(1, 3).contiguous().transpose(1, 3),
              wide[..., :8], torch.ones((), dtype=torch.float16).expand(shape)):
        s = attention._strided(g)
        assert torch.equal(s, g) and s.data_ptr() % 16 == 0 and s.stride(3) == 1
        assert all(st % 8 == 0 for st in s.stride()[:3]) and s.stride(1) != 0
    assert attention._strided(x) is x  # nothing copied without need
