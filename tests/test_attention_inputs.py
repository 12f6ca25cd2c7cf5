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


def test_plugin_takes_masks_of_both_types():
    """key_mask is bool or uint8; descriptors of uint8 tensors carry kINT8, as those of NV12 frames do."""
    import torch
    from whirlwind_trt_plugins_b200 import plugins as pl
    p = pl.get_plugin_creator("CrossAttention").create_plugin({"use_mask": 1})
    q, k = (torch.zeros(s, dtype=torch.float16) for s in ((2, 5, 8, 64), (2, 7, 4, 64)))
    for t, ok in ((torch.bool, True), (torch.uint8, True), (torch.float16, False), (torch.int32, False)):
        io = [pl.TensorDesc.of(x) for x in (q, k, k, torch.zeros((2, 7), dtype=t), q)]
        assert p.supports_format_combination(3, io, 4, 1) is ok
