"""Second derivatives of the differentiable forms are refused, not dropped."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def env():
    import torch
    import whirlwind_trt_plugins_b200 as ww
    return torch, ww


@pytest.mark.parametrize("which", ["attention", "norm"])
def test_second_derivatives_raise(env, which):
    torch, ww = env
    q, k = (torch.randn((2, 20, 2, 32), device="cuda", dtype=torch.float16).requires_grad_(True) for _ in range(2))
    if which == "attention":
        y = ww.cross_attention_autograd(q, k, k)
    else:
        w = torch.ones(32, device="cuda", dtype=torch.float16, requires_grad=True)
        angle = torch.rand((20, 16), device="cuda")
        y = torch.cat(ww.qk_norm_rope_autograd(q, k, w, w, angle.cos(), angle.sin()))
    g, = torch.autograd.grad(y.float().square().sum(), q, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        (y.float().sum() + g.float().square().sum()).backward()  # a gradient penalty beside the loss


def test_gradient_of_a_concatenation(env):
    """The incoming gradient is a contiguous view two bytes into a buffer."""
    torch, ww = env
    q, k = (torch.randn((2, 20, 2, 32), device="cuda", dtype=torch.float16).requires_grad_(True) for _ in range(2))
    w = torch.ones(32, device="cuda", dtype=torch.float16)
    angle = torch.rand((20, 16), device="cuda")
    weights = torch.randn(1 + q.numel(), device="cuda").half()
    one = torch.ones(1, device="cuda", dtype=torch.float16)
    for fn in (lambda: ww.cross_attention_autograd(q, k, k),
               lambda: ww.qk_norm_rope_autograd(q, k, w, w, angle.cos(), angle.sin())[0]):
        got, = torch.autograd.grad((torch.cat([one, fn().flatten()]) * weights).sum(), q)
        want, = torch.autograd.grad(fn(), q, weights[1:].clone().view(q.shape))
        assert torch.equal(got, want)
