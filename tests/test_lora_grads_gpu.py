"""Trained adapters beside a projection: gradients of gradients, and the projection that is kept for them."""
import pytest
import torch

from polyrl_b200 import ops

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def case(t=130, k=256, n=256, r=16):
    g = torch.Generator().manual_seed(t)
    rnd = lambda *s: (torch.randn(*s, generator=g) * s[-1] ** -0.5).to(BF).cuda().requires_grad_(True)  # noqa: E731
    return rnd(t, k), rnd(n, k), rnd(r, k), rnd(n, r)


@pytest.mark.parametrize("swiglu", [False, True])
def test_a_second_gradient_is_refused(swiglu):
    """Gradients taken with create_graph are what they are without; asked for gradients of their own, they raise instead of being constants."""
    x, w, a, b = case()
    b2 = b[:128].detach().clone().requires_grad_(True)
    res = torch.randn(130, 256, device="cuda").to(BF).requires_grad_(True)
    fn = (lambda: ops.lora_linear_swiglu(x, w, (a, b2), None, 0.5)) if swiglu else (lambda: ops.lora_linear(x, w, [(a, b)], 0.5, residual=res))
    leaves = [x, w, a, b2] if swiglu else [x, w, a, b, res]
    plain = torch.autograd.grad(fn().float().square().sum(), leaves)
    deep = torch.autograd.grad(fn().float().square().sum(), leaves, create_graph=True)
    assert all(torch.equal(p, d) for p, d in zip(plain, deep)) and not any(p.requires_grad for p in plain) and all(d.requires_grad for d in deep)
    for d in deep[:4]:
        with pytest.raises(RuntimeError, match="differentiated once"):
            d.float().square().sum().backward(retain_graph=True)
    # a penalty on top of the loss is refused as a whole
    y = fn().float().square().sum()
    with pytest.raises(RuntimeError, match="differentiated once"):
        (y + torch.autograd.grad(y, x, create_graph=True)[0].float().square().sum()).backward()
    if not swiglu:          # the residual's gradient is dy itself
        (gr,) = torch.autograd.grad(ops.lora_linear(x.detach(), w.detach(), [(a.detach(), b.detach())], 0.5, residual=res).float().square().sum(), res, create_graph=True)
        (second,) = torch.autograd.grad(gr.float().sum(), res)
        assert torch.equal(second, torch.full_like(second, 2.0))
