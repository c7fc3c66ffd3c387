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


@pytest.mark.parametrize("t,k,f", [(130, 64, 128), (300, 128, 512), (5, 256, 128)])
def test_saved_projection_is_rounded(t, k, f):
    """Sums of whole numbers that fp32 holds exactly (below 2^24): what is kept of them is the nearest 24-bit value, half of its last place off at most."""
    g = torch.Generator().manual_seed(t)
    whole = lambda *s: torch.randint(-200, 201, s, generator=g).to(BF).cuda()  # noqa: E731
    x, w, low, b = whole(t, k), whole(2 * f, k), whole(t, 8), whole(2 * f, 8)
    exact = x.double() @ w.double().t() + low.double() @ b.double().t()
    assert (x.double().abs() @ w.double().abs().t() + low.double().abs() @ b.double().abs().t()).max() < 2 ** 24
    _, gu, lo = ops.ext().lora_gemm_swiglu(x, w, low, b, True)
    got = ((gu.view(torch.int16).int() << 16) | (lo.int() << 8)).view(torch.float32).double()
    step = torch.exp2(torch.floor(torch.log2(exact.abs().clamp(min=1))) - 15)               # of 16 bits of mantissa, the leading one among them
    assert ((got - exact).abs() <= step / 2).all() and ((got - exact).abs() > step / 4).any()
