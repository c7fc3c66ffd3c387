"""Trained adapters beside a projection (ops.lora_linear): plain form, gradients against differences, refusals."""
import pytest
import torch

from polyrl_b200 import ops

from .requests_oracle import check_near, lora64


def lora_case(t, k, widths, ranks, seed, dtype=torch.float32, device="cpu", bias=False, residual=False, swiglu=False):
    g = torch.Generator().manual_seed(seed)
    n = sum(widths)
    rnd = lambda *s, scale=1.0: (torch.randn(*s, generator=g) * scale).to(dtype).to(device)  # noqa: E731
    return dict(x=rnd(t, k), w=rnd(n, k, scale=0.05), parts=[None if r == 0 else (rnd(r, k, scale=k ** -0.5), rnd(m, r, scale=0.2)) for r, m in zip(ranks, widths)],
                widths=widths, scale=2.0, dy=rnd(t, n // 2 if swiglu else n), bias=rnd(n) if bias else None, residual=rnd(t, n) if residual else None, swiglu=swiglu)


def run_lora(c, need=("x", "parts")):
    """Outputs by name, as lora64 names them."""
    x = c["x"].detach().requires_grad_("x" in need)
    parts = [p if p is None else tuple(m.detach().requires_grad_("parts" in need) for m in p) for p in c["parts"]]
    if c["swiglu"]:
        y = ops.lora_linear_swiglu(x, c["w"], *parts, c["scale"])
    else:
        y = ops.lora_linear(x, c["w"], [m if p is None else p for p, m in zip(parts, c["widths"])], c["scale"], c["bias"], c["residual"])
    leaves = ([("dx", x)] if "x" in need else []) + [(f"d{n}{i}", m) for i, p in enumerate(parts) if p is not None and "parts" in need for n, m in zip("ab", p)]
    grads = torch.autograd.grad(y, [t for _, t in leaves], c["dy"]) if leaves else []
    return {"y": y.detach(), **{n: g for (n, _), g in zip(leaves, grads)}}


def check_lora(c, **kw):
    ref = lora64(**c)
    got = run_lora(c, **kw)
    for name, t in got.items():
        assert t.shape == ref[name][0].shape
        check_near(t, *ref[name])
    return got


@pytest.mark.parametrize("t,k,widths,ranks,swiglu", [(1, 8, (8,), (1,), False), (5, 24, (16, 8, 8), (3, 0, 4), False), (7, 16, (128, 128), (4, 2), True),
                                                     (7, 16, (128, 128), (0, 2), True)])
def test_plain_form(t, k, widths, ranks, swiglu):
    check_lora(lora_case(t, k, widths, ranks, 0, bias=not swiglu, residual=not swiglu, swiglu=swiglu))


def test_plain_form_against_differences():
    c = lora_case(3, 8, (8, 16), (2, 3), 1, torch.float64)
    flat = [m.requires_grad_() for p in c["parts"] for m in p]
    assert torch.autograd.gradcheck(lambda x, *ab: ops.lora_linear(x, c["w"], [ab[:2], ab[2:]], 2.0), (c["x"].requires_grad_(), *flat))


def test_leading_dimensions_and_no_adapter():
    c = lora_case(6, 8, (8, 8), (2, 0), 2)
    y = ops.lora_linear(c["x"].view(2, 3, 8), c["w"], [c["parts"][0], 8], 2.0, residual=c["dy"].view(2, 3, 16))
    assert torch.allclose(y.view(6, 16), ops.lora_linear(c["x"], c["w"], [c["parts"][0], 8], 2.0, residual=c["dy"]))


def test_refusals():
    c = lora_case(4, 8, (8, 16), (2, 3), 3)
    x, w, (p, q) = c["x"], c["w"], c["parts"]
    for bad in ([p], [p, q, 8], [q, p, 8], [p, (q[0], q[1][:8])], [p, (q[0][:, :4], q[1])], [p, (q[0], p[1])], [8, 8, 8, 0]):
        with pytest.raises(ValueError):
            ops.lora_linear(x, w, bad, 1.0)
    with pytest.raises(ValueError, match="rows"):
        ops.lora_linear(x[:, :4], w, [p, q], 1.0)
    with pytest.raises(ValueError, match="bias"):
        ops.lora_linear(x, w, [p, q], 1.0, bias=torch.zeros(8))
    with pytest.raises(ValueError, match="residual"):
        ops.lora_linear(x, w, [p, q], 1.0, residual=torch.zeros(4, 8))
    with pytest.raises(ValueError, match="128"):
        ops.lora_linear_swiglu(x, w, None, None, 1.0)
