"""Rules on logits and adapters of requests on the CPU: the plain forms against the 64-bit oracle, and what is refused."""
import pytest
import torch

from polyrl_b200 import ops
from polyrl_b200.ops import LogitRules
from .requests_oracle import adapters64, check_near, check_rules, swiglu64


def rules_case(rows, v, n, seed, dtype=torch.float32, device="cpu", m=5):
    g = torch.Generator().manual_seed(seed)
    i32 = lambda lo, hi, *s: torch.randint(lo, hi, s, generator=g, dtype=torch.int32)  # noqa: E731
    lens = i32(0, n + 1, rows)
    lens[0] = n
    case = dict(tokens=i32(-1, v + 2, rows, n), lens=lens, prompt_lens=(lens * torch.rand(rows, generator=g)).int(),
                repetition=torch.tensor([1.0, 1.2, 0.8])[i32(0, 3, rows).long()], presence=torch.tensor([0.0, 0.7, -0.3])[i32(0, 3, rows).long()],
                frequency=torch.tensor([0.0, 0.2])[i32(0, 2, rows).long()], bias_ids=i32(-1, v + 2, rows, m), bias_values=torch.randn(rows, m, generator=g) * 3,
                stop_ids=i32(-1, v, rows, 2), min_lens=lens + i32(-1, 2, rows), masks=i32(-2 ** 31, 2 ** 31 - 1, 3, (v + 31) // 32), mask_rows=i32(-1, 4, rows))
    z = (torch.randn(rows, v, generator=g) * 4).to(dtype)
    return z.to(device), {k: t.to(device) for k, t in case.items()}


@pytest.mark.parametrize("rows,v,n", [(1, 7, 0), (1, 33, 1), (4, 64, 9), (9, 257, 40)])
def test_rules_plain_form(rows, v, n):
    z, case = rules_case(rows, v, n, rows + v)
    check_rules(ops.adjust_logits(z, LogitRules(**case)), z, **case)
    out = z.clone()
    assert ops.adjust_logits(out, LogitRules(**case), out=out) is out
    check_rules(out, z, **case)
    check_rules(ops.adjust_logits(z, LogitRules()), z)


def test_rules_refusals():
    z, case = rules_case(3, 40, 6, 0)
    for match, logits, kw in [
        ("bf16 or fp32", z.half(), {}),
        ("bf16 or fp32", z[0], {}),
        ("rows", z, dict(lens=case["lens"][:2], tokens=case["tokens"])),
        ("int32", z, dict(tokens=case["tokens"].long())),
        ("float32", z, dict(repetition=case["repetition"].double(), tokens=case["tokens"])),
        ("need the rows' tokens", z, dict(presence=case["presence"])),
        ("less than 1048576", z, dict(tokens=torch.zeros(3, 1, dtype=torch.int32).expand(3, 1 << 20))),
        ("belong together", z, dict(bias_ids=case["bias_ids"])),
        ("belong together", z, dict(bias_ids=case["bias_ids"], bias_values=case["bias_values"][:, :2])),
        ("at most 2046", z, dict(bias_ids=torch.zeros(3, 2047, dtype=torch.int32), bias_values=torch.zeros(3, 2047))),
        ("belong together", z, dict(stop_ids=case["stop_ids"], lens=case["lens"])),
        ("belong together", z, dict(stop_ids=case["stop_ids"], min_lens=case["min_lens"])),
        ("without masks", z, dict(mask_rows=case["mask_rows"])),
        ("masks", z, dict(masks=case["masks"][:, :1], mask_rows=case["mask_rows"])),
        ("masks", z, dict(masks=case["masks"][:2])),
    ]:
        with pytest.raises(ValueError, match=match):
            ops.adjust_logits(logits, LogitRules(**kw))
    with pytest.raises(ValueError, match="out must be"):
        ops.adjust_logits(z, LogitRules(), out=z[:2])


def test_token_mask():
    for v in (1, 31, 32, 33, 100):
        ids = sorted({0, v - 1, v // 2})
        m = ops.token_mask(ids, v)
        assert m.dtype == torch.int32 and m.shape == ((v + 31) // 32,)
        assert [t for t in range(v) if (int(m[t // 32]) >> (t % 32)) & 1] == ids
    with pytest.raises(ValueError):
        ops.token_mask([5], 5)


def adapters_case(t, k, widths, rank, num, seed, dtype=torch.float32, device="cpu", ids=None, extra=True):
    g = torch.Generator().manual_seed(seed)
    n = sum(widths)
    rnd = lambda *s, scale=1.0: (torch.randn(*s, generator=g) * scale).to(dtype).to(device)  # noqa: E731
    if ids is None:
        ids = torch.randint(-1, num + 2, (t,), generator=g, dtype=torch.int32)
    return dict(x=rnd(t, k), w=rnd(n, k, scale=0.05), a=rnd(num, len(widths) * rank, k, scale=k ** -0.5), b=rnd(num, n, rank, scale=0.3),
                scales=(torch.rand(num, generator=g) * 2).to(device), ids=ids.to(device), bias=rnd(n) if extra else None, residual=rnd(t, n) if extra else None)


@pytest.mark.parametrize("t,k,widths,rank,num", [(0, 32, (32,), 16, 1), (1, 32, (32,), 16, 1), (7, 64, (64, 32, 32), 16, 3), (20, 96, (32, 96), 32, 5)])
def test_adapters_plain_form(t, k, widths, rank, num):
    c = adapters_case(t, k, widths, rank, num, t)
    plan = ops.adapter_plan(c["ids"], num)
    y = ops.adapter_linear(c["x"], c["w"], c["a"], c["b"], c["scales"], plan, widths, c["bias"], c["residual"])
    check_near(y, *adapters64(**c, widths=widths))


def test_adapters_swiglu_plain_form():
    c = adapters_case(9, 64, (128, 128), 16, 4, 1, extra=False)
    y = ops.adapter_linear_swiglu(c["x"], c["w"], c["a"], c["b"], c["scales"], ops.adapter_plan(c["ids"], 4))
    check_near(y, *swiglu64(*adapters64(**c, widths=(128, 128), interleaved=True)))


def test_adapters_refusals():
    with pytest.raises(ValueError, match="int32"):
        ops.adapter_plan(torch.zeros(3, dtype=torch.int64), 1)
    with pytest.raises(ValueError, match="1 to 1024"):
        ops.adapter_plan(torch.zeros(3, dtype=torch.int32), 0)
    c = adapters_case(6, 64, (64, 32), 16, 2, 0)
    plan = ops.adapter_plan(c["ids"], 2)
    args = [c["x"], c["w"], c["a"], c["b"], c["scales"], plan]
    for match, at, value in [("rows", 0, c["x"][:, :32]), ("plan is of", 0, c["x"][:5]), ("stacked|expected", 2, c["a"][:1]), ("do not fit", 2, c["a"][:, :16]),
                             ("do not fit", 3, c["b"][:, :64]), ("fp32 scale", 4, c["scales"].double()), ("type", 2, c["a"].bfloat16())]:
        bad = list(args)
        bad[at] = value
        with pytest.raises(ValueError, match=match):
            ops.adapter_linear(*bad, widths=(64, 32))
    for widths, match in [((96, 32), "do not fit"), ((80, 16), "multiple of 32")]:
        with pytest.raises(ValueError, match=match):
            ops.adapter_linear(*args, widths=widths)
    with pytest.raises(ValueError, match="rank"):
        ops.adapter_linear(c["x"], c["w"], c["a"][:, :16], c["b"][:, :, :8].contiguous(), c["scales"], plan, widths=(64, 32))
    with pytest.raises(ValueError, match="bias"):
        ops.adapter_linear(*args, widths=(64, 32), bias=c["bias"][:64])
    with pytest.raises(ValueError, match="128"):
        c = adapters_case(6, 64, (64, 64), 16, 2, 0)
        ops.adapter_linear_swiglu(c["x"], c["w"], c["a"], c["b"], c["scales"], plan)
