"""Logits under rules, and the samplers that take them: what the rules ban does not come, with top-k, nucleus or neither."""
import pytest
import torch

from polyrl_b200 import ops
from polyrl_b200.ops import LogitRules

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("top_k,top_p", [(-1, 1.0), (50, 1.0), (-1, 0.9), (5, 0.5), (1, 1.0)])
def test_banned_tokens_do_not_come(dtype, top_k, top_p):
    rows, v = 33, 5003
    g = torch.Generator().manual_seed(rows)
    allowed = [sorted(torch.randperm(v, generator=g)[:n].tolist()) for n in [1, 1, 2, 3, 7, 40, 3000] * 4 + [1] * 5]
    masks = torch.stack([ops.token_mask(a, v) for a in allowed]).cuda()
    z = (torch.randn(rows, v, generator=g) * 4).to(dtype).cuda()
    rules = LogitRules(masks=masks, tokens=torch.randint(0, v, (rows, 300), generator=g, dtype=torch.int32).cuda(),
                       frequency=torch.full((rows,), 1e20, device="cuda"), presence=torch.full((rows,), 1e20, device="cuda"))
    out = ops.adjust_logits(z, rules)
    for temp in (1.0, 0.0, 1e-6, 1e-30):
        for seed in range(3):
            seeds = torch.arange(rows, device="cuda") * 7919 + seed
            tok, lp = ops.sample_tokens(out, torch.full((rows,), temp, device="cuda"), seeds, top_k=top_k, top_p=top_p)
            for t, p, a in zip(tok.tolist(), lp.tolist(), allowed):
                assert t in a and p <= 1e-5 and p > -float("inf"), (temp, t, p, len(a))
                assert len(a) > 1 or abs(p) < 1e-5
