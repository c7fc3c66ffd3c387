"""Rules on logits and adapters of requests: the sm_100a kernels against the 64-bit oracle."""
import pytest
import torch

from polyrl_b200 import ops
from polyrl_b200.ops import LogitRules
from .requests_oracle import adapters64, check_near, check_rules, swiglu64
from .test_requests_cpu import adapters_case, rules_case

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------------------------------------ rules
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,v,n,m", [(1, 1, 1, 1), (1, 31, 0, 0), (3, 32, 5, 3), (2, 2047, 300, 9), (5, 2048, 17, 40), (4, 4104, 1500, 7), (3, 16390, 999, 2046), (2, 33000, 8300, 30), (3, 100, 9000, 3)])
def test_rules(rows, v, n, m, dtype):
    z, case = rules_case(rows, v, n, rows * 7 + v, dtype, "cuda", m)
    z0 = z.clone()
    check_rules(ops.adjust_logits(z, LogitRules(**case)), z, **case)
    assert torch.equal(z.view(torch.uint8), z0.view(torch.uint8))
    ops.adjust_logits(z, LogitRules(**case), out=z)
    check_rules(z, z0, **case)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rules_one_at_a_time(dtype):
    z, case = rules_case(6, 5003, 250, 3, dtype, "cuda")
    hist = {k: case[k] for k in ("tokens", "lens", "prompt_lens")}
    for kw in [dict(hist, repetition=case["repetition"]), dict(hist, presence=case["presence"]), dict(tokens=case["tokens"], frequency=case["frequency"]),
               dict(bias_ids=case["bias_ids"], bias_values=case["bias_values"]), dict(lens=case["lens"], stop_ids=case["stop_ids"], min_lens=case["min_lens"]),
               dict(masks=case["masks"], mask_rows=case["mask_rows"]), dict(masks=case["masks"].repeat(2, 1)), {}]:
        check_rules(ops.adjust_logits(z, LogitRules(**kw)), z, **kw)
        y = z.clone()
        check_rules(ops.adjust_logits(y, LogitRules(**kw), out=y), z, **kw)


def test_rules_counts_long_histories():
    """One token repeated through a long history, prompt and output."""
    n = 70001
    z = torch.full((2, 600), 3.0, device="cuda")
    tokens = torch.full((2, n), 577, dtype=torch.int32, device="cuda")
    case = dict(tokens=tokens, lens=torch.tensor([n, n - 1], dtype=torch.int32, device="cuda"), prompt_lens=torch.tensor([0, 1000], dtype=torch.int32, device="cuda"),
                frequency=torch.tensor([0.5, 2.0], device="cuda"), repetition=torch.tensor([1.5, 1.5], device="cuda"))
    check_rules(ops.adjust_logits(z, LogitRules(**case)), z, **case)


@pytest.mark.parametrize("start", [0, 1, 2, 3])
@pytest.mark.parametrize("n", [8192, 8193, 8195])
def test_rules_long_histories_start_and_end_anywhere(n, start):
    z, case = rules_case(12, 3000, n + 8, n + start, torch.bfloat16, "cuda")
    wide = case["tokens"]
    case["tokens"] = wide[:, start:start + n]
    case["lens"] = torch.tensor([0, 1, 2, 3, 4, 5, 8, 4099, 6151, 8190, n - 1, n], dtype=torch.int32, device="cuda")
    case["prompt_lens"] = case["lens"] // 3
    assert case["tokens"].data_ptr() % 16 == 4 * start % 16
    check_rules(ops.adjust_logits(z, LogitRules(**case)), z, **case)
    y = z.clone()
    ops.adjust_logits(y, LogitRules(**case), out=y)
    check_rules(y, z, **case)
    odd = wide.reshape(-1)[start:start + 12 * (n + 3)].view(12, n + 3)         # every row starts somewhere else
    check_rules(ops.adjust_logits(z, LogitRules(**{**case, "tokens": odd})), z, **{**case, "tokens": odd})


def test_rules_masked_places_may_hold_anything():
    z, case = rules_case(4, 300, 20, 1, torch.bfloat16, "cuda")
    z[:, ::3], z[:, 1::7], z[:, 5::11] = float("nan"), float("inf"), torch.finfo(torch.bfloat16).min
    masks = torch.zeros(4, 10, dtype=torch.int32, device="cuda")
    masks[1], masks[2] = -1, 0x55555555
    kw = dict(masks=masks)
    out = ops.adjust_logits(z, LogitRules(**kw))
    check_rules(out, z, **kw)
    assert torch.isneginf(out[0]).all()                                 # nothing allowed


def test_rules_strides_views_and_odd_starts():
    wide = torch.randn(6, 1000, device="cuda").bfloat16()
    _, case = rules_case(3, 500, 30, 2, torch.bfloat16, "cuda")
    for z in (wide[::2, :500], wide[:3, 7:507], wide[1:4, 8:508]):
        check_rules(ops.adjust_logits(z, LogitRules(**case)), z, **case)
        buf = torch.full((3, 504), 7.0, device="cuda", dtype=torch.bfloat16)
        out = buf[:, 3:503]
        assert ops.adjust_logits(z, LogitRules(**case), out=out).data_ptr() == out.data_ptr()
        check_rules(out, z, **case)
        assert (buf[:, :3] == 7).all() and (buf[:, 503:] == 7).all()
    views = dict(case, tokens=torch.stack([case["tokens"], case["tokens"]], 1)[:, 1], masks=torch.cat([case["masks"], case["masks"]], 1)[:, : case["masks"].shape[1]])
    check_rules(ops.adjust_logits(wide[:3, :500], LogitRules(**views)), wide[:3, :500], **case)


def test_rules_refused_by_the_kernel_entry():
    z = torch.randn(4, 64, device="cuda")
    with pytest.raises(ValueError, match="device"):
        ops.adjust_logits(z, LogitRules(tokens=torch.zeros(4, 3, dtype=torch.int32)))
    with pytest.raises(ValueError, match="apart"):
        ops.adjust_logits(z[:2], LogitRules(), out=z[1:3])
    with pytest.raises(ValueError, match="unit inner stride"):
        ops.adjust_logits(z.t(), LogitRules())
    _, c = rules_case(4, 64, 6, 0, torch.float32, "cuda")
    for kw in [dict(lens=c["lens"][:2], tokens=c["tokens"]), dict(tokens=c["tokens"].long()), dict(repetition=c["repetition"].double(), tokens=c["tokens"]),
               dict(presence=c["presence"]), dict(tokens=torch.zeros(4, 1, dtype=torch.int32, device="cuda").expand(4, 1 << 20)), dict(bias_ids=c["bias_ids"]),
               dict(bias_ids=c["bias_ids"], bias_values=c["bias_values"][:, :2]), dict(bias_ids=c["bias_ids"].repeat(1, 500), bias_values=c["bias_values"].repeat(1, 500)),
               dict(stop_ids=c["stop_ids"], lens=c["lens"]), dict(stop_ids=c["stop_ids"], min_lens=c["min_lens"]), dict(mask_rows=c["mask_rows"]),
               dict(masks=c["masks"][:, :1], mask_rows=c["mask_rows"]), dict(masks=c["masks"][:2])]:
        with pytest.raises(ValueError, match="adjust_logits"):
            ops.adjust_logits(z, LogitRules(**kw))
    for bad, out in ((z.half(), None), (z[0], None), (z, z[:2]), (z, z.bfloat16())):
        with pytest.raises(ValueError, match="adjust_logits"):
            ops.adjust_logits(bad, LogitRules(), out=out)


def test_rules_stream_and_graph():
    z, case = rules_case(5, 3001, 64, 9, torch.bfloat16, "cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = ops.adjust_logits(z, LogitRules(**case))
    side.synchronize()
    check_rules(out, z, **case)
    rules, buf = LogitRules(**case), z.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.adjust_logits(buf, rules, out=buf)
    for seed in (1, 2):
        z2, case2 = rules_case(5, 3001, 64, seed, torch.bfloat16, "cuda")
        buf.copy_(z2)
        for k, t in case.items():
            t.copy_(case2[k])
        graph.replay()
        check_rules(buf, z2, **case2)


# ------------------------------------------------------------------------------------------------------------------ adapters
def near64(c, widths):
    """Up to 256 rows the adapters add to `linear`'s result."""
    return adapters64(**c, widths=widths, base=ops.linear(c["x"], c["w"], c["bias"]) if c["x"].shape[0] <= 256 else None)


def run_adapters(c, widths, num):
    plan = ops.adapter_plan(c["ids"], num)
    return ops.adapter_linear(c["x"], c["w"], c["a"], c["b"], c["scales"], plan, widths, c["bias"], c["residual"])


@pytest.mark.parametrize("t,num,kind", [(1, 1, "all"), (5, 3, "mixed"), (33, 2, "one"), (256, 40, "mixed"), (257, 1, "none"), (700, 5, "runs"), (3000, 1000, "mixed"),
                                        (1025, 3, "mixed"), (4098, 6, "runs"), (20011, 1024, "mixed"), (9999, 8, "mixed")])
def test_plan_sorts_rows(t, num, kind):
    ids = {"all": torch.zeros(t), "one": torch.ones(t), "none": torch.full((t,), -7.0), "mixed": torch.randint(-1, num + 1, (t,)).float(),
           "runs": torch.arange(num).repeat_interleave(t // num).float()}[kind].int().cuda()
    p = ops.adapter_plan(ids, num)
    buf = p.buf.cpu()
    used, tiles, order = int(buf[0]), buf[4:4 + 4 * p.max_tiles].view(-1, 4), buf[4 + 4 * p.max_tiles:]
    assert sorted(order.tolist()) == list(range(t)) and used <= p.max_tiles
    at = 0
    for l, first, rows, _ in tiles[:used].tolist():
        assert first == at and 1 <= rows <= p.tile_rows
        mine = order[first:first + rows]
        own = ids.cpu()[mine.long()]
        assert ((own == l) if l >= 0 else (own < 0) | (own >= num)).all()
        assert (mine[1:] > mine[:-1]).all()                              # stable
        at += rows
    assert at == t


@pytest.mark.parametrize("t,k,widths,rank,num", [
    (1, 32, (32,), 16, 1), (1, 896, (896, 128, 128), 16, 4), (2, 96, (32, 64), 48, 2), (15, 4096, (4096, 1024, 1024), 16, 3), (16, 256, (256,), 64, 1),
    (17, 256, (128,), 128, 2), (64, 2048, (2048,), 32, 40), (200, 512, (512, 64, 64), 16, 1), (256, 160, (96,), 16, 300), (257, 160, (96,), 16, 3),
    (300, 896, (896,), 64, 6), (1000, 224, (64, 32, 32), 128, 2), (1531, 64, (64,), 16, 9)])
def test_adapters(t, k, widths, rank, num):
    c = adapters_case(t, k, widths, rank, num, t + k, torch.bfloat16, "cuda")
    check_near(run_adapters(c, widths, num), *near64(c, widths))
    c = dict(c, bias=None, residual=None, ids=torch.sort(c["ids"])[0])
    check_near(run_adapters(c, widths, num), *near64(c, widths))


@pytest.mark.parametrize("t,k,widths,rank,num,together", [
    (257, 64, (64,), 16, 2, True), (300, 896, (896, 128, 128), 16, 8, True), (515, 2048, (1024,), 64, 11, False), (1300, 256, (512, 64, 64), 32, 20, False),
    (2049, 512, (1536,), 128, 3, True)])
def test_adapters_many_rows_both_ways(t, k, widths, rank, num, together, monkeypatch):
    """Through the large product, or in a pass of its own: the rule's choice and the other one, each within its bound."""
    c = adapters_case(t, k, widths, rank, num, t, torch.bfloat16, "cuda")
    assert ops.adapters._together(c["a"], c["b"]) == together
    ref = adapters64(**c, widths=widths)
    for way in (True, False):
        monkeypatch.setattr(ops.adapters, "_together", lambda a, b, way=way: way)
        for d in (c, dict(c, residual=None), dict(c, bias=None)):
            check_near(run_adapters(d, widths, num), *(ref if d is c else adapters64(**d, widths=widths)))
    c = adapters_case(t, k, (256, 256), rank, num, t, torch.bfloat16, "cuda", extra=False)
    for way in (True, False):
        monkeypatch.setattr(ops.adapters, "_together", lambda a, b, way=way: way)
        y = ops.adapter_linear_swiglu(c["x"], c["w"], c["a"], c["b"], c["scales"], ops.adapter_plan(c["ids"], num))
        check_near(y, *swiglu64(*adapters64(**c, widths=(256, 256), interleaved=True)))


def test_many_rows_that_are_not_finite_stay_alone(monkeypatch):
    c = adapters_case(400, 256, (256, 64, 64), 16, 4, 0, torch.bfloat16, "cuda")
    bad = c["x"].clone()
    bad[13], bad[340] = float("nan"), float("inf")
    rest = torch.ones(400, dtype=torch.bool, device="cuda")
    rest[[13, 340]] = False
    for way in (True, False):
        monkeypatch.setattr(ops.adapters, "_together", lambda a, b, way=way: way)
        assert torch.equal(run_adapters(dict(c, x=bad), (256, 64, 64), 4)[rest], run_adapters(c, (256, 64, 64), 4)[rest])


@pytest.mark.parametrize("value", [-1, 0, 2, 2 ** 31 - 1])
@pytest.mark.parametrize("t", [3, 80, 333])
def test_adapters_all_rows_alike(value, t):
    c = adapters_case(t, 128, (64, 64), 16, 3, t, torch.bfloat16, "cuda", ids=torch.full((t,), value, dtype=torch.int32))
    check_near(run_adapters(c, (64, 64), 3), *near64(c, (64, 64)))


@pytest.mark.parametrize("t,k,f,rank,num", [(1, 64, 128, 16, 1), (45, 896, 4864, 32, 9), (128, 256, 512, 16, 3), (129, 256, 512, 16, 3), (600, 256, 1280, 64, 2),
                                            (60, 128, 11008, 16, 4)])
def test_adapters_swiglu(t, k, f, rank, num):
    c = adapters_case(t, k, (f, f), rank, num, t, torch.bfloat16, "cuda", extra=False)
    y = ops.adapter_linear_swiglu(c["x"], c["w"], c["a"], c["b"], c["scales"], ops.adapter_plan(c["ids"], num))
    check_near(y, *swiglu64(*adapters64(**c, widths=(f, f), interleaved=True)))


def test_adapters_over_fp8_weights():
    """The shared product is the fp8 one; the adapters' part is unchanged."""
    for t in (5, 300):
        c = adapters_case(t, 256, (512,), 16, 3, t, torch.bfloat16, "cuda", extra=False)
        w = ops.quantize_weight_fp8(c["w"])
        none = torch.full((t,), -1, dtype=torch.int32, device="cuda")
        args = (c["x"], w, c["a"], c["b"], c["scales"])
        base = ops.adapter_linear(*args, ops.adapter_plan(none, 3)).double()
        y = ops.adapter_linear(*args, ops.adapter_plan(c["ids"], 3))
        assert torch.equal(base.bfloat16(), ops.linear(c["x"], w))
        check_near(y, *adapters64(**c, widths=(512,), base=base))
        c = adapters_case(t, 256, (256, 256), 16, 3, t, torch.bfloat16, "cuda", extra=False)
        w = ops.quantize_weight_fp8(c["w"])
        gu = ops.linear(c["x"], w).double()
        ref, err = adapters64(**dict(c, w=torch.zeros_like(c["w"])), widths=(256, 256), interleaved=True)
        y = ops.adapter_linear_swiglu(c["x"], w, c["a"], c["b"], c["scales"], ops.adapter_plan(c["ids"], 3))
        # sums rounded to bf16 before the activation where the rows are many (twice), and in `gu` here
        check_near(y, *swiglu64(gu + ref, err + 3 * 2.0 ** -8 * (gu.abs() + ref.abs())))


def test_rows_without_an_adapter_are_linears():
    for t in (1, 30, 256):
        c = dict(adapters_case(t, 256, (256, 64, 64), 16, 4, t, torch.bfloat16, "cuda"), residual=None)
        y, base = run_adapters(c, (256, 64, 64), 4), ops.linear(c["x"], c["w"], c["bias"])
        none = (c["ids"] < 0) | (c["ids"] >= 4)
        assert torch.equal(y[none], base[none])


def test_adapters_rows_are_their_own():
    """A row's result does not depend on the rows beside it, nor on the order of the batch; rows that are not finite stay alone."""
    c = adapters_case(70, 256, (256, 64, 64), 16, 4, 0, torch.bfloat16, "cuda")
    y = run_adapters(c, (256, 64, 64), 4)
    perm = torch.randperm(70, device="cuda")
    p = dict(c, x=c["x"][perm], ids=c["ids"][perm], residual=c["residual"][perm])
    assert torch.equal(run_adapters(p, (256, 64, 64), 4), y[perm])
    bad = c["x"].clone()
    bad[13], bad[40] = float("nan"), float("inf")
    rest = torch.ones(70, dtype=torch.bool, device="cuda")
    rest[[13, 40]] = False
    assert torch.equal(run_adapters(dict(c, x=bad), (256, 64, 64), 4)[rest], y[rest])


def test_adapters_views_streams_and_graph():
    c = adapters_case(21, 128, (128, 64), 16, 3, 5, torch.bfloat16, "cuda")
    ref = near64(c, (128, 64))
    wide = torch.randn(21, 400, device="cuda").bfloat16()
    for x in (wide[:, 8:136], wide[:, 3:131]):                               # a pitch, and rows that start on an odd element
        x.copy_(c["x"])
        check_near(run_adapters(dict(c, x=x), (128, 64), 3), *ref)
    odd = torch.randn(193, device="cuda").bfloat16()[1:]
    odd.copy_(c["bias"])
    check_near(run_adapters(dict(c, bias=odd), (128, 64), 3), *ref)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = run_adapters(c, (128, 64), 3)
    side.synchronize()
    check_near(y, *ref)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = run_adapters(c, (128, 64), 3)
    for shift in (1, 2):
        c["ids"].copy_((c["ids"] + shift) % 4)
        c["x"].mul_(0.5)
        graph.replay()
        check_near(y, *near64(c, (128, 64)))


def test_no_rows_and_one_row_of_an_odd_pitch():
    c = adapters_case(0, 64, (256,), 16, 2, 0, torch.bfloat16, "cuda")
    assert run_adapters(c, (256,), 2).shape == (0, 256)
    c["b"], c["a"] = c["b"], torch.cat([c["a"], c["a"]], 1)
    assert ops.adapter_linear_swiglu(c["x"], c["w"], c["a"], c["b"], c["scales"], ops.adapter_plan(c["ids"], 2)).shape == (0, 128)
    wide = torch.randn(5, 77, device="cuda").bfloat16()
    for t in (1, 2):
        c = adapters_case(t, 64, (64,), 16, 2, 1, torch.bfloat16, "cuda")
        for x in (wide[2:2 + t, 1:65], wide[2:2 + t, 8:72]):
            x.copy_(c["x"])
            check_near(run_adapters(dict(c, x=x, residual=x), (64,), 2), *near64(dict(c, residual=x), (64,)))


def test_rules_in_place_count_as_a_change():
    z, case = rules_case(2, 40, 5, 0, torch.float32, "cuda")
    before = z._version
    ops.adjust_logits(z, LogitRules(**case))
    assert z._version == before
    ops.adjust_logits(z, LogitRules(**case), out=z)
    assert z._version > before


def test_adapters_refused_by_the_kernel_entry():
    c = adapters_case(4, 64, (64,), 16, 2, 0, torch.bfloat16, "cuda")
    plan = ops.adapter_plan(c["ids"], 2)
    with pytest.raises(ValueError, match="unit inner stride"):
        ops.adapter_linear(c["x"], c["w"], c["a"], c["b"].transpose(1, 2).contiguous().transpose(1, 2), c["scales"], plan)
    with pytest.raises(ValueError, match="plan is of"):
        ops.adapter_linear(c["x"], c["w"], c["a"], c["b"], c["scales"], ops.adapter_plan(c["ids"].cpu(), 2))


@pytest.mark.parametrize("t", [1, 4, 300])
def test_adapters_refuse_the_plan_of_other_stacks(t):
    c = adapters_case(t, 64, (128, 128), 16, 2, 0, torch.bfloat16, "cuda")
    for num in (1, 3, 24):
        plan = ops.adapter_plan(c["ids"], num)
        with pytest.raises(ValueError, match="a plan for"):
            ops.adapter_linear(c["x"], c["w"], c["a"], c["b"], c["scales"], plan, (128, 128))
        with pytest.raises(ValueError, match="a plan for"):
            ops.adapter_linear_swiglu(c["x"], c["w"], c["a"], c["b"], c["scales"], plan)


@pytest.mark.parametrize("t", [5, 300])
def test_adapters_plain_form_of_fp32_rows(t):
    c = adapters_case(t, 64, (64, 32), 16, 3, t, torch.float32, "cuda")
    check_near(run_adapters(c, (64, 32), 3), *adapters64(**c, widths=(64, 32)))


def test_adapter_linear_leaves_no_graph():
    c = adapters_case(6, 64, (64,), 16, 2, 0, torch.bfloat16, "cuda")
    w, x = c["w"].clone().requires_grad_(), c["x"].clone().requires_grad_()
    y = ops.adapter_linear(x, w, c["a"], c["b"], c["scales"], ops.adapter_plan(c["ids"], 2))
    assert not y.requires_grad and torch.is_grad_enabled()
    assert torch.equal(y, ops.adapter_linear(c["x"], c["w"], c["a"], c["b"], c["scales"], ops.adapter_plan(c["ids"], 2)))
