"""Trained adapters beside a projection: the sm_100a kernels against the 64-bit oracle and against differences of it."""
import pytest
import torch

from polyrl_b200 import ops

from .requests_oracle import check_near, half_step, lora64, lora_value64
from .test_lora_ops_cpu import check_lora, lora_case, run_lora

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


@pytest.mark.parametrize("m,r,k,split", [(1, 8, 64, 0), (128, 16, 64, 1), (130, 24, 200, 2), (300, 48, 4096, 8), (77, 256, 512, 4), (257, 264, 1000, 0), (64, 520, 136, 1)])
@pytest.mark.parametrize("layout", [0, 1, 2, 3])
def test_thin_products(layout, m, r, k, split):
    g = torch.Generator().manual_seed(m + r)
    m8 = (m + 7) // 8 * 8 if layout >= 2 else m
    a, b = torch.randn(m8, k, generator=g).to(BF).cuda(), torch.randn(r, k, generator=g).to(BF).cuda()
    ref, mag = 0.5 * (a.double() @ b.double().t()), 0.5 * (a.double().abs() @ b.double().abs().t())
    pad = 8 if layout < 3 else 0
    got = ops.ext().lora_thin(a.t().contiguous() if layout >= 2 else a, b if layout == 0 else b.t().contiguous(), layout, 0.5, 0, pad, False, 0, split)
    if layout == 3:
        got = got.t()
    else:
        assert (got[:, r] == 1).all() and (got[:, r + 1:] == 0).all()
        got = got[:, :r]
    check_near(got, ref, (k + 2) * 2.0 ** -24 * mag)


@pytest.mark.parametrize("t,r,k,n,pad", [(70, 8, 64, 72, 0), (130, 48, 200, 136, 8), (515, 64, 512, 128, 8), (300, 136, 264, 200, 0), (257, 264, 136, 72, 8)])
def test_halves(t, r, k, n, pad):
    """A thin product in two bf16 halves, and the products over tokens that read both: as if it had 16 bits of mantissa."""
    g = torch.Generator().manual_seed(t)
    rnd = lambda *s: torch.randn(*s, generator=g).to(BF).cuda()  # noqa: E731
    x, a, dy = rnd(t, k), rnd(r, k), rnd(t, n)
    C = ops.ext()
    low = C.lora_thin(x, a, 0, 0.5, 0, pad, True)
    ref, mag = 0.5 * (x.double() @ a.double().t()), 0.5 * (x.double().abs() @ a.double().abs().t())
    both = low[:, :r].double() + low[:, r + pad:].double()
    assert low.shape[1] == 2 * r + pad and ((both - ref).abs() <= 2.0 ** -16 * ref.abs() + (k + 2) * 2.0 ** -24 * mag).all()
    assert torch.equal(low[:, :r + pad], C.lora_thin(x, a, 0, 0.5, 0, pad))
    want, most = dy.double().t() @ both, dy.double().abs().t() @ (both.abs() * (1 + 2.0 ** -7))
    for split in (0, 1, 2):
        check_near(C.lora_thin(dy, low, 2, 1.0, r, 0, False, r + pad, split), want, (2 * t + 4) * 2.0 ** -24 * most)
        check_near(C.lora_thin(dy, low, 3, 1.0, r, 0, False, r + pad, split).t(), want, (2 * t + 4) * 2.0 ** -24 * most)


@pytest.mark.parametrize("t,k,widths,ranks", [
    (1, 8, (8,), (1,)), (1, 64, (64,), (8,)), (3, 72, (40,), (5,)), (127, 896, (896, 128, 128), (8, 8, 8)), (129, 256, (128,), (16,)), (256, 200, (136,), (64,)),
    (300, 896, (896, 128, 128), (3, 0, 20)), (515, 512, (512, 64, 64), (0, 16, 16)), (640, 2048, (896,), (128,)), (1000, 264, (264, 264, 264), (96, 88, 100)),
    (2100, 1000, (520,), (64,))])
@pytest.mark.parametrize("extra", [False, True])
def test_lora_linear(t, k, widths, ranks, extra):
    check_lora(lora_case(t, k, widths, ranks, t + k, BF, "cuda", bias=extra, residual=extra))


@pytest.mark.parametrize("t,k,f,ranks", [(1, 64, 128, (8, 8)), (65, 896, 4864, (8, 8)), (300, 256, 512, (0, 5)), (301, 256, 512, (33, 0)), (777, 520, 1280, (64, 64))])
def test_lora_linear_swiglu(t, k, f, ranks):
    check_lora(lora_case(t, k, (f, f), ranks, t, BF, "cuda", swiglu=True))


@pytest.mark.parametrize("t,k,n,r,pad", [(1, 8, 8, 8, 0), (70, 72, 520, 8, 8), (130, 1032, 136, 48, 0), (515, 256, 384, 136, 8), (300, 136, 2048, 264, 0)])
def test_both_gradients_in_one_launch(t, k, n, r, pad):
    """The same values as each product by itself, split the same way."""
    g = torch.Generator().manual_seed(t + k)
    rnd = lambda *s: torch.randn(*s, generator=g).to(BF).cuda()  # noqa: E731
    x, dy, dt, low = rnd(t, k), rnd(t, n), rnd(t, 2 * r), rnd(t, 2 * r + pad)
    C = ops.ext()
    for split in (1, 2):
        if split > (t + 63) // 64:
            continue
        da, db = C.lora_grads(x, dt, dy, low, r, r + pad, split)
        assert torch.equal(da, C.lora_thin(x, dt, 3, 1.0, r, 0, False, r, split)) and torch.equal(db, C.lora_thin(dy, low, 2, 1.0, r, 0, False, r + pad, split))
    da, db = C.lora_grads(x, dt, dy, low, r, r + pad)
    both = lambda v, lo: v[:, :r].double() + v[:, lo:lo + r].double()  # noqa: E731
    for got, a, b in ((da, both(dt, r), x.double()), (db, dy.double(), both(low, r + pad))):
        check_near(got, a.t() @ b, (2 * t + 4) * 2.0 ** -24 * (a.abs().t() @ b.abs()) * (1 + 2.0 ** -7))


@pytest.mark.parametrize("t,k,f,r", [(1, 64, 128, 8), (300, 264, 256, 24), (700, 2048, 384, 16)])
def test_saved_projection_has_sixteen_bits_of_mantissa(t, k, f, r):
    """Gate and up as the backward gets them: truncated to 24 bits (2^-16); values that are not finite stay what they are."""
    g = torch.Generator().manual_seed(t)
    rnd = lambda *s: torch.randn(*s, generator=g).to(BF).cuda()  # noqa: E731
    x, w, low, b = rnd(t, k), rnd(2 * f, k), rnd(t, r), rnd(2 * f, r)
    x[0, 0], w[5, 0], w[6, 0] = float("inf"), 1.0, 0.0
    h, gu, lo = ops.ext().lora_gemm_swiglu(x, w, low, b, True)
    got = ((gu.view(torch.int16).int() << 16) | (lo.int() << 8)).view(torch.float32).double()
    ref = x.double() @ w.double().t() + low.double() @ b.double().t()
    mag = x.double().abs() @ w.double().abs().t() + low.double().abs() @ b.double().abs().t()
    fine = torch.isfinite(ref)
    assert ((got - ref).abs() <= 2.0 ** -16 * ref.abs() + (k + r + 2) * 2.0 ** -24 * mag)[fine].all()
    assert got[0, 5] == float("inf") and got[0, 6].isnan() and fine[1:].all()
    dh = rnd(t, f)
    near = ops.ext().swiglu_bwd(gu, dh, lo)
    v = got.float()
    gate, up = (v.view(t, -1, 2, 128)[:, :, i].reshape(t, f).double() for i in (0, 1))
    sig = torch.sigmoid(gate)
    want = torch.stack([dh.double() * up * sig * (1 + gate * (1 - sig)), dh.double() * gate * sig], 1).view(t, 2, -1, 128).transpose(1, 2).reshape(t, 2 * f)
    size = torch.stack([dh.double().abs() * up.abs() * (1 + gate.abs()), dh.double().abs() * gate.abs()], 1).view(t, 2, -1, 128).transpose(1, 2).reshape(t, 2 * f)
    assert ((near.double() - want).abs() <= half_step(BF) * want.abs() + 2.0 ** -19 * size + 2.0 ** -133)[1:].all()      # exp, quotients and four products of fp32


def test_adapters_part_is_not_lost_beside_a_frozen_bias():
    """Every output that a subset of the leaves asks for, and the gradient of a trained weight."""
    c = lora_case(200, 128, (128, 64), (8, 16), 0, BF, "cuda", bias=True, residual=True)
    full = run_lora(c)
    for need in (("x",), ("parts",), ()):
        for name, t in run_lora(c, need).items():
            assert torch.equal(t, full[name]), name
    leaves = {n: c[n].detach().requires_grad_() for n in ("x", "w", "bias", "residual")}
    y = ops.lora_linear(leaves["x"], leaves["w"], c["parts"], 2.0, leaves["bias"], leaves["residual"])
    dx, dw, db, dr = torch.autograd.grad(y, list(leaves.values()), c["dy"])
    assert torch.equal(dx, full["dx"]) and torch.equal(dr, c["dy"])
    d, x = c["dy"].double(), c["x"].double()
    check_near(dw, d.t() @ x, 202 * 2.0 ** -24 * (d.abs().t() @ x.abs()))
    check_near(db, d.sum(0), 202 * 2.0 ** -24 * d.abs().sum(0))


@pytest.mark.parametrize("swiglu", [False, True])
def test_gradients_against_differences(swiglu):
    """Along a random direction, the kernels' gradients give the slope of the 64-bit value: to the sum of their bounds."""
    c = lora_case(96, 128, (256, 256) if swiglu else (128, 64), (8, 4), 3, BF, "cuda", swiglu=swiglu)
    ref, got = lora64(**c), run_lora(c)
    g = torch.Generator(device="cuda").manual_seed(0)
    for name, get, put in [("dx", lambda: c["x"], lambda v: dict(c, x=v))] + [
            (f"d{n}{i}", lambda i=i, j=j: c["parts"][i][j], lambda v, i=i, j=j: dict(c, parts=[tuple(v if (a, b) == (i, j) else c["parts"][a][b] for b in (0, 1)) for a in (0, 1)]))
            for i in (0, 1) for j, n in enumerate("ab")]:
        at = get().double()
        v = torch.randn(at.shape, generator=g, device="cuda", dtype=torch.float64)
        h = 1e-4
        slope = (lora_value64(**put(at + h * v)) - lora_value64(**put(at - h * v))) / (2 * h)
        value, err = ref[name]
        tol = ((err + half_step(BF) * (value.abs() + err)) * v.abs()).sum() + 1e-6 * (value.abs() * v.abs()).sum()
        assert (slope - (got[name].double() * v).sum()).abs() <= tol
        assert (slope - (value * v).sum()).abs() <= 1e-6 * (value.abs() * v.abs()).sum()


def test_views_and_odd_starts():
    c = lora_case(150, 64, (64, 32), (8, 8), 5, BF, "cuda", bias=True, residual=True)
    full = run_lora(c)

    def shifted(t, by):
        buf = torch.empty(t.shape[0], t.shape[1] + 16, dtype=t.dtype, device="cuda")
        v = buf[:, by:by + t.shape[1]]
        v.copy_(t)
        return v

    one = {k: (v[:1] if k in ("x", "dy", "residual") else v) for k, v in c.items()}
    wide = torch.empty(3, 77, dtype=BF, device="cuda")[1:2, 5:69]             # a single row of an odd pitch
    wide.copy_(one["x"])
    for (n, t), u in zip(run_lora(dict(one, x=wide)).items(), run_lora(one).values()):
        assert torch.equal(t, u), n
    for by in (8, 3):
        o = dict(c, x=shifted(c["x"], by), w=shifted(c["w"], by), dy=shifted(c["dy"], by), residual=shifted(c["residual"], by),
                 parts=[tuple(shifted(m, by) for m in p) for p in c["parts"]])
        for name, t in run_lora(o).items():
            assert torch.equal(t, full[name]), name


def test_stream_and_graph():
    c = lora_case(260, 128, (128, 64), (8, 8), 6, BF, "cuda", residual=True)
    full = run_lora(c)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run_lora(c)
        graph = torch.cuda.CUDAGraph()
    side.synchronize()
    assert all(torch.equal(got[n], full[n]) for n in full)
    with torch.cuda.graph(graph):
        got = run_lora(c)
    c["x"].mul_(2.0)
    graph.replay()
    ref = lora64(**c)
    for name, t in got.items():
        check_near(t, *ref[name])


def test_rows_that_are_not_finite_stay_alone():
    c = lora_case(300, 128, (128,), (16,), 7, BF, "cuda")
    full = run_lora(c)
    x = c["x"].clone()
    x[17], x[299] = float("nan"), float("inf")
    got = run_lora(dict(c, x=x))
    rest = torch.ones(300, dtype=torch.bool, device="cuda")
    rest[[17, 299]] = False
    for name in ("y", "dx"):
        assert torch.equal(got[name][rest], full[name][rest])


def test_no_rows():
    c = lora_case(0, 64, (64,), (8,), 0, BF, "cuda")
    got = run_lora(c)
    assert got["y"].shape == (0, 64) and got["dx"].shape == (0, 64) and not got["da0"].any() and not got["db0"].any()
