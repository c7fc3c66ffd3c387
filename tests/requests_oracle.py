"""64-bit forms of what a request brings to a batch (rules on its logits, its adapter), written from the definitions, and how far a kernel
may be from them.  A bf16 rounding is off by 2^-8 of the value at most, an fp32 operation by 2^-24, a sum of n products in fp32 by
(n + 1) 2^-24 of the sum of their magnitudes."""
import torch

U32 = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def rules64(z, tokens=None, lens=None, prompt_lens=None, repetition=None, presence=None, frequency=None, bias_ids=None, bias_values=None, stop_ids=None,
            min_lens=None, masks=None, mask_rows=None):
    """(values, largest intermediate of a touched element or 0) on the CPU, element by element."""
    out, most = z.double().cpu().clone(), torch.zeros(z.shape, dtype=torch.float64)
    cpu = lambda t: None if t is None else t.cpu().tolist()  # noqa: E731
    tokens, lens, prompt_lens, repetition, presence, frequency, bias_ids, bias_values, stop_ids, min_lens, masks, mask_rows = map(
        cpu, (tokens, lens, prompt_lens, repetition, presence, frequency, bias_ids, bias_values, stop_ids, min_lens, masks, mask_rows))
    rows, v = z.shape
    for b in range(rows):
        hist = tokens[b] if tokens is not None else []
        n = max(0, min(lens[b] if lens is not None else len(hist), len(hist)))
        p = min(prompt_lens[b], n) if prompt_lens is not None else 0
        count, seen = {}, set()
        for i, t in enumerate(hist[:n]):
            if 0 <= t < v:
                seen.add(t)
                if i >= p:
                    count[t] = count.get(t, 0) + 1
        rep = repetition[b] if repetition is not None else 1.0
        bias = {t: x for t, x in zip(bias_ids[b], bias_values[b]) if 0 <= t < v} if bias_ids is not None else {}
        for t in seen | set(bias):
            x = out[b, t].item()
            steps = [abs(x)]
            if t in seen and rep != 1.0:
                x = x / rep if x > 0 else x * rep
                steps.append(abs(x))
            if t in count:
                f, q = (frequency[b] if frequency is not None else 0.0) * count[t], presence[b] if presence is not None else 0.0
                x = x - f - q
                steps += [abs(f), abs(q)]
            if t in bias:
                x += bias[t]
                steps.append(abs(bias[t]))
            out[b, t], most[b, t] = x, sum(steps)
        if stop_ids is not None and lens[b] < min_lens[b]:
            for t in stop_ids[b]:
                if 0 <= t < v:
                    out[b, t] = float("-inf")
        m = -1 if masks is None else mask_rows[b] if mask_rows is not None else b
        if masks is not None and 0 <= m < len(masks):
            for t in range(v):
                if not (masks[m][t // 32] >> (t % 32)) & 1:
                    out[b, t] = float("-inf")
    return out, most


def check_rules(got, z, **rules):
    """Untouched elements as they were, bit for bit; touched ones within six fp32 operations on values no larger than `most` and one rounding."""
    ref, most = rules64(z, **rules)
    g = got.cpu()
    same = ((most == 0) & ~torch.isneginf(ref)) | torch.isnan(z.cpu().double()) & ~torch.isneginf(ref)
    raw = torch.int16 if g.dtype == torch.bfloat16 else torch.int32
    keep = same & ~torch.isnan(z.cpu().double())
    assert torch.equal(g.contiguous().view(raw)[keep], z.cpu().contiguous().view(raw)[keep])
    assert torch.equal(torch.isnan(g), torch.isnan(ref))
    inf = torch.isinf(ref)
    assert torch.equal(g.double()[inf], ref[inf])
    rest = ~same & ~inf & ~torch.isnan(ref)
    tol = (half_step(g.dtype) * ref.abs() + 6 * U32 * most * (1 + half_step(g.dtype)))[rest]
    err = (g.double() - ref)[rest].abs()
    assert not (err > tol).any(), f"{(err / tol).max().item()} times the bound"


def part_of(n, widths, interleaved):
    return (torch.arange(n) // 128) % 2 if interleaved else torch.repeat_interleave(torch.arange(len(widths)), torch.tensor(widths))


def adapters64(x, w, a, b, scales, ids, widths, interleaved=False, bias=None, residual=None, base=None):
    """(projection in 64 bits, bound of its error before the last rounding): low-rank values rounded to bf16, what the adapters add (with bias
    and residual) rounded to bf16, all sums in fp32.  `base`: the projection (with its bias) as it is; what the adapters and the residual add goes on
    top in fp32."""
    dev = x.device
    x, w, a, b, s = (t.double() for t in (x, w, a, b, scales))
    n, k, r = w.shape[0], w.shape[1], b.shape[2]
    part = part_of(n, widths, interleaved).to(dev)
    d, err = torch.zeros(x.shape[0], n, dtype=torch.float64, device=dev), torch.zeros(x.shape[0], n, dtype=torch.float64, device=dev)
    u = 2.0 ** -8
    for l in range(a.shape[0]):
        rows = torch.nonzero(ids == l).flatten()
        for i in range(len(widths)):
            cols = torch.nonzero(part == i).flatten()
            if rows.numel() == 0:
                continue
            ai, bi = a[l, i * r:(i + 1) * r], b[l, cols]
            t, mag = s[l] * (x[rows] @ ai.t()), s[l].abs() * (x[rows].abs() @ ai.abs().t())
            et = u * t.abs() + (k + 3) * U32 * mag
            d[rows[:, None], cols] = t @ bi.t()
            err[rows[:, None], cols] = et @ bi.abs().t() + (r + 1) * U32 * ((t.abs() + et) @ bi.abs().t())
    for extra in (bias, residual) if base is None else (residual,):
        if extra is not None:
            d = d + extra.double()
            err = err + 2 * U32 * (d.abs() + extra.double().abs())
    if base is not None:
        return base.double() + d, err + 2 * U32 * (base.double().abs() + d.abs())
    base = x @ w.t()
    err = err + u * (d.abs() + err) + (k + 2) * U32 * (x.abs() @ w.abs().t() + d.abs())
    return base + d, err


def check_near(got, ref, err):
    """One rounding to the output's type on top of `err`."""
    tol = err + half_step(got.dtype) * (ref.abs() + err) + 1e-30
    off = (got.double() - ref).abs()
    assert torch.isfinite(got.float()).all()
    assert not (off > tol).any(), f"{(off / tol).max().item()} times the bound"


def swiglu64(z, err):
    """silu(gate) * up of an interleaved projection with error bound `err`: |silu'| <= 1.1, silu and the product a few fp32 operations (2^-18 covers
    the fast exponential)."""
    v, e = z.unflatten(-1, (-1, 2, 128)), err.unflatten(-1, (-1, 2, 128))
    g, up = v[..., 0, :].flatten(-2), v[..., 1, :].flatten(-2)
    eg, eu = e[..., 0, :].flatten(-2), e[..., 1, :].flatten(-2)
    s = g / (1 + torch.exp(-g))
    return s * up, 1.1 * eg * (up.abs() + eu) + (s.abs() + 1.1 * eg) * eu + 2.0 ** -18 * (s * up).abs()


def merged64(w, parts, widths, scale, interleaved=False):
    """The projection's weight with its adapters in it."""
    part = part_of(w.shape[0], widths, interleaved).to(w.device)
    m = w.double().clone()
    for i, p in enumerate(parts):
        if p is not None:
            cols = torch.nonzero(part == i).flatten()
            m[cols] += scale * (p[1].double() @ p[0].double())
    return m


def lora_value64(x, w, parts, widths, scale, dy, bias=None, residual=None, swiglu=False):
    """sum(dy * y) in 64 bits."""
    z = x.double() @ merged64(w, parts, widths, scale, swiglu).t()
    for extra in (bias, residual):
        if extra is not None:
            z = z + extra.double()
    if swiglu:
        v = z.unflatten(-1, (-1, 2, 128))
        g, up = v[..., 0, :].flatten(-2), v[..., 1, :].flatten(-2)
        z = g / (1 + torch.exp(-g)) * up
    return (dy.double() * z).sum()


def lora64(x, w, parts, widths, scale, dy, bias=None, residual=None, swiglu=False):
    """{name: (value, bound before the last rounding)} of y, dx and of every part's da, db: low-rank values and their gradients are rounded to bf16
    (for da and db to two bf16 numbers, 2^-8 of 2^-8 of the value), with swiglu the projection and its gradient too; sums in fp32."""
    u, u2 = 2.0 ** -8, 2.0 ** -16
    x, w, dy = x.double(), w.double(), dy.double()
    (t_rows, k), n, dev = x.shape, w.shape[0], x.device
    part = part_of(n, widths, swiglu).to(dev)
    ab = [None if p is None else (p[0].double(), p[1].double()) for p in parts]
    cols = [torch.nonzero(part == i).flatten() for i in range(len(widths))]
    z, mag, err = x @ w.t(), x.abs() @ w.abs().t(), torch.zeros(t_rows, n, dtype=torch.float64, device=dev)
    low = []
    for c, p in zip(cols, ab):
        if p is None:
            low.append(None)
            continue
        a, b = p
        t = scale * (x @ a.t())
        sums = (k + 3) * U32 * abs(scale) * (x.abs() @ a.abs().t())
        et = u * t.abs() + sums
        z[:, c] += t @ b.t()
        mag[:, c] += t.abs() @ b.abs().t()
        err[:, c] += et @ b.abs().t()
        low.append((t, u2 * t.abs() + 2 * sums))
    for extra in (bias, residual):
        if extra is not None:
            z, mag = z + extra.double(), mag + extra.double().abs()
    err = err + (k + 400) * U32 * mag
    out, ed = {}, torch.zeros_like(err)
    if swiglu:
        out["y"] = swiglu64(z, err)
        v, e = z.unflatten(-1, (-1, 2, 128)), (err + u * (z.abs() + err)).unflatten(-1, (-1, 2, 128))
        g, up, eg, eu = v[..., 0, :].flatten(-2), v[..., 1, :].flatten(-2), e[..., 0, :].flatten(-2), e[..., 1, :].flatten(-2)
        s = 1 / (1 + torch.exp(-g))
        d1 = s * (1 + g * (1 - s))                                         # silu', |silu'| <= 1.1, |silu''| <= 1/2
        dg, du = dy * up * d1, dy * g * s
        edg = dy.abs() * (eu * d1.abs() + 0.5 * eg * (up.abs() + eu)) + 2.0 ** -18 * dy.abs() * up.abs() * (1 + g.abs())
        edu = dy.abs() * 1.1 * eg + 2.0 ** -18 * (dy * g).abs()
        edg, edu = edg + u * (dg.abs() + edg), edu + u * (du.abs() + edu)
        join = lambda p, q: torch.stack([p.unflatten(-1, (-1, 128)), q.unflatten(-1, (-1, 128))], -2).flatten(-3)  # noqa: E731
        dy, ed = join(dg, du), join(edg, edu)
    else:
        out["y"] = (z, err)
    dx, edx, mdx = dy @ w, ed @ w.abs(), dy.abs() @ w.abs()
    for i, (c, p, l) in enumerate(zip(cols, ab, low)):
        if p is None:
            continue
        (a, b), (t, et), d, e = p, l, dy[:, c], ed[:, c]
        dt = scale * (d @ b)
        edt = abs(scale) * (e @ b.abs())
        edt = edt + (n + 3) * U32 * abs(scale) * ((d.abs() + e) @ b.abs())
        dx, edx, mdx = dx + dt @ a, edx + (edt + u * (dt.abs() + edt)) @ a.abs(), mdx + dt.abs() @ a.abs()
        edt = edt + u2 * (dt.abs() + edt)
        out[f"da{i}"] = (dt.t() @ x, edt.t() @ x.abs() + (2 * t_rows + 8) * U32 * (dt.abs().t() @ x.abs()))
        out[f"db{i}"] = (d.t() @ t, e.t() @ (t.abs() + et) + d.abs().t() @ et + (2 * t_rows + 8) * U32 * (d.abs().t() @ t.abs()))
    out["dx"] = (dx, edx + (n + 400) * U32 * (mdx + edx))
    return out
