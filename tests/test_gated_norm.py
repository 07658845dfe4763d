"""Gate, residual and norm in one pass (gated_residual_norm_with_tangent).

CPU: the oracle (oracle/block.py) against element-wise loops and differences; refusals; what watches operators, with the
oracle in place of the launches. GPU: the kernels against the oracle on the same inputs.

The kernels compute in float32 and round once, so an element is off by half a step of its type, u = finfo.eps / 2, plus
float32 errors of the terms it is made of. A sum over at most 8192 channels is at most 32 additions in a thread and 10
across threads, so a mean is off by 42 half steps of float32 of the mean magnitude; with the products and one
reciprocal root around it, every result is off by less than STEPS = 128 half steps of the magnitudes that `_reference`
adds up for it. Sums over tokens (gradients of small operands) are at most 43 additions in a wave, 4 waves and 32 more
of each of 32 strands in these tests: the same bound.
"""
import contextlib
import ctypes
import math
import weakref

import pytest
import torch

from oracle import block as ob

F32 = 2.0 ** -24
STEPS = 128
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SMALL, PER_CHANNEL = ("gate", "scale", "shift"), ("weight", "bias", "post_weight")


def _check(name, got, ref, size):
    u, tiny = torch.finfo(got.dtype).eps / 2, torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps
    tol = u * ref.abs() * (1 + 1e-3) + STEPS * F32 * size + tiny
    got, tol, ref = got.detach().cpu().double(), tol.detach(), ref.detach()
    assert torch.isfinite(got).all(), name
    err = (got - ref).abs()
    worst = float((err / tol).max()) if err.numel() else 0.0
    print(f"  {name}: worst error {worst:.2f} of its bound", flush=True)
    assert worst <= 1.0, name


# ---------------------------------------------------------------- the oracle


def test_oracle_matches_loops():
    g = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(s, generator=g, dtype=torch.float64)  # noqa: E731
    B, S, C, F = 2, 6, 8, 3
    x, y, gate, scale, shift = r(B, S, C), r(B, S, C), r(B, F, C), r(B, F, C), r(B, F, C)
    w, b, p = r(C), r(C), r(C)
    for kind in ("layer", "rms"):
        xo, n = ob.gated_norm(x, y, gate, scale, shift, w, b, p, 1e-3, kind, 0.5)
        for i in range(B):
            for s in range(S):
                f = s // 2
                ry = 1 / math.sqrt(sum(float(v) ** 2 for v in y[i, s]) / C + 1e-3)
                row = [float(x[i, s, c]) + 0.5 * float(gate[i, f, c]) * float(y[i, s, c]) * ry * float(p[c]) for c in range(C)]
                m = sum(row) / C if kind == "layer" else 0.0
                rn = 1 / math.sqrt(sum((v - m) ** 2 for v in row) / C + 1e-3)
                for c in range(C):
                    z = ((row[c] - m) * rn * float(w[c]) + float(b[c])) * (1 + float(scale[i, f, c])) + float(shift[i, f, c])
                    assert abs(row[c] - float(xo[i, s, c])) < 1e-12 and abs(z - float(n[i, s, c])) < 1e-11


def test_oracle_tangent_is_the_difference_quotient():
    g = torch.Generator().manual_seed(1)
    r = lambda *s: torch.randn(s, generator=g, dtype=torch.float64)  # noqa: E731
    ops = {n: r(1, 4, 8) for n in ("x", "y")} | {n: r(1, 2, 8) for n in SMALL} | {n: r(8) for n in PER_CHANNEL}
    along = {n: r(*ops[n].shape) for n in ("x", "y", *SMALL)}
    t = ob.gated_norm_tangent(ops, along, kind="layer", eps=1e-3)
    h = 1e-6
    moved = [ob.gated_norm(**{n: v + s * h * along.get(n, torch.zeros_like(v)) for n, v in ops.items()}, kind="layer", eps=1e-3)
             for s in (1, -1)]
    for a, b, c in zip(t, *moved):
        assert torch.allclose(a, (b - c) / (2 * h), rtol=1e-6, atol=1e-7)


# ---------------------------------------------------------------- on the GPU


def _inputs(B, S, C, F, dtype, wdtype, there, seed, layout="plain"):
    """Operands by name (those in ``there``), tangents "t...", gradients "gx", "gn"."""
    g = torch.Generator().manual_seed(seed)

    def r(*shape, sd=1.0, mean=0.0):
        return torch.randn(shape, generator=g) * sd + mean

    if layout == "slices":  # of one wider tensor
        both = r(B, S, 2 * C + 8).to(dtype)
        x = {"x": both[:, :, 8:C + 8], "y": both[:, :, C + 8:]}
    elif layout == "sbc":
        x = {n: r(S, B, C).to(dtype).transpose(0, 1) for n in ("x", "y")}
    else:
        x = {n: (r(B, S, C) + 0.5 * r(C)).to(dtype) for n in ("x", "y")}
    mods = r(B, F, 3 * C, sd=0.3).to(wdtype)  # chunks of one projection
    for i, n in enumerate(SMALL):
        x[n] = mods[..., i * C:(i + 1) * C]
    for n, mean in (("weight", 1.0), ("bias", 0.0), ("post_weight", 1.0)):
        x[n] = r(C, sd=0.2, mean=mean).to(wdtype)
    x = {n: t for n, t in x.items() if n in there}
    for n in ("x", "y", *SMALL):
        if n in x:
            x["t" + n] = r(*x[n].shape, sd=0.3).to(x[n].dtype)
    x["gx"], x["gn"] = r(B, S, C).to(dtype), r(B, S, C).to(dtype)
    return x


def _to(t, dev):
    return torch.empty_strided(t.shape, t.stride(), dtype=t.dtype, device=dev).copy_(t) if 0 not in t.stride() else t.to(dev)


def _reference(x, there, kind, eps, rs, with_gx):
    """Outputs, tangents and gradients in float64, and the magnitudes ("s...") of what each is made of."""
    ops = {n: x[n].double().requires_grad_(True) for n in ob.OPERANDS if n in there}
    S = ops["x"].shape[1]
    xo, n = ob.gated_norm(**ops, eps=eps, kind=kind, rs=rs)
    outs, into = ((xo, n), (x["gx"].double(), x["gn"].double())) if with_gx else ((n,), (x["gn"].double(),))
    ref = {"d" + k: g for k, g in zip(ops, torch.autograd.grad(outs, list(ops.values()), into))}
    ref["x'"], ref["n"] = xo.detach(), n.detach()
    ref["tx'"], ref["tn"] = ob.gated_norm_tangent(ops, {k[1:]: v for k, v in x.items() if k.startswith("t")}, kind=kind, eps=eps, rs=rs)

    v = {k: t.detach() for k, t in ops.items()}
    mean = lambda t: t.mean(-1, keepdim=True)  # noqa: E731
    rows = {k: ob.rows_of(v[k], S) for k in SMALL if k in v}
    one, zero = torch.ones(()).double(), torch.zeros(()).double()
    G = abs(rs) * rows.get("gate", one).abs()
    s = {}
    yn = yr = None
    if "y" in v:
        y, ty = v["y"], x["ty"].double()
        sy, sty = y.abs(), ty.abs()
        if "post_weight" in v:
            yr = (mean(y.pow(2)) + eps).rsqrt()
            yn, p = y * yr, v["post_weight"].abs()
            sy, sty = yn.abs() * p, yr * (ty.abs() + yn.abs() * mean((yn * ty).abs())) * p
        size = v["x"].abs() + G * sy
        st = x["tx"].double().abs() + G * sty
        if "tgate" in x:
            st = st + abs(rs) * ob.rows_of(x["tgate"].double(), S).abs() * sy
    else:
        sy, size, st = None, v["x"].abs(), x["tx"].double().abs()
    s["x'"], s["tx'"] = size, st
    z = ref["x'"]
    c = z - mean(z) if kind == "layer" else z
    r = (mean(c.pow(2)) + eps).rsqrt()
    N = c * r
    rho = 1 + r.pow(2) * mean(c.abs() * size)          # relative error of r
    eN = r * (size + mean(size)) + N.abs() * rho       # error of N
    w, b = v.get("weight", one).abs(), v.get("bias", zero).abs()
    one_s = 1 + rows.get("scale", zero).abs()
    A = w * (1 + rows.get("scale", zero)).abs()
    s["n"] = (eN + N.abs()) * w * one_s + b * one_s + rows.get("shift", zero).abs()
    t = ref["tx'"]
    s["tn"] = w * one_s * r * (rho * (st + mean(st) + N.abs() * mean(N.abs() * st)) + eN * mean((N * t).abs()) + N.abs() * mean(eN * t.abs()))
    if "tscale" in x:
        s["tn"] = s["tn"] + ob.rows_of(x["tscale"].double(), S).abs() * ((eN + N.abs()) * w + b)
    if "tshift" in x:
        s["tn"] = s["tn"] + ob.rows_of(x["tshift"].double(), S).abs()
    gn = x["gn"].double()
    a = (gn * A).abs()
    sa = gn.abs() * w * one_s
    sdx = (x["gx"].double().abs() if with_gx else zero) + r * rho * (sa + mean(sa) + N.abs() * mean(sa * N.abs())) + \
        r * (eN * mean(a * N.abs()) + N.abs() * mean(sa * eN))
    s["dx"] = sdx
    per = lambda q: q.view(q.shape[0], -1, S // F_of(v), q.shape[2]).sum(2)  # noqa: E731
    if "y" in v:
        sdy = G * sdx
        if "post_weight" in v:
            s["dpost_weight"] = (sdy * yn.abs()).sum((0, 1))
            q = sdy * v["post_weight"].abs()
            sdy = yr * (q + yn.abs() * mean(q * yn.abs()))
        s["dy"] = sdy
        if "gate" in v:
            s["dgate"] = abs(rs) * per(sdx * sy)
    if "scale" in v:
        s["dscale"] = per(gn.abs() * ((N.abs() + eN) * w + b))
    if "shift" in v:
        s["dshift"] = per(gn.abs())
    if "weight" in v:
        s["dweight"] = (gn.abs() * one_s * (N.abs() + eN)).sum((0, 1))
    if "bias" in v:
        s["dbias"] = (gn.abs() * one_s * one).sum((0, 1))
    return ref, s


def F_of(v):
    return next((v[k].shape[1] for k in SMALL if k in v), 1)


def _call(d, kind="layer", eps=1e-6, rs=1.0, tangents=True):
    from dmad_amd import gated_residual_norm_with_tangent

    pair = lambda n: (d.get(n), d.get("t" + n) if tangents else None)  # noqa: E731
    return gated_residual_norm_with_tangent(pair("x"), pair("y"), *(pair(n) for n in SMALL), *(d.get(n) for n in PER_CHANNEL), eps,
                                            kind, rs)


ALL = ob.OPERANDS
WAN = ("x", "y", "gate", "scale", "shift")
CASES = [
    # B, S, C, F, dtype, small operands' dtype, norm, operands, layout, residual scale
    (1, 1, 8, 1, "bf16", "bf16", "layer", WAN, "plain", 1.0),
    (2, 5, 16, 5, "fp16", "fp32", "rms", ALL, "plain", 0.5),
    (1, 256, 128, 1, "fp32", "fp32", "layer", WAN, "plain", 1.0),
    (3, 37, 520, 1, "bf16", "fp32", "layer", ALL, "slices", 1.0),
    (2, 42, 512, 21, "fp16", "fp16", "layer", WAN, "sbc", 1.0),
    (2, 63, 1536, 3, "bf16", "bf16", "layer", ("x", "y", "gate", "scale", "shift", "weight", "bias"), "plain", 1.0),
    (1, 300, 1536, 1, "bf16", "fp32", "layer", ("x", "weight", "bias"), "plain", 1.0),
    (3, 99, 1536, 1, "fp16", "fp32", "rms", ("x", "y", "weight", "post_weight"), "plain", 1.0),
    (1, 40, 1544, 1, "fp32", "fp32", "rms", ALL, "sbc", -2.0),
    (1, 33, 2048, 33, "bf16", "fp32", "rms", ("x", "scale", "shift"), "plain", 1.0),
    (2, 20, 2056, 2, "bf16", "bf16", "layer", WAN, "slices", 1.0),
    (32, 1, 5120, 1, "bf16", "bf16", "layer", WAN, "plain", 1.0),
    (1, 130, 5120, 1, "bf16", "fp32", "layer", ALL, "plain", 1.0),
    (1, 9, 5120, 9, "fp16", "fp32", "rms", ("x", "y", "gate", "shift", "post_weight"), "plain", 0.25),
    (1, 31, 6152, 1, "fp32", "fp32", "layer", ("x", "y", "gate", "weight"), "plain", 1.0),
    (2, 12, 8192, 4, "bf16", "bf16", "rms", ALL, "plain", 1.0),
    (1, 7, 8192, 1, "fp16", "fp16", "layer", ("x", "y", "scale"), "slices", 1.0),
    (2, 1024, 64, 1, "bf16", "fp32", "layer", WAN, "plain", 1.0),
    (1, 1600, 24, 1, "fp32", "fp32", "rms", ("x", "y"), "plain", 1.0),
    (2, 3500, 40, 1, "bf16", "fp32", "layer", ALL, "plain", 1.0),
]


@pytest.mark.gpu
@pytest.mark.parametrize("B,S,C,F,dtype,wdtype,kind,there,layout,rs", CASES)
def test_forward_tangent_backward(gpu, B, S, C, F, dtype, wdtype, kind, there, layout, rs):
    print(f"case gated norm B={B} S={S} C={C} F={F} {dtype} {wdtype} {kind} {there} {layout}", flush=True)
    x = _inputs(B, S, C, F, DTYPES[dtype], DTYPES[wdtype], there, seed=C + S, layout=layout)
    branch = "y" in there
    ref, size = _reference(x, there, kind, 1e-6, rs, branch)
    d = {n: _to(t, gpu) for n, t in x.items()}
    leaves = [d[n].requires_grad_(True) for n in ALL if n in there]
    (xo, txo), (n, tn) = _call(d, kind, 1e-6, rs)
    assert n.requires_grad and not tn.requires_grad and n.is_contiguous() and n.shape == (B, S, C) and n.dtype == DTYPES[dtype]
    if branch:
        assert xo.requires_grad and not txo.requires_grad
    else:
        assert xo is d["x"] and txo is d["tx"]
    outs, into = ((xo, n), (d["gx"], d["gn"])) if branch else ((n,), (d["gn"],))
    grads = torch.autograd.grad(outs, leaves, into, retain_graph=True)
    torch.cuda.synchronize()
    for name, got in ((("x'", xo), ("tx'", txo)) if branch else ()) + (("n", n), ("tn", tn)):
        _check(name, got, ref[name], size[name])
    for name, leaf, got in zip([n for n in ALL if n in there], leaves, grads):
        assert got.dtype == leaf.dtype and got.shape == leaf.shape
        _check("d" + name, got, ref["d" + name], size["d" + name])
    # the same again bit for bit; the primal alone is the same
    for a, b in zip(torch.autograd.grad(outs, leaves, into), grads):
        assert torch.equal(a, b)
    with torch.no_grad():
        (xp, none), (np_, tnone) = _call(d, kind, 1e-6, rs, tangents=False)
    assert none is None and tnone is None and torch.equal(np_, n) and torch.equal(xp, xo)


@pytest.mark.gpu
@pytest.mark.parametrize("C", [512, 5120])
def test_calls_past_the_caches(gpu, C):
    """Calls of more than the caches hold (256 MB): bit for bit what their chunks of tokens give, and the gradient of a
    chunk's shift, a sum of 1500 terms in float32 in some order: n eps / 2 times the sum of their sizes, and its rounding."""
    parts, n = 4, 1500 * (5120 // C)
    S = parts * n
    assert 6 * S * C * 2 > 256e6 > 8 * n * C * 2
    g = torch.Generator(device=gpu).manual_seed(3)
    d = {k: torch.randn(1, S, C, generator=g, device=gpu).to(torch.bfloat16) for k in ("x", "tx", "y", "ty", "gx", "gn")}
    d.update({k: torch.randn(1, parts, C, generator=g, device=gpu) for k in ("gate", "scale", "shift")})

    def run(rows, group):
        x, y = (d[k][:, rows].detach().requires_grad_() for k in "xy")
        small = {k: d[k][:, group].detach().requires_grad_() for k in ("gate", "scale", "shift")}
        print(f"case past caches C={C} rows={x.shape[1]}", flush=True)
        (xo, txo), (o, to) = _call({"x": x, "tx": d["tx"][:, rows], "y": y, "ty": d["ty"][:, rows], **small})
        torch.autograd.backward((xo, o), (d["gx"][:, rows], d["gn"][:, rows]))
        return (xo.detach(), txo, o.detach(), to, x.grad, y.grad), small["shift"].grad

    every = slice(None)
    whole, dshift = run(every, every)
    assert all(torch.isfinite(t).all() for t in whole)
    for i in range(parts):
        rows = slice(i * n, (i + 1) * n)
        some, part = run(rows, slice(i, i + 1))
        for a, b in zip(whole, some):
            assert torch.equal(a[:, rows], b)
        ref, size = d["gn"][0, rows].double().sum(0), d["gn"][0, rows].double().abs().sum(0)
        for got in (dshift[0, i], part[0, 0]):
            assert ((got.double() - ref).abs() <= (n + 1) * 2.0 ** -24 * size).all()


def _check_within(name, got, ref, size, steps):
    u, tiny = torch.finfo(got.dtype).eps / 2, torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps
    tol = u * ref.abs() * (1 + 1e-3) + steps * F32 * size + tiny
    assert torch.isfinite(got).all(), name
    worst = float(((got.double() - ref).abs() / tol).max())
    print(f"  {name}: worst error {worst:.2f} of its bound", flush=True)
    assert worst <= 1.0, name


def _on_device(gpu, B, S, C, F, dtype, wdtype, there, seed):
    """As _inputs(), made on the device, for large calls."""
    g = torch.Generator(device=gpu).manual_seed(seed)
    r = lambda *shape, sd=1.0, mean=0.0: torch.randn(shape, generator=g, device=gpu) * sd + mean  # noqa: E731
    x = {n: r(B, S, C).to(dtype) for n in ("x", "y", "tx", "ty", "gx", "gn")}
    x.update({n: r(B, F, C, sd=0.3).to(wdtype) for n in ("gate", "scale", "shift")})
    x.update({n: r(C, sd=0.2, mean=m).to(wdtype) for n, m in (("weight", 1.0), ("bias", 0.0), ("post_weight", 1.0))})
    return {n: t for n, t in x.items() if n in there or n in ("tx", "gx", "gn") or (n == "ty" and "y" in there)}


@pytest.mark.gpu
@pytest.mark.parametrize("S,C,F,dtype,wdtype,kind,there,rs", [
    (60000, 512, 4, "bf16", "fp32", "layer", ALL, 1.0),
    (6000, 5120, 3, "fp16", "fp16", "rms", ALL, 0.5),
    (12000, 1544, 1, "fp32", "fp32", "layer", ("x", "y", "weight", "post_weight"), -1.0),
    (30000, 1536, 4, "bf16", "bf16", "layer", ("x", "scale", "weight", "bias"), 1.0),
    (90000, 504, 1, "bf16", "fp32", "rms", ("x", "weight"), 1.0),
    (31000, 1536, 2, "fp16", "fp32", "layer", WAN, 1.0),
])
def test_gradients_of_calls_past_the_caches(gpu, S, C, F, dtype, wdtype, kind, there, rs):
    """Every gradient of calls of more than the caches hold, with and without a branch and a norm after it, against
    float64. Sums over tokens are up to 30 additions in a wave, 4 waves, and 40 of each of 32 strands, together fewer than
    the module's bound counts."""
    d = _on_device(gpu, 1, S, C, F, DTYPES[dtype], DTYPES[wdtype], there, C)
    assert (6 if "y" in there else 3) * S * C * d["x"].element_size() > 2 ** 28
    branch = "y" in there
    print(f"case past caches S={S} C={C} F={F} {dtype} {wdtype} {kind} {there}", flush=True)
    leaves = [d[n].requires_grad_(True) for n in ALL if n in there]
    (xo, _), (n, _) = _call(d, kind, 1e-6, rs, tangents=False)
    outs, into = ((xo, n), (d["gx"], d["gn"])) if branch else ((n,), (d["gn"],))
    grads = torch.autograd.grad(outs, leaves, into)
    torch.cuda.synchronize()
    ref, size = _reference({k: t.detach() for k, t in d.items()}, there, kind, 1e-6, rs, branch)
    for name, leaf, got in zip([n for n in ALL if n in there], leaves, grads):
        assert got.dtype == leaf.dtype and got.shape == leaf.shape
        _check_within("d" + name, got, ref["d" + name], size["d" + name], STEPS)


@pytest.mark.gpu
def test_more_groups_than_rows_of_a_grid(gpu):
    """34000 groups of two tokens, whose gradients take two launches; those of the weights are sums over 34000 workgroups,
    of which a strand adds 1063 after one another: as many half steps more."""
    B, F, C = 2, 17000, 64
    d = _on_device(gpu, B, 2 * F, C, F, torch.bfloat16, torch.float32, ALL, 8)
    assert B * F > 32768
    leaves = [d[n].requires_grad_(True) for n in ALL]
    print(f"case groups {B * F}", flush=True)
    (xo, _), (n, _) = _call(d, tangents=False)
    grads = torch.autograd.grad((xo, n), leaves, (d["gx"], d["gn"]))
    torch.cuda.synchronize()
    ref, size = _reference({k: t.detach() for k, t in d.items()}, ALL, "layer", 1e-6, 1.0, True)
    for name, got in zip(ALL, grads):
        _check_within("d" + name, got, ref["d" + name], size["d" + name], STEPS + (1063 if name in PER_CHANNEL else 0))


@pytest.mark.gpu
@pytest.mark.parametrize("S,C", [(270000, 8192), (4400000, 504)])
def test_more_elements_than_32_bits_count(gpu, S, C):
    """The last tokens of calls of more than 2^31 elements: bit for bit what a call of them alone gives."""
    F, n = S // 1000, 2000
    assert S * C > 2 ** 31
    print(f"case beyond 32 bits S={S} C={C}", flush=True)
    d = {k: torch.empty(1, S, C, device=gpu, dtype=torch.bfloat16) for k in ("x", "tx", "y", "ty", "gx", "gn")}
    for t in d.values():
        t.view(-1, 1000 * C)[:] = torch.randn(1000 * C, device=gpu).to(torch.bfloat16)
        t[:, -n:] = torch.randn(n, C, device=gpu).to(torch.bfloat16)
    d.update({k: torch.randn(1, F, C, device=gpu) for k in ("gate", "scale", "shift")})

    def run(rows, groups):
        y = {k: t[:, groups if k in SMALL else rows] for k, t in d.items()}
        leaves = [y[k].detach().requires_grad_() for k in WAN]
        y.update(zip(WAN, leaves))
        (xo, txo), (o, to) = _call(y)
        grads = torch.autograd.grad((xo, o), leaves[:2], (y["gx"], y["gn"]))
        return [t.detach()[:, -n:].clone() for t in (xo, txo, o, to, *grads)]

    for a, b in zip(run(slice(None), slice(None)), run(slice(S - n, S), slice(F - n // 1000, F))):
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("wdtype", ["same", "fp32"])
@pytest.mark.parametrize("C", [512, 1536])
@pytest.mark.parametrize("there", [("x", "scale", "shift", "weight", "bias"), WAN, ALL])
def test_bits_do_not_depend_on_tangents_or_gradients(gpu, dtype, wdtype, C, there):
    """Over a million elements: outputs with tangents and without, gradients with those of the weights and without."""
    d = _on_device(gpu, 1, 2 ** 21 // C // 8 * 8, C, 8, DTYPES[dtype], DTYPES[dtype if wdtype == "same" else wdtype], there, 3)
    print(f"case bits {dtype} {wdtype} C={C} {there}", flush=True)

    def run(tangents, leaves):
        ops = {n: t.detach().requires_grad_(n in leaves) for n, t in d.items()}
        (xo, txo), (n, tn) = _call(ops, tangents=tangents)
        outs, into = ((xo, n), (d["gx"], d["gn"])) if "y" in there else ((n,), (d["gn"],))
        return [xo.detach(), n.detach()], dict(zip(leaves, torch.autograd.grad(outs, [ops[m] for m in leaves], into)))

    every = [n for n in ALL if n in there]
    outs, grads = run(True, every)
    for tangents, leaves in ((False, every), (False, [n for n in every if n not in PER_CHANNEL]), (False, ["x"])):
        o, g = run(tangents, leaves)
        assert all(torch.equal(a, b) for a, b in zip(o, outs))
        for n in leaves:
            assert torch.equal(g[n], grads[n]), n


@pytest.mark.gpu
@pytest.mark.parametrize("C", [64, 1536])
def test_one_shape_at_many_places(gpu, C):
    """Calls of one shape, some of whose operands start off 16 bytes: what is planned for the shape holds for none else."""
    d = {k: torch.randn(2, 6, C, device=gpu).to(torch.bfloat16) for k in ("x", "y")}
    d["gate"] = torch.randn(2, 1, C, device=gpu)

    def off(t):
        at = torch.empty(t.numel() + 1, device=gpu, dtype=t.dtype)[1:].view(t.shape)
        return at.copy_(t)

    (want, _), (wn, _) = _call(d)
    for moved in ((), ("x",), ("gate",), ("y", "x"), ()):
        (xo, _), (n, _) = _call({k: off(t) if k in moved else t for k, t in d.items()})
        assert torch.equal(xo, want) and torch.equal(n, wn)
    with pytest.raises(ValueError, match="eps"):
        _call(d, eps=-1.0)
    with pytest.raises(ValueError, match="residual_scale"):
        _call(d, rs=math.inf)


@pytest.mark.gpu
def test_gradient_is_the_difference_quotient(gpu):
    """fp32 gradients against central differences of the kernel's own outputs. With step h = 2^-6 the quotient of
    sum(x' gx + n gn) is off by h^2 / 6 times a third derivative of order 10 and by the outputs' float32 errors, 64 half
    steps of the sum's magnitude over h: together under 1e-3 of the gradient's size here."""
    x = _inputs(1, 6, 32, 2, torch.float32, torch.float32, ALL, 3)
    d = {n: t.to(gpu) for n, t in x.items()}
    names = list(ALL)
    leaves = [d[n].clone().requires_grad_(True) for n in names]
    g = torch.Generator().manual_seed(4)
    along = [torch.randn(t.shape, generator=g).to(gpu) for t in leaves]

    def loss(ts):
        (xo, _), (n, _) = _call(dict(zip(names, ts)), tangents=False)
        return (xo.double() * d["gx"].double()).sum() + (n.double() * d["gn"].double()).sum()

    grads = torch.autograd.grad(loss(leaves), leaves)
    h = 2.0 ** -6
    with torch.no_grad():
        for i, (gr, a) in enumerate(zip(grads, along)):
            moved = [loss([t + s * h * a if j == i else t for j, t in enumerate(leaves)]) for s in (1, -1)]
            num, size = float((moved[0] - moved[1]) / (2 * h)), float((gr * a).abs().sum())
            assert abs(float((gr.double() * a.double()).sum()) - num) <= 1e-3 * size, names[i]


@pytest.mark.gpu
@pytest.mark.parametrize("C", [64, 5120])
def test_partial_gradients(gpu, C):
    """A loss of one output, and operands that want none: what is left is what it is with all of them."""
    x = _inputs(2, 12, C, 2, torch.bfloat16, torch.float32, ALL, 5)
    d = {n: t.to(gpu) for n, t in x.items()}

    def grads(leaves, use):
        y = {n: t.detach().requires_grad_(n in leaves) for n, t in d.items()}
        (xo, _), (n, _) = _call(y, tangents=False)
        outs = {"x'": (xo, d["gx"]), "n": (n, d["gn"])}
        return dict(zip(leaves, torch.autograd.grad([outs[u][0] for u in use], [y[m] for m in leaves], [outs[u][1] for u in use],
                                                    allow_unused=True)))

    everything = grads(list(ALL), ["x'", "n"])
    for only in (["x"], ["gate"], ["weight", "y"], ["bias"], ["shift", "scale"], ["post_weight"]):
        for n, t in grads(only, ["x'", "n"]).items():
            assert torch.equal(t, everything[n]), n
    # of x' alone: the norm behind it adds nothing
    zero = {n: t.clone() for n, t in d.items()}
    zero["gn"].zero_()
    kept, d = d, zero
    want = grads(list(ALL), ["x'", "n"])
    d = kept
    got = grads(list(ALL), ["x'"])
    for n in ALL:
        assert torch.equal(got[n], want[n]), n
    # of n alone
    zero = {n: t.clone() for n, t in d.items()}
    zero["gx"].zero_()
    kept, d = d, zero
    want = grads(list(ALL), ["x'", "n"])
    d = kept
    got = grads(list(ALL), ["n"])
    for n in ALL:
        assert torch.equal(got[n], want[n]), n


@pytest.mark.gpu
@pytest.mark.parametrize("C", [256, 1536])
def test_a_row_per_token_takes_no_workspace(gpu, C):
    """Gate, scale and shift per token, whose gradients the workgroups write themselves: the backward allocates them and
    those of x and y, and nothing beside them."""
    S = 2048
    x = _inputs(1, S, C, S, torch.bfloat16, torch.bfloat16, WAN, 23)
    d = {n: t.to(gpu).contiguous() for n, t in x.items()}
    leaves = [d[n].requires_grad_(True) for n in WAN]
    (xo, _), (n, _) = _call(d, tangents=False)
    print(f"case a row per token C={C}", flush=True)
    before = torch.cuda.memory_stats()["requested_bytes.all.current"]
    torch.cuda.reset_peak_memory_stats()
    grads = torch.autograd.grad((xo, n), leaves, (d["gx"], d["gn"]))
    took = torch.cuda.memory_stats()["requested_bytes.all.peak"] - before
    assert took == sum(t.numel() * t.element_size() for t in grads)
    ref, size = _reference(x, WAN, "layer", 1e-6, 1.0, True)
    for name, got in zip(WAN, grads):
        _check("d" + name, got, ref["d" + name], size["d" + name])


@pytest.mark.gpu
def test_no_second_derivative(gpu):
    x = _inputs(1, 4, 32, 1, torch.float32, torch.float32, WAN, 6)
    d = {n: t.to(gpu) for n, t in x.items()}
    d["x"].requires_grad_(True)

    def grad(create_graph):
        (xo, _), (n, _) = _call(d, tangents=False)
        return torch.autograd.grad(n.square().sum() + xo.sum(), d["x"], create_graph=create_graph)[0]

    g = grad(True)
    assert torch.equal(g.detach(), grad(False))
    with pytest.raises(RuntimeError, match="differentiate twice"):
        g.sum().backward()


@pytest.mark.gpu
def test_broadcast_unaligned_and_mixed_operands(gpu):
    """Expanded operands are read in place and their gradients summed by autograd; rows that start unaligned are copied;
    small operands of several types are read as float32."""
    g = torch.Generator().manual_seed(7)
    r = lambda *s: torch.randn(s, generator=g)  # noqa: E731
    x, y = (r(2, 6, 64).bfloat16().to(gpu) for _ in range(2))
    gate = r(1, 1, 64).to(gpu).requires_grad_(True)
    shift = r(64).to(gpu).requires_grad_(True)
    one = r(1, 6, 64).bfloat16().to(gpu).requires_grad_(True)
    a = _call(dict(x=one.expand(2, 6, 64), y=y, gate=gate.expand(2, 1, 64), shift=shift.expand(2, 1, 64)))
    b = _call(dict(x=one.detach().repeat(2, 1, 1), y=y, gate=gate.detach().repeat(2, 1, 1), shift=shift.detach().repeat(2, 1, 1)))
    assert torch.equal(a[0][0], b[0][0]) and torch.equal(a[1][0], b[1][0])
    a[1][0].float().sum().backward()
    assert one.grad.shape == one.shape and gate.grad.shape == gate.shape and shift.grad.shape == shift.shape
    assert torch.equal(shift.grad, torch.full_like(shift.grad, 12.0))
    flat = torch.zeros(2 * 6 * 64 + 1, device=gpu, dtype=torch.bfloat16)
    flat[1:] = x.reshape(-1)
    odd = flat[1:].view(2, 6, 64)
    small = torch.zeros(2 * 64 + 1, device=gpu)
    small[1:] = 0.25
    c = _call(dict(x=odd, y=y, gate=small[1:].view(2, 1, 64)))
    e = _call(dict(x=x, y=y, gate=torch.full((2, 1, 64), 0.25, device=gpu)))
    assert torch.equal(c[1][0], e[1][0]) and torch.equal(c[0][0], e[0][0])
    w = r(64).half().to(gpu)
    a = _call(dict(x=x, y=y, gate=gate.detach().expand(2, 1, 64).bfloat16(), weight=w))
    b = _call(dict(x=x, y=y, gate=gate.detach().expand(2, 1, 64).bfloat16().float(), weight=w.float()))
    assert torch.equal(a[1][0], b[1][0])


@pytest.mark.gpu
@pytest.mark.parametrize("C", [32, 4096])
def test_extremes(gpu, C):
    """Rows of zeros, far from zero, infinite and NaN: each stays with its own row and its own results."""
    g = torch.Generator().manual_seed(8)
    x = torch.randn(1, 9, C, generator=g)
    x[0, 1] = 0.0
    x[0, 2] += 1000.0
    x[0, 3] *= 1e15
    x[0, 4] *= 1e-15
    y = torch.randn(1, 9, C, generator=g)
    y[0, 1] = 0.0
    y[0, 3:5] = 0.0
    v = {"x": x, "y": y, "gx": torch.zeros(1, 9, C), "gn": torch.randn(1, 9, C, generator=g), "tx": torch.zeros(1, 9, C),
         "ty": torch.zeros(1, 9, C)}
    for kind in ("layer", "rms"):
        ref, size = _reference(v, ("x", "y"), kind, 1e-6, 1.0, True)
        d = {n: t.to(gpu) for n, t in v.items()}
        (xo, _), (n, _) = _call(d, kind, tangents=False)
        _check("x'", xo, ref["x'"], size["x'"])
        _check("n", n, ref["n"], size["n"])
        bad = {k: t.clone() for k, t in d.items()}
        bad["x"][0, 5, 3], bad["y"][0, 6, 0] = math.inf, math.nan
        for t in (bad["x"], bad["y"]):
            t.requires_grad_(True)
        (xb, _), (nb, _) = _call(bad, kind, tangents=False)
        for row in range(9):
            if row in (5, 6):
                assert not torch.isfinite(nb[0, row]).all()
            else:
                assert torch.equal(nb[0, row], n[0, row]) and torch.equal(xb[0, row], xo[0, row])
        dx, dy = torch.autograd.grad(nb, (bad["x"], bad["y"]), d["gn"])
        rows = [i for i in range(9) if i not in (5, 6)]
        assert torch.isfinite(dx[0, rows]).all() and torch.isfinite(dy[0, rows]).all()
        # eps = 0: a row of zeros (constant, for the layer norm) has no norm, the others have
        (_, _), (n0, _) = _call(d, kind, eps=0.0, tangents=False)
        assert torch.isnan(n0[0, 1]).all() and torch.isfinite(n0[0, 2:]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(0, 4, 32), (2, 0, 32)])
def test_no_rows(gpu, shape):
    x = torch.zeros(shape, device=gpu, requires_grad=True)
    y = torch.zeros(shape, device=gpu, requires_grad=True)
    gate, w = torch.ones(shape[0], 1, 32, device=gpu, requires_grad=True), torch.ones(32, device=gpu, requires_grad=True)
    (xo, _), (n, _) = _call(dict(x=x, y=y, gate=gate, weight=w))
    grads = torch.autograd.grad(xo.sum() + n.sum(), (x, y, gate, w))
    assert n.shape == shape and xo.shape == shape
    for g, t in zip(grads, (x, y, gate, w)):
        assert g.shape == t.shape and torch.equal(g, torch.zeros_like(g))


@pytest.mark.gpu
@pytest.mark.parametrize("C,dtype", [(256, "bf16"), (5120, "bf16"), (1536, "fp32")])
def test_captured_and_on_another_stream(gpu, C, dtype):
    x = _inputs(2, 300, C, 2, DTYPES[dtype], torch.float32, ALL, 15)
    d = {n: t.to(gpu) for n, t in x.items()}

    def step():
        y = {n: t.detach().requires_grad_(n in ALL) for n, t in d.items()}
        (xo, txo), (n, tn) = _call(y)
        return [xo.detach(), txo, n.detach(), tn, *torch.autograd.grad((xo, n), [y[m] for m in ALL], (d["gx"], d["gn"]))]

    ref = [t.clone() for t in step()]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(other, ref))
    # two graphs at once, each with scratch of its own
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for graph in graphs:
        with torch.cuda.graph(graph):
            outs.append(step())
    for _ in range(3):
        junk = torch.randn(1024, 1024, device=gpu)
        (junk @ junk).sum().item()
        for o in outs:
            for t in o:
                t.zero_()
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for o in outs:
            assert all(torch.equal(a, b) for a, b in zip(o, ref))


# ---------------------------------------------------------------- refusals


def test_refusals_on_the_cpu():
    from dmad_amd import gated_residual_norm_with_tangent

    with pytest.raises(RuntimeError, match="GPU only"):
        gated_residual_norm_with_tangent((torch.randn(1, 2, 32), None))


REFUSED = [
    (ValueError, "x must be given", dict(x=None)),
    (ValueError, r"\[B, S, C\]", dict(x=(6, 32))),
    (NotImplementedError, "channels", dict(x=(2, 6, 36))),
    (NotImplementedError, "channels", dict(x=(2, 6, 8200))),
    (NotImplementedError, "dtype", dict(x=torch.float64)),
    (ValueError, "y must have", dict(y=(2, 5, 32))),
    (ValueError, "y must have", dict(y=torch.float16)),
    (ValueError, "belong to y", dict(y=None, ty=None)),
    (ValueError, "tangents of both", dict(ty=None)),
    (ValueError, "tangents of both", dict(tx=None)),
    (ValueError, "a tangent of gate", dict(tx=None, ty=None)),
    (ValueError, "a tangent of shift", dict(shift=None)),
    (ValueError, "shape and type", dict(tx=torch.float16)),
    (ValueError, "shape and type", dict(tscale=(2, 1, 32))),
    (ValueError, "one F", dict(gate=(2, 4, 32), tgate=(2, 4, 32))),
    (ValueError, "one F", dict(shift=(2, 1, 32), tshift=(2, 1, 32))),
    (ValueError, "one F", dict(scale=(1, 3, 32), tscale=(1, 3, 32))),
    (ValueError, "operands' type or float32", dict(gate=torch.float64, tgate=None)),
    (ValueError, "weight must be", dict(weight=(16,))),
    (ValueError, "bias must be", dict(bias=torch.float64)),
    (ValueError, "eps", dict(eps=-1.0)),
    (ValueError, "eps", dict(eps=math.nan)),
    (ValueError, "norm", dict(kind="batch")),
    (ValueError, "residual_scale", dict(rs=math.inf)),
]


def _small(device="cpu", grad=False, dtype=torch.float32):
    """A little call with everything in it."""
    x = {n: t.to(device, dtype).clone() for n, t in _inputs(2, 6, 32, 3, torch.float32, torch.float32, ALL, 3).items()}
    for n in ALL:
        x[n].requires_grad_(grad)
    return x


@pytest.mark.parametrize("error,match,over", REFUSED)
def test_refusals(monkeypatch, error, match, over):
    """The checks are the host's: refused before anything is launched."""
    _mock_kernels(monkeypatch)
    x = _small()
    how = {k: over[k] for k in ("kind", "eps", "rs") if k in over}
    for n, v in over.items():
        if n in how:
            continue
        x[n] = None if v is None else torch.zeros(v) if isinstance(v, tuple) else x[n].detach().to(v)
    with pytest.raises(error, match=match):
        _call(x, **how)


def _sizes(**over):
    from dmad_amd import _native as nat

    a = dict(dtype=0, wdtype=0, norm=0, B=1, S=4, C=64, F=2)
    strides = dict(x=(256, 64, 1), small=(128, 64, 1))
    for k, v in over.items():
        (strides if k in strides else a)[k] = v
    arr = lambda s: (ctypes.c_int64 * 3)(*s)  # noqa: E731
    return nat.GatedNormSizes(*a.values(), *(arr(strides["x"]) for _ in range(4)), *(arr(strides["small"]) for _ in range(6)))


@pytest.mark.parametrize("sizes,over,code,needle", [
    (dict(C=60), {}, 2, "channels"),
    (dict(C=8200), {}, 2, "channels"),
    (dict(dtype=9), {}, 2, "dtype"),
    (dict(wdtype=1), {}, 2, "small operands"),
    (dict(norm=2), {}, 1, "norm"),
    (dict(F=3), {}, 1, "groups"),
    (dict(F=0), {}, 1, "groups"),
    (dict(S=-1), {}, 1, "sizes"),
    (dict(B=1 << 13, S=1 << 13), {}, 2, "too many"),
    (dict(x=(256, 60, 1)), {}, 1, "multiples of 8"),
    (dict(x=(256, 64, 2)), {}, 1, "channels must be 1"),
    (dict(x=(-256, 64, 1)), {}, 1, "non-negative"),
    (dict(small=(128, 4, 1)), {}, 1, "multiples of 8"),
    ({}, dict(x=0), 1, "null"),
    ({}, dict(x=264), 1, "aligned"),
    ({}, dict(gate=258), 1, "aligned"),
    ({}, dict(weight=2), 1, "aligned"),
    ({}, dict(xo=0), 1, "x'"),
    ({}, dict(no=0), 1, "null"),
    ({}, dict(y=0, xo=0), 1, "without y"),
    ({}, dict(tx=256), 1, "tangents"),
    ({}, dict(tgate=256), 1, "a tangent without"),
    ({}, dict(eps=-1.0), 1, "eps"),
    ({}, dict(rs=math.nan), 1, "residual_scale"),
])
def test_c_entry_rejects_bad_arguments(sizes, over, code, needle):
    from dmad_amd import _native as nat

    a = dict(x=256, tx=0, y=256, ty=0, gate=256, tgate=0, scale=256, tscale=0, shift=256, tshift=0, weight=0, bias=0, post=0,
             eps=1e-6, rs=1.0, xo=256, txo=0, no=256, tno=0)
    a.update(over)
    z = _sizes(**sizes)
    rc = nat.lib().dmad_gated_norm(ctypes.byref(z), *(v if isinstance(v, float) else ctypes.c_void_p(v) for v in a.values()),
                                   ctypes.c_void_p(0))
    assert rc == code, nat.lib().dmad_last_error()
    assert needle in nat.lib().dmad_last_error().decode()


def test_c_backward_rejects_bad_arguments():
    from dmad_amd import _native as nat

    p, n, lib, z = ctypes.c_void_p, ctypes.c_size_t(0), nat.lib(), _sizes()
    assert lib.dmad_gated_norm_bwd_workspace_bytes(ctypes.byref(z), ctypes.byref(n)) == 0 and n.value > 0
    assert lib.dmad_gated_norm_bwd_workspace_bytes(None, ctypes.byref(n)) == 1

    def call(size=1 << 30, z=z, **over):
        a = dict(x=256, y=256, gx=256, gn=256, gate=256, scale=256, weight=256, bias=0, post=0, eps=1e-6, rs=1.0, dx=256, dy=256,
                 dgate=256, dscale=256, dshift=256, dweight=256, dbias=0, dpost=0, ws=256)
        a.update(over)
        return lib.dmad_gated_norm_bwd(ctypes.byref(z), *(v if isinstance(v, float) else p(v) for v in a.values()), size, p(0))

    assert call(gx=0, gn=0) == 1 and b"gradients" in lib.dmad_last_error()
    assert call(dx=0) == 1 and call(x=0) == 1
    assert call(gate=0) == 1 and b"not there" in lib.dmad_last_error()
    assert call(weight=0) == 1 and call(scale=0) == 1 and call(dbias=256) == 1 and call(dpost=256) == 1
    assert call(y=0, gate=0, dgate=0) == 1 and b"without y" in lib.dmad_last_error()
    assert call(ws=0) == 3 and call(size=16) == 3 and call(ws=264) == 3
    assert call(z=_sizes(B=0)) == 1 and b"no rows" in lib.dmad_last_error()


def test_workspace_goes_by_the_gradients_that_are_wanted():
    """3 rows of sums per workgroup where gradients run over all groups or several workgroups share one; else none."""
    from dmad_amd import _native as nat

    def size(per_channel, **over):
        z, n = _sizes(**over), ctypes.c_size_t(99)
        assert nat.lib().dmad_gated_norm_bwd_workspace_bytes_for(ctypes.byref(z), per_channel, ctypes.byref(n)) == 0
        most = ctypes.c_size_t(99)
        assert nat.lib().dmad_gated_norm_bwd_workspace_bytes(ctypes.byref(z), ctypes.byref(most)) == 0
        assert n.value <= most.value and (not per_channel or n.value == most.value)
        return n.value

    for C in (256, 5120):
        assert size(0, S=32760, F=32760, C=C) == 0
        assert size(1, S=32760, F=32760, C=C) == 32760 * 3 * C * 4
        assert size(0, S=32760, F=1, C=C) == size(1, S=32760, F=1, C=C) > 0
        assert size(0, S=0, F=1, C=C) == size(1, S=0, F=1, C=C) == 0
    z, n = _sizes(), ctypes.c_size_t(0)
    assert nat.lib().dmad_gated_norm_bwd_workspace_bytes_for(None, 0, ctypes.byref(n)) == 1
    assert nat.lib().dmad_gated_norm_bwd_workspace_bytes_for(ctypes.byref(z), 0, None) == 1


# ---------------------------------------------------------------- what watches operators, and tensors that are not their memory


def _mock_kernels(monkeypatch):
    """Stand-ins in plain torch for the launches, which read the memory of their operands: dense CPU tensors with
    data of their own only."""
    from dmad_amd import block_ops

    def values(*ts):
        for t in ts:
            assert t is None or (t.data_ptr() and not t.is_neg()), "a tensor whose memory does not hold its values"

    def forward(call, x, tx, y, ty, tgate, tscale, tshift):
        small = [getattr(call, n) for n in (*SMALL, *PER_CHANNEL)]
        values(x, tx, y, ty, tgate, tscale, tshift, *small)
        d = lambda t: None if t is None else t.detach().double()  # noqa: E731
        kind = ("layer", "rms")[call.plan.norm]
        xo, n = ob.gated_norm(d(x), d(y), *map(d, small), call.eps, kind, call.residual_scale)
        txo = tn = None
        if tx is not None:  # by hand: forward mode may be on around this
            S, z = call.plan.S, torch.zeros((), dtype=torch.float64)
            g, s, h = (z if t is None else ob.rows_of(d(t), S) for t in (tgate, tscale, tshift))
            gate = 1.0 if call.gate is None else ob.rows_of(d(call.gate), S)
            txo = d(tx)
            if y is not None:
                yy, ry, tyy = d(y), 1.0, d(ty)
                if call.post_weight is not None:
                    ry = (yy.pow(2).mean(-1, keepdim=True) + call.eps).rsqrt()
                    yy = yy * ry
                    tyy = ry * (tyy - yy * (yy * tyy).mean(-1, keepdim=True)) * d(call.post_weight)
                    yy = yy * d(call.post_weight)
                txo = txo + call.residual_scale * (g * yy + gate * tyy)
            c = xo - xo.mean(-1, keepdim=True) if kind == "layer" else xo
            r = (c.pow(2).mean(-1, keepdim=True) + call.eps).rsqrt()
            N = c * r
            t = txo - N * (N * txo).mean(-1, keepdim=True)
            t = (t - t.mean(-1, keepdim=True) if kind == "layer" else t) * r
            w = 1.0 if call.weight is None else d(call.weight)
            b = 0.0 if call.bias is None else d(call.bias)
            sc = 0.0 if call.scale is None else ob.rows_of(d(call.scale), S)
            tn = t * w * (1 + sc) + (N * w + b) * s + h
        as_x = lambda t: None if t is None else t.to(x.dtype)  # noqa: E731
        return None if y is None else as_x(xo), None if ty is None else as_x(txo), as_x(n), as_x(tn), x, y

    def gradients(call, x, y, gx, gn, originals, need):
        """By hand: a registered op runs below autograd."""
        values(x, y, gx, gn, *originals)
        kind, S, rs = ("layer", "rms")[call.plan.norm], call.plan.S, call.residual_scale
        d = lambda t: None if t is None else t.detach().double()  # noqa: E731
        mean = lambda t: t.mean(-1, keepdim=True)  # noqa: E731
        one, zero = torch.ones(()).double(), torch.zeros(()).double()
        gate, scale, shift, weight, bias, post = map(d, originals)
        z, _ = ob.gated_norm(d(x), d(y), gate, scale, shift, weight, bias, post, call.eps, kind, rs)
        c = z - mean(z) if kind == "layer" else z
        r = (mean(c.pow(2)) + call.eps).rsqrt()
        N, gn = c * r, torch.zeros_like(z) if gn is None else d(gn)
        by = one if scale is None else 1 + ob.rows_of(scale, S)
        w, b = one if weight is None else weight, zero if bias is None else bias
        a = gn * w * by
        a = a - N * mean(a * N)
        dx = r * (a - mean(a) if kind == "layer" else a) + (zero if gx is None else d(gx))
        per = lambda t: t.view(call.plan.B, call.plan.F, -1, call.plan.C).sum(2)  # noqa: E731
        out = [dx, None, None, per(gn * (N * w + b)), per(gn), (gn * by * N).sum((0, 1)), (gn * by * one).sum((0, 1)), None]
        if y is not None:
            g, yy, ry = one if gate is None else ob.rows_of(gate, S), d(y), one
            if post is not None:
                ry = (mean(yy.pow(2)) + call.eps).rsqrt()
                yy = yy * ry
            dy = rs * g * dx
            out[2] = per(rs * dx * (yy if post is None else yy * post))
            out[7] = (dy * yy).sum((0, 1))
            if post is not None:
                dy = dy * post
                dy = ry * (dy - yy * mean(dy * yy))
            out[1] = dy
        return tuple(None if o is None or not (need[i] or i == 0) else out[i].to(o.dtype)
                     for i, o in enumerate((x, y, *originals)))

    monkeypatch.setattr(block_ops, "_check_same_device", lambda op, *ts: None)
    monkeypatch.setattr(block_ops, "_norm_forward", forward)
    monkeypatch.setattr(block_ops, "_norm_gradients", gradients)


BOTH = pytest.mark.parametrize("device", ["cpu", pytest.param("gpu", marks=pytest.mark.gpu)])
EVERY = ("x", "tx", "y", "ty", "gate", "tgate", "scale", "tscale", "shift", "tshift", "weight", "bias", "post_weight")


def _set_up(request, monkeypatch, device, **how):
    if device == "cpu":
        _mock_kernels(monkeypatch)
    return _small(request.getfixturevalue("gpu") if device == "gpu" else device, **how)


def _run(x):
    (xo, txo), (n, tn) = _call(x)
    return xo, txo, n, tn


@BOTH
@pytest.mark.parametrize("name", EVERY)
def test_forward_mode_is_refused(request, monkeypatch, device, name):
    x = _set_up(request, monkeypatch, device)
    with torch.no_grad(), torch.autograd.forward_ad.dual_level():
        _run(x)  # none of them
        dual = torch.autograd.forward_ad.make_dual(x[name], torch.ones_like(x[name]))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            _run({**x, name: dual})
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(lambda t: _run({**x, name: t})[2], (x[name],), (torch.ones_like(x[name]),))


@BOTH
@pytest.mark.parametrize("name", EVERY)
def test_negated_views_have_their_sign(request, monkeypatch, device, name):
    x = _set_up(request, monkeypatch, device)
    want = _run({**x, name: -x[name]})
    odd = torch._neg_view(x[name])
    assert odd.is_neg()
    for a, b in zip(_run({**x, name: odd}), want):
        assert torch.equal(a, b)
    x = {**x, **{n: x[n].clone().requires_grad_(True) for n in ("x", "gate")}}
    n = _run(x)[2]
    g = torch.ones_like(n)
    assert torch.equal(torch.autograd.grad(n, x["gate"], torch._neg_view(g), retain_graph=True)[0],
                       torch.autograd.grad(n, x["gate"], -g)[0])


def test_meta_tensors_give_shapes():
    x = _small("meta", grad=True)
    outs = _run(x)
    assert all(o.is_meta and o.shape == (2, 6, 32) for o in outs)
    assert outs[0].requires_grad and not outs[1].requires_grad and not outs[3].requires_grad
    leaves = [x[n] for n in ALL]
    for t, g in zip(leaves, torch.autograd.grad(outs[0].sum() + outs[2].sum(), leaves)):
        assert g.is_meta and g.shape == t.shape


def test_batched_cotangents(monkeypatch):
    _mock_kernels(monkeypatch)
    x = _small(grad=True)
    xo, _, n, _ = _run(x)
    leaves = [x[m] for m in ALL]
    cts = [torch.randn(3, *o.shape) for o in (xo, n)]
    got = torch.autograd.grad((xo, n), leaves, cts, is_grads_batched=True, retain_graph=True)
    for i in range(3):
        for a, b in zip(got, torch.autograd.grad((xo, n), leaves, [c[i] for c in cts], retain_graph=True)):
            torch.testing.assert_close(a[i], b)


def test_fake_trace_has_one_node_per_pass():
    from torch.fx.experimental.proxy_tensor import make_fx

    def step(*ts):
        x = dict(zip(EVERY, ts))
        outs = _run(x)
        return torch.autograd.grad(outs[0].square().sum() + outs[2].sum(), [x[n] for n in ALL])

    x = _small("meta", grad=True)
    gm = make_fx(step, tracing_mode="fake")(*(x[n] for n in EVERY))
    ops = [n.target for n in gm.graph.nodes if n.op == "call_function" and "dmad" in str(n.target)]
    assert ops == [torch.ops.dmad.gated_norm_fwd.default, torch.ops.dmad.gated_norm_bwd.default]


@BOTH
@pytest.mark.parametrize("how", ["dispatch mode", "profiled", "compiled"])
@pytest.mark.parametrize("absent", [(), ("y", "ty", "gate", "tgate", "post_weight"), ("tscale", "shift", "tshift", "weight"),
                                    tuple(n for n in EVERY if n.startswith("t"))])
def test_op_and_direct_calls_agree_bitwise(request, monkeypatch, device, how, absent):
    from torch.utils._python_dispatch import TorchDispatchMode

    x = _set_up(request, monkeypatch, device, grad=True)
    x.update({n: None for n in absent})
    names = [n for n in ALL if x[n] is not None]
    seen = []

    class Names(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(str(func))
            return func(*args, **(kwargs or {}))

    def step(*ls):
        outs = _run({**x, **dict(zip(names, ls))})
        outs = [o for o in (outs if x["y"] is not None else outs[2:]) if o is not None]
        loss = sum(o.float().square().sum() for o in outs if o.requires_grad)
        return outs + list(torch.autograd.grad(loss, ls))

    args = [x[n] for n in names]
    want = step(*args)
    if how == "compiled":
        def forward(*ls):
            outs = _run({**x, **dict(zip(names, ls))})
            return [o for o in (outs if x["y"] is not None else outs[2:]) if o is not None]

        outs = torch.compile(forward, fullgraph=True, backend="aot_eager")(*args)
        got = list(outs) + list(torch.autograd.grad(sum(o.float().square().sum() for o in outs if o.requires_grad), args))
    elif how == "profiled":
        with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CPU]) as p:
            got = step(*args)
        assert {"dmad::gated_norm_fwd", "dmad::gated_norm_bwd"} <= {e.key for e in p.key_averages()}
    else:
        with Names():
            got = step(*args)
        assert [n for n in seen if "dmad" in n] == ["dmad.gated_norm_fwd.default", "dmad.gated_norm_bwd.default"]
    assert len(got) == len(want)
    for a, b in zip(got, want):
        assert a.requires_grad == b.requires_grad and torch.equal(a, b)


@pytest.mark.gpu
def test_registered_ops_do_what_they_declare(gpu):
    x = _small(gpu, grad=True)
    fwd, bwd = torch.ops.dmad.gated_norm_fwd.default, torch.ops.dmad.gated_norm_bwd.default
    torch.library.opcheck(fwd, (*(x[n] for n in EVERY), 1e-6, True, 0.5))
    torch.library.opcheck(fwd, (x["x"], *[None] * 9, x["weight"], None, None, 1e-6, False, 1.0))
    y = {n: t.detach() for n, t in x.items()}
    torch.library.opcheck(bwd, (y["x"], y["y"], y["gx"], y["gn"], y["gate"], y["scale"], y["shift"], y["weight"], y["bias"],
                                y["post_weight"], 1e-6, True, 0.5, [True] * 5 + [False] * 3))


HOOKS = {"type": lambda t: t.to(torch.bfloat16), "shape": lambda t: t[:, :3], "place": lambda t: t.to("meta")}


@pytest.mark.parametrize("kind", [*HOOKS, "a copy"])
def test_saved_operands_are_checked(kind):
    from dmad_amd.block_ops import _check_norm_saved

    x, g = torch.zeros(2, 5, 16), torch.zeros(2, 5, 16)
    if kind == "a copy":
        _check_norm_saved(x.clone(), g)
        return
    with pytest.raises(RuntimeError, match="as the forward read it"):
        _check_norm_saved(HOOKS[kind](x), g)
    with pytest.raises(RuntimeError, match="nothing"):
        _check_norm_saved(None, g)


@pytest.mark.gpu
def test_saved_tensor_hooks(gpu):
    x = _small(gpu, grad=True)
    leaves = [x[n] for n in ALL]

    def grads(pack, unpack):
        with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
            xo, _, n, _ = _run(x)
        return torch.autograd.grad(xo.square().sum() + n.sum(), leaves)

    want = grads(lambda t: t, lambda t: t)
    for a, b in zip(grads(lambda t: t.cpu(), lambda t: t.to(gpu)), want):
        assert torch.equal(a, b)
    for unpack in (lambda t: t.to(torch.bfloat16), lambda t: t[:1], lambda t: t.cpu()):
        with pytest.raises(RuntimeError):
            grads(lambda t: t, lambda t: unpack(t) if t.dim() == 3 and t.shape[1] == 6 else t)


@BOTH
@pytest.mark.parametrize("when", ["packed", "after the backward"])
def test_operands_are_kept_by_their_saved_tensors_alone(request, monkeypatch, device, when):
    """Hooks that move what is saved move all of it, and a graph that lives on after its backward holds no operand."""
    leaves = _set_up(request, monkeypatch, device, grad=True)
    x = {n: t if n.startswith("g") and n != "gate" else t * 1 for n, t in leaves.items()}
    there = {n: weakref.ref(t) for n, t in x.items() if n in ALL}
    clone = (lambda t: t.clone(), lambda t: t)
    with torch.autograd.graph.saved_tensors_hooks(*clone) if when == "packed" else contextlib.nullcontext():
        outs = _run(x)
    if when != "packed":
        torch.autograd.grad(outs[2].sum(), [leaves[n] for n in ALL], allow_unused=True)
    del x
    assert [n for n, r in there.items() if r() is not None] == []
    assert outs[2].requires_grad


@pytest.mark.gpu
@pytest.mark.parametrize("wdtype", ["bf16", "fp32", "mixed"])
def test_hooks_that_offload_leave_nothing_on_the_device(gpu, wdtype):
    """Nor do copies of small operands of several types stay, and what comes back may lie otherwise than it did."""
    x = _inputs(2, 6, 1536, 2, torch.bfloat16, torch.float32 if wdtype != "bf16" else torch.bfloat16, ALL, 31)
    if wdtype == "mixed":
        x["gate"], x["weight"] = x["gate"].to(torch.bfloat16), x["weight"].to(torch.bfloat16)
    d = {n: t.to(gpu).requires_grad_(n in ALL) for n, t in x.items()}
    into = (d["gx"], d["gn"])

    def current():
        torch.cuda.synchronize()
        return torch.cuda.memory_stats()["requested_bytes.all.current"]

    def run(*hooks):
        before = current()
        with torch.autograd.graph.saved_tensors_hooks(*hooks):
            (xo, _), (n, _) = _call({m: d[m] * 1 for m in ALL}, tangents=False)
        kept = current() - before - 2 * n.numel() * n.element_size()
        return kept, torch.autograd.grad((xo, n), [d[m] for m in ALL], into)

    kept, want = run(lambda t: t, lambda t: t)
    assert kept >= sum(d[m].numel() * d[m].element_size() for m in ALL)
    wide = lambda t: torch.stack((t, t), -2)[..., 0, :]  # noqa: E731
    for back in (lambda t: t.to(gpu), lambda t: wide(t.to(gpu)), lambda t: torch.cat((t.new_zeros(1), t.flatten())).to(gpu)[1:].view(t.shape)):
        kept, got = run(lambda t: t.cpu(), back)
        assert kept == 0
        for a, b in zip(got, want):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_small_operands_from_hooks_are_checked(gpu):
    x = _small(gpu, grad=True)
    for name in (*SMALL, *PER_CHANNEL):
        for change in (lambda t: t.to(torch.float16), lambda t: t[..., :-8], lambda t: t.cpu(), lambda t: t[:1] if t.dim() == 3 else t[None]):
            at = x[name].data_ptr()
            with torch.autograd.graph.saved_tensors_hooks(lambda t: (t, t.data_ptr() == at), lambda p: change(p[0]) if p[1] else p[0]):
                xo, _, n, _ = _run(x)
            with pytest.raises(RuntimeError, match="as the forward read it"):
                torch.autograd.grad(xo.square().sum() + n.sum(), [x[m] for m in ALL])


@BOTH
def test_registered_ops_refuse_what_the_calls_refuse(request, monkeypatch, device):
    x = _set_up(request, monkeypatch, device)
    t = [x[n] for n in EVERY]
    fwd, bwd = torch.ops.dmad.gated_norm_fwd, torch.ops.dmad.gated_norm_bwd
    for i, bad in ((1, x["tx"][:1]), (2, x["y"][:, :3]), (4, x["gate"][:, :2]), (10, x["weight"][:16]), (3, None)):
        with pytest.raises(ValueError):
            fwd(*t[:i], bad, *t[i + 1:], 1e-6, False, 1.0)
    small = [x[n] for n in (*SMALL, *PER_CHANNEL)]
    with pytest.raises(RuntimeError, match="as the forward read it"):
        bwd(x["x"], x["y"], x["gx"][:1], x["gn"], *small, 1e-6, False, 1.0, [True] * 8)
    with pytest.raises(ValueError, match="neither"):
        bwd(x["x"], x["y"], None, None, *small, 1e-6, False, 1.0, [True] * 8)
    with pytest.raises(ValueError, match="belong to y"):
        bwd(x["x"], None, x["gx"], x["gn"], *small, 1e-6, False, 1.0, [True] * 8)


@BOTH
def test_a_change_in_place_is_noticed(request, monkeypatch, device):
    x = _set_up(request, monkeypatch, device, grad=True)
    n = _run(x)[2]
    with torch.no_grad():
        x["gate"].add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        n.sum().backward()
