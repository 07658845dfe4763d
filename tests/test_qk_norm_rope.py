"""RMSNorm of queries and keys per head with the rotation in the same pass (qk_norm_rope_with_tangent).

CPU: the oracle (oracle/streaming.py) against differences and element-wise loops. GPU: the kernels
against the oracle on the same inputs. The kernels compute in float32 and round once, so an element is
off by half a step of its type, u = finfo.eps / 2, plus float32 errors of the terms it is made of: the
mean of D squares (8 sequential and at most 5 pairwise additions), one reciprocal root, sine and cosine
and four products come to less than 64 half steps of float32 of the larger element of its pair.
"""
import math

import pytest
import torch

from oracle import streaming as st

F32 = 2.0 ** -24
FP32_STEPS = 64
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _half_step(dtype):
    return torch.finfo(dtype).eps / 2


def _pair_size(x):
    """The larger magnitude of each pair, for both of its elements."""
    a = x.abs().reshape(*x.shape[:-1], -1, 2).amax(-1, keepdim=True)
    return a.expand(*a.shape[:-1], 2).reshape(x.shape)


def _check(name, got, ref, scale):
    """|got - ref| <= u |ref| + steps of float32 of `scale` (+ half the smallest subnormal)."""
    tiny = torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps
    tol = _half_step(got.dtype) * ref.abs() * (1 + 1e-3) + FP32_STEPS * F32 * scale + tiny
    err = (got.detach().cpu().double() - ref).abs()
    assert torch.isfinite(got.detach().cpu().double()).all(), name
    worst = float((err / tol).max()) if err.numel() else 0.0
    print(f"  {name}: worst error {worst:.2f} of its bound", flush=True)
    assert worst <= 1.0, name


# ---------------------------------------------------------------- the oracle


def test_oracle_matches_loops():
    g = torch.Generator().manual_seed(0)
    x = torch.randn(2, 3, 2, 8, generator=g, dtype=torch.float64)
    w = torch.rand(8, generator=g, dtype=torch.float64)
    f = torch.rand(3, 4, generator=g, dtype=torch.float64) * 6
    y = st.norm_rope(x, w, 1e-3, f)
    for b in range(2):
        for s in range(3):
            for h in range(2):
                row = x[b, s, h].tolist()
                r = 1 / math.sqrt(sum(v * v for v in row) / 8 + 1e-3)
                z = [v * r * float(w[i]) for i, v in enumerate(row)]
                for i in range(4):
                    c, n = math.cos(float(f[s, i])), math.sin(float(f[s, i]))
                    assert abs(z[2 * i] * c - z[2 * i + 1] * n - float(y[b, s, h, 2 * i])) < 1e-12
                    assert abs(z[2 * i + 1] * c + z[2 * i] * n - float(y[b, s, h, 2 * i + 1])) < 1e-12


def test_oracle_tangent_is_the_difference_quotient():
    g = torch.Generator().manual_seed(1)
    x, t = (torch.randn(1, 2, 3, 16, generator=g, dtype=torch.float64) for _ in range(2))
    w, f = torch.rand(16, generator=g, dtype=torch.float64), torch.rand(2, 8, generator=g, dtype=torch.float64)
    d = (st.norm_rope(x + 1e-6 * t, w, 1e-6, f) - st.norm_rope(x - 1e-6 * t, w, 1e-6, f)) / 2e-6
    assert torch.allclose(st.norm_rope_tangent(x, t, w, 1e-6, f), d, rtol=1e-6, atol=1e-8)


# ---------------------------------------------------------------- inputs


def _inputs(B, S, Hq, Hk, D, dtype, wdtype, seed, layout):
    g = torch.Generator().manual_seed(seed)

    def r(*shape, sd=1.0):
        return (torch.randn(shape, generator=g) * sd).to(dtype)

    if layout == "fused":  # slices of one projection's output
        qkv = r(B, S, Hq + 2 * Hk, D)
        q, k = qkv[:, :, :Hq], qkv[:, :, Hq:Hq + Hk]
    elif layout == "bhsd":
        q, k = r(B, Hq, S, D).transpose(1, 2), r(B, Hk, S, D).transpose(1, 2)
    else:
        q, k = r(B, S, Hq, D), r(B, S, Hk, D)
    x = dict(q=q, k=k, tq=r(B, S, Hq, D, sd=0.1), tk=r(B, Hk, S, D, sd=0.1).transpose(1, 2), gq=r(B, S, Hq, D),
             gk=r(B, S, Hk, D))
    for n in ("wq", "wk"):
        x[n] = (1 + 0.3 * torch.randn(D, generator=g)).to(wdtype)
    x["freqs"] = torch.rand(S, D // 2, generator=g) * 200 - 100
    x["freqs3"] = torch.rand(B, S, D // 2, generator=g) * 200 - 100
    return x


def _to(x, dev):
    """The same tensor on the device, with its strides."""
    base = torch.empty_strided(x.shape, x.stride(), dtype=x.dtype, device=dev) if x.is_contiguous() or 0 not in x.stride() else x.to(dev)
    base.copy_(x)
    return base


def _reference(x, wq, wk, eps, freqs, jvp):
    out = {}
    for n, w in (("q", wq), ("k", wk)):
        z = x[n].double().requires_grad_(True)
        wz = None if w is None else w.double().requires_grad_(True)
        y = st.norm_rope(z, wz, eps, freqs)
        y.backward(x["g" + n].double())
        out[n], out["d" + n] = y.detach(), z.grad
        if w is not None:
            out["dw" + n] = wz.grad
            u = st.rotate(x["g" + n].double(), None if freqs is None else -freqs.double())
            m = z.detach() / (z.detach().pow(2).mean(-1, keepdim=True) + eps).sqrt()
            out["sum" + n] = (u * m).abs().sum((0, 1, 2))  # what the weight's gradient is the sum of
            a, r = u * w.double(), (z.detach().pow(2).mean(-1, keepdim=True) + eps).rsqrt()
            out["size" + n] = r * (_pair_size(a) + m.abs() * (a * m).abs().mean(-1, keepdim=True))
        else:
            out["size" + n] = _pair_size(out["d" + n])
        if jvp:
            out["t" + n] = st.norm_rope_tangent(x[n], x["t" + n], w, eps, freqs)
            z, t = x[n].double(), x["t" + n].double()
            if w is not None:
                r = (z.pow(2).mean(-1, keepdim=True) + eps).rsqrt()
                parts = (t.abs() + (z * r).abs() * (z * r * t).abs().mean(-1, keepdim=True)) * r * w.double().abs()
            else:
                parts = t
            out["tsize" + n] = _pair_size(parts)
    return out


CASES = [
    # B, S, Hq, Hk, D, dtype, weights' dtype, layout, weights, rotation
    (1, 1, 1, 1, 16, "bf16", "bf16", "plain", True, "shared"),
    (2, 37, 3, 1, 16, "fp16", "fp32", "fused", True, "batch"),
    (1, 65, 40, 8, 32, "bf16", "fp32", "bhsd", True, "shared"),
    (3, 21, 5, 5, 64, "fp16", "fp16", "fused", True, "shared"),
    (1, 256, 2, 2, 64, "fp32", "fp32", "plain", True, "shared"),
    (2, 130, 12, 12, 128, "bf16", "bf16", "plain", True, "shared"),
    (1, 77, 9, 3, 128, "fp32", "fp32", "fused", True, "batch"),
    (1, 999, 40, 40, 128, "bf16", "bf16", "fused", True, "shared"),
    (2, 33, 7, 1, 256, "bf16", "fp32", "bhsd", True, "batch"),
    (1, 50, 4, 2, 256, "fp32", "fp32", "plain", True, "shared"),
    (2, 40, 6, 2, 128, "bf16", "bf16", "plain", False, "shared"),
    (2, 40, 6, 2, 64, "fp16", "fp16", "plain", True, None),
]


@pytest.mark.gpu
@pytest.mark.parametrize("B,S,Hq,Hk,D,dtype,wdtype,layout,norm,rope", CASES)
def test_forward_tangent_backward(gpu, B, S, Hq, Hk, D, dtype, wdtype, layout, norm, rope):
    from dmad_amd import qk_norm_rope_with_tangent

    print(f"case norm B={B} S={S} Hq={Hq} Hk={Hk} D={D} {dtype} weights {wdtype if norm else None} {layout} rope={rope}", flush=True)
    x = _inputs(B, S, Hq, Hk, D, DTYPES[dtype], DTYPES[wdtype], seed=D + S, layout=layout)
    wq, wk = (x["wq"], x["wk"]) if norm else (None, None)
    freqs = {"shared": x["freqs"], "batch": x["freqs3"], None: None}[rope]
    ref = _reference(x, wq, wk, 1e-6, freqs, True)
    d = {n: _to(v, gpu) for n, v in x.items()}
    leaves = [d["q"].requires_grad_(True), d["k"].requires_grad_(True)]
    if norm:
        leaves += [d["wq"].requires_grad_(True), d["wk"].requires_grad_(True)]
    f = None if freqs is None else freqs.to(gpu)
    args = ((d["wq"], d["wk"]) if norm else (None, None)) + (1e-6, f)
    (q, tq), (k, tk) = qk_norm_rope_with_tangent((d["q"], d["tq"]), (d["k"], d["tk"]), *args)
    assert q.requires_grad and k.requires_grad and not tq.requires_grad and not tk.requires_grad
    assert q.is_contiguous() and q.shape == (B, S, Hq, D) and k.shape == (B, S, Hk, D)
    grads = torch.autograd.grad((q, k), leaves, (d["gq"], d["gk"]))
    torch.cuda.synchronize()
    for n, y, ty in (("q", q, tq), ("k", k, tk)):
        _check(n, y, ref[n], _pair_size(ref[n]))
        _check("t" + n, ty, ref["t" + n], ref["tsize" + n])
    for n, got in zip(("q", "k"), grads):
        _check("d" + n, got, ref["d" + n], ref["size" + n])
    if norm:
        for n, got in zip(("q", "k"), grads[2:]):
            assert got.dtype == DTYPES[wdtype]
            _check("dw" + n, got, ref["dw" + n], ref["sum" + n])
    # the primal alone is the same
    with torch.no_grad():
        (q2, t2), (k2, _) = qk_norm_rope_with_tangent((d["q"], None), (d["k"], None), *args)
    assert t2 is None and torch.equal(q2, q) and torch.equal(k2, k)


@pytest.mark.gpu
def test_gradient_is_the_difference_quotient(gpu):
    """fp32 gradients against central differences of the kernel's own outputs. With step h = 2^-6 the
    quotient of sum(y g) is off by h^2 / 6 times a third derivative of order 10 and by the outputs' float32
    errors, 64 half steps of sum |y g| over h: together under 1e-3 of the gradient's size here."""
    from dmad_amd import qk_norm_rope_with_tangent

    g = torch.Generator().manual_seed(5)
    x = torch.randn(1, 3, 2, 16, generator=g).to(gpu).requires_grad_(True)
    w = (1 + 0.2 * torch.randn(16, generator=g)).to(gpu).requires_grad_(True)
    f, go, dx, dw = torch.rand(3, 8, generator=g).to(gpu), *(torch.randn(s, generator=g).to(gpu) for s in ((1, 3, 2, 16), (1, 3, 2, 16), (16,)))

    def loss(a, b):
        return (qk_norm_rope_with_tangent((a, None), (None, None), b, None, 1e-6, f)[0][0].double() * go.double()).sum()

    gx, gw = torch.autograd.grad(loss(x, w), (x, w))
    h = 2.0 ** -6
    with torch.no_grad():
        num_x = (loss(x + h * dx, w) - loss(x - h * dx, w)) / (2 * h)
        num_w = (loss(x, w + h * dw) - loss(x, w - h * dw)) / (2 * h)
    size_x, size_w = float((gx * dx).abs().sum()), float((gw * dw).abs().sum())
    assert abs(float((gx.double() * dx).sum() - num_x)) <= 1e-3 * size_x
    assert abs(float((gw.double() * dw).sum() - num_w)) <= 1e-3 * size_w


@pytest.mark.gpu
def test_one_operand_and_partial_gradients(gpu):
    from dmad_amd import qk_norm_rope_with_tangent

    x = _inputs(2, 19, 4, 2, 64, torch.bfloat16, torch.bfloat16, 7, "plain")
    d = {n: v.to(gpu) for n, v in x.items()}
    both = qk_norm_rope_with_tangent((d["q"], d["tq"]), (d["k"], d["tk"]), d["wq"], d["wk"], 1e-6, d["freqs"])
    (q, tq), none = qk_norm_rope_with_tangent((d["q"], d["tq"]), (None, None), d["wq"], None, 1e-6, d["freqs"])
    assert none == (None, None) and torch.equal(q, both[0][0]) and torch.equal(tq, both[0][1])
    none, (k, _) = qk_norm_rope_with_tangent((None, None), (d["k"], None), None, d["wk"], 1e-6, d["freqs"])
    assert none == (None, None) and torch.equal(k, both[1][0])
    # a loss of k alone leaves q and its weight without a gradient
    for n in ("q", "k", "wq", "wk"):
        d[n].requires_grad_(True)
    (_, _), (k, _) = qk_norm_rope_with_tangent((d["q"], None), (d["k"], None), d["wq"], d["wk"], 1e-6, d["freqs"])
    k.float().square().sum().backward()
    assert d["q"].grad is None and d["wq"].grad is None and d["k"].grad is not None and d["wk"].grad is not None
    # a summed output's gradient is an expanded scalar; a frozen weight gets none
    d["wk"].requires_grad_(False)
    (q, _), (k, _) = qk_norm_rope_with_tangent((d["q"], None), (d["k"], None), d["wq"], d["wk"], 1e-6, d["freqs"])
    gq, gw = torch.autograd.grad(q.sum() + k.sum(), (d["q"], d["wq"]))
    ones = torch.ones_like(q)
    (q, _), (k, _) = qk_norm_rope_with_tangent((d["q"], None), (d["k"], None), d["wq"], d["wk"], 1e-6, d["freqs"])
    hq, hw = torch.autograd.grad((q,), (d["q"], d["wq"]), (ones,))
    assert torch.equal(gq, hq) and torch.equal(gw, hw)


@pytest.mark.gpu
def test_no_second_derivative(gpu):
    """A gradient taken with create_graph is right, and differentiating it raises instead of giving zero."""
    from dmad_amd import qk_norm_rope_with_tangent

    x = torch.randn(1, 4, 2, 32, device=gpu, requires_grad=True)
    w, f = torch.ones(32, device=gpu), torch.rand(4, 16, device=gpu)

    def grad(create_graph):
        (y, _), _ = qk_norm_rope_with_tangent((x, None), (None, None), w, None, 1e-6, f)
        return torch.autograd.grad(y.square().sum() + y.sum(), x, create_graph=create_graph)[0]

    g = grad(True)
    assert torch.equal(g.detach(), grad(False))
    with pytest.raises(RuntimeError, match="differentiate twice"):
        g.sum().backward()


@pytest.mark.gpu
def test_broadcast_and_unaligned_inputs(gpu):
    """An expanded operand is read in place and its gradient summed; rows that start unaligned are copied."""
    from dmad_amd import qk_norm_rope_with_tangent

    g = torch.Generator().manual_seed(9)
    one = torch.randn(1, 11, 1, 128, generator=g).to(torch.bfloat16).to(gpu).requires_grad_(True)
    w, f = torch.ones(128, device=gpu, dtype=torch.bfloat16), torch.rand(11, 64, generator=g).to(gpu)
    (q, _), _ = qk_norm_rope_with_tangent((one.expand(2, 11, 3, 128), None), (None, None), w, None, 1e-6, f)
    (r, _), _ = qk_norm_rope_with_tangent((one, None), (None, None), w, None, 1e-6, f)
    assert torch.equal(q, r.expand_as(q))
    q.float().sum().backward()
    assert one.grad.shape == one.shape
    flat = torch.randn(1 * 5 * 2 * 64 + 1, generator=g).to(torch.bfloat16).to(gpu)
    odd = flat[1:].view(1, 5, 2, 64)
    w, f = torch.ones(64, device=gpu, dtype=torch.bfloat16), torch.rand(5, 32, generator=g).to(gpu)
    a = qk_norm_rope_with_tangent((odd, None), (None, None), w, None, 1e-6, f)[0][0]
    b = qk_norm_rope_with_tangent((odd.clone(), None), (None, None), w, None, 1e-6, f)[0][0]
    assert torch.equal(a, b)


@pytest.mark.gpu
def test_extremes(gpu):
    """Zero rows, with eps = 0 too (0/0 is NaN in that row alone), large and small values, an empty batch."""
    from dmad_amd import qk_norm_rope_with_tangent

    w, f = torch.ones(32, device=gpu), torch.rand(4, 16, device=gpu)
    x = torch.zeros(1, 4, 3, 32, device=gpu)
    x[0, 1] = 1e18
    x[0, 2] = 1e-18
    x.requires_grad_(True)
    (y, _), _ = qk_norm_rope_with_tangent((x, None), (None, None), w, None, 1e-30, f)
    ref = st.norm_rope(x.detach().cpu(), w.cpu(), 1e-30, f.cpu())
    _check("y", y, ref, _pair_size(ref))
    (y, _), _ = qk_norm_rope_with_tangent((x, None), (None, None), w, None, 0.0, f)
    assert torch.isnan(y[0, 0]).all() and torch.isfinite(y[0, 1]).all()
    # three heads of 32 leave most of a wave without a row: those add nothing to the weight's gradient
    z = torch.randn(1, 4, 3, 32, device=gpu)
    wz = w.clone().requires_grad_(True)
    (y, _), _ = qk_norm_rope_with_tangent((z, None), (None, None), wz, None, 0.0, f)
    assert torch.isfinite(torch.autograd.grad(y.sum(), wz)[0]).all()
    e = torch.zeros(0, 4, 3, 32, device=gpu, requires_grad=True)
    we = w.clone().requires_grad_(True)
    (y, _), _ = qk_norm_rope_with_tangent((e, None), (None, None), we, None, 1e-6, f)
    ge, gw = torch.autograd.grad(y.sum(), (e, we))
    assert y.shape == e.shape and ge.shape == e.shape and torch.equal(gw, torch.zeros_like(gw))


@pytest.mark.gpu
def test_long_sums_of_the_weight_gradient_repeat(gpu):
    from dmad_amd import qk_norm_rope_with_tangent

    x = _inputs(1, 7000, 12, 4, 128, torch.bfloat16, torch.float32, 11, "plain")
    ref = _reference(x, x["wq"], x["wk"], 1e-6, x["freqs"], False)
    d = {n: v.to(gpu) for n, v in x.items()}
    for n in ("q", "k", "wq", "wk"):
        d[n].requires_grad_(True)
    runs = []
    for _ in range(3):
        (q, _), (k, _) = qk_norm_rope_with_tangent((d["q"], None), (d["k"], None), d["wq"], d["wk"], 1e-6, d["freqs"])
        runs.append(torch.autograd.grad((q, k), (d["wq"], d["wk"]), (d["gq"], d["gk"])))
    _check("dwq", runs[0][0], ref["dwq"], ref["sumq"])
    _check("dwk", runs[0][1], ref["dwk"], ref["sumk"])
    for r in runs[1:]:
        assert torch.equal(r[0], runs[0][0]) and torch.equal(r[1], runs[0][1])


@pytest.mark.gpu
def test_feeds_the_jvp_attention(gpu):
    """The operator in its place: projections' outputs and tangents, normed and rotated, into the JVP attention."""
    from dmad_amd import qk_norm_rope_with_tangent, torch_attention_op_withT
    from oracle import attention as orc

    x = _inputs(1, 200, 4, 4, 64, torch.bfloat16, torch.bfloat16, 13, "fused")
    g = torch.Generator().manual_seed(14)
    v = torch.randn(1, 200, 4, 64, generator=g).to(torch.bfloat16)
    tv = (torch.randn(1, 200, 4, 64, generator=g) * 0.1).to(torch.bfloat16)
    d = {n: t.to(gpu) for n, t in x.items()}
    d["q"].requires_grad_(True)
    qT, kT = qk_norm_rope_with_tangent((d["q"], d["tq"]), (d["k"], d["tk"]), d["wq"], d["wk"], 1e-6, d["freqs"])
    o, to = torch_attention_op_withT(qT, kT, (v.to(gpu), tv.to(gpu)))
    o.float().sum().backward()
    hd = lambda t: t.transpose(1, 2).double()  # noqa: E731
    q, k = (st.norm_rope(x[n], x["w" + n], 1e-6, x["freqs"]).to(torch.bfloat16) for n in ("q", "k"))
    tq, tk = (st.norm_rope_tangent(x[n], x["t" + n], x["w" + n], 1e-6, x["freqs"]).to(torch.bfloat16) for n in ("q", "k"))
    ro, rto, _, _ = orc.jvp_closed_form(hd(q), hd(k), hd(v), hd(tq), hd(tk), hd(tv))
    assert orc.rel_l2(o.detach().transpose(1, 2).cpu(), ro) < 1e-2
    assert orc.rel_l2(to.transpose(1, 2).cpu(), rto) < 1e-2
    assert torch.isfinite(d["q"].grad.float()).all() and float(d["q"].grad.float().norm()) > 0


@pytest.mark.gpu
def test_captured_and_on_another_stream(gpu):
    from dmad_amd import qk_norm_rope_with_tangent

    x = _inputs(2, 300, 6, 2, 128, torch.bfloat16, torch.bfloat16, 15, "plain")
    d = {n: v.to(gpu) for n, v in x.items()}

    def step():
        leaves = [d[n].detach().requires_grad_(True) for n in ("q", "k", "wq", "wk")]
        (q, _), (k, _) = qk_norm_rope_with_tangent((leaves[0], None), (leaves[1], None), leaves[2], leaves[3], 1e-6, d["freqs"])
        return [q.detach(), k.detach(), *torch.autograd.grad((q, k), leaves, (d["gq"], d["gk"]))]

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
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(3):
        junk = torch.randn(1024, 1024, device=gpu)
        (junk @ junk).sum().item()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, ref))


# ---------------------------------------------------------------- refusals


def test_refusals_on_the_cpu():
    from dmad_amd import qk_norm_rope_with_tangent

    q = torch.randn(1, 2, 3, 32)
    with pytest.raises(RuntimeError, match="GPU only"):
        qk_norm_rope_with_tangent((q, None), (None, None), None, None, 1e-6, torch.zeros(2, 16))


@pytest.mark.gpu
def test_refusals(gpu):
    from dmad_amd import qk_norm_rope_with_tangent as op

    q = torch.randn(2, 5, 4, 64, device=gpu, dtype=torch.bfloat16)
    k, w, f = q[:, :, :2].contiguous(), torch.ones(64, device=gpu, dtype=torch.bfloat16), torch.zeros(5, 32, device=gpu)
    bad = [
        (ValueError, "neither", (None, None), (None, None), w, w, 1e-6, f),
        (ValueError, "heads", (q, None), (k[:, :4], None), w, w, 1e-6, f),
        (ValueError, "and k", (q, None), (k.half(), None), w, w, 1e-6, f),
        (NotImplementedError, "head dim", (q[..., :48], None), (None, None), None, None, 1e-6, None),
        (NotImplementedError, "dtype", (q.double(), None), (None, None), None, None, 1e-6, f),
        (ValueError, "weights", (q, None), (k, None), w[:32], w, 1e-6, f),
        (ValueError, "weights", (q, None), (k, None), w.double(), w, 1e-6, f),
        (ValueError, "freqs", (q, None), (k, None), w, w, 1e-6, f[:4]),
        (ValueError, "freqs", (q, None), (k, None), w, w, 1e-6, f[None].expand(3, 5, 32)),
        (ValueError, "eps", (q, None), (k, None), w, w, -1.0, f),
        (ValueError, "eps", (q, None), (k, None), w, w, math.nan, f),
        (ValueError, "tangent", (q, q[:1]), (k, k), w, w, 1e-6, f),
        (ValueError, "tangents of both", (q, q), (k, None), w, w, 1e-6, f),
        (ValueError, r"\[B, S, H, D\]", (q[0], None), (None, None), w, w, 1e-6, f),
        (RuntimeError, "GPU only", (q, None), (k.cpu(), None), w, w, 1e-6, f),
    ]
    for error, match, *args in bad:
        with pytest.raises(error, match=match):
            op(*args)
    # a weight of another 16-bit type is widened with its partner
    a = op((q, None), (k, None), w, w.float(), 1e-6, f)
    b = op((q, None), (k, None), w.float(), w.float(), 1e-6, f)
    assert torch.equal(a[0][0], b[0][0]) and torch.equal(a[1][0], b[1][0])


def _strides(*v):
    import ctypes

    return (ctypes.c_int64 * 4)(*v)


@pytest.mark.parametrize("over,code,needle", [
    (dict(D=48), 2, "head dim"),
    (dict(dtype=9), 2, "dtype"),
    (dict(wdtype=1), 2, "weights"),
    (dict(Hq=0, Hk=0), 1, "sizes"),
    (dict(S=-1), 1, "sizes"),
    (dict(eps=-1.0), 1, "eps"),
    (dict(q=0), 1, "q: null"),
    (dict(Hk=0), 1, "no heads"),
    (dict(tq=256), 1, "neither"),
    (dict(q=264), 1, "aligned"),
    (dict(wq=2), 1, "aligned"),
    (dict(qs=_strides(512, 256, 60, 1)), 1, "multiples of 8"),
    (dict(qs=_strides(512, 256, 64, 2)), 1, "head dim must be 1"),
    (dict(ks=_strides(512, -256, 64, 1)), 1, "non-negative"),
    (dict(ok=0), 1, "output"),
    (dict(fb=-1), 1, "freqs"),
    (dict(B=1 << 20, S=1 << 20), 2, "too many"),
    (dict(B=1 << 15, S=1 << 15, Hq=64), 2, "too many"),
])
def test_c_entry_rejects_bad_arguments(over, code, needle):
    import ctypes

    from dmad_amd import _native as nat

    a = dict(dtype=0, wdtype=0, B=1, S=2, Hq=4, Hk=2, D=64, q=256, tq=0, k=256, tk=0, qs=_strides(512, 256, 64, 1), wq=256,
             ks=_strides(256, 128, 64, 1), wk=256, f=256, fb=0, eps=1e-6, oq=256, ok=256)
    a.update(over)
    p = ctypes.c_void_p
    rc = nat.lib().dmad_qk_norm_rope(a["dtype"], a["wdtype"], a["B"], a["S"], a["Hq"], a["Hk"], a["D"], p(a["q"]), p(a["tq"]),
                                     p(a["k"]), p(a["tk"]), a["qs"], a["qs"], a["ks"], a["ks"], p(a["wq"]), p(a["wk"]),
                                     p(a["f"]), a["fb"], a["eps"], p(a["oq"]), p(0), p(a["ok"]), p(0), p(0))
    assert rc == code, nat.lib().dmad_last_error()
    assert needle in nat.lib().dmad_last_error().decode()


def test_c_backward_rejects_bad_arguments():
    import ctypes

    from dmad_amd import _native as nat

    p, n = ctypes.c_void_p, ctypes.c_size_t(0)
    lib = nat.lib()
    assert lib.dmad_qk_norm_rope_bwd_workspace_bytes(1, 5, 4, 2, 64, ctypes.byref(n)) == 0 and n.value > 0
    s = _strides(512, 256, 64, 1)

    def call(wq=256, dwq=256, gq=256, ws=256, size=1 << 30, B=1):
        return lib.dmad_qk_norm_rope_bwd(0, 0, B, 2, 4, 4, 64, p(256), p(gq), p(256), p(256), s, s, s, s, p(wq), p(256), p(256),
                                         0, 1e-6, p(256), p(256), p(dwq), p(256), p(ws), size, p(0))

    assert call(wq=0) == 1 and b"weight" in lib.dmad_last_error()
    assert call(gq=0) == 1 and b"gradient" in lib.dmad_last_error()
    assert call(ws=0) == 3 and call(size=16) == 3
    assert call(B=0) == 1


# ---------------------------------------------------------------- what watches operators, and tensors that are not their memory


def _mock_kernels(monkeypatch):
    """Stand-ins in plain torch for the launches, which read the memory of their operands: dense CPU tensors with
    data of their own only."""
    from dmad_amd import prologue

    def values(*ts):
        for t in ts:
            assert t is None or (t.data_ptr() and not t.is_neg()), "a tensor whose memory does not hold its values"

    def forward(call, q, tq, k, tk):
        values(q, tq, k, tk, call.wq, call.wk, call.freqs)
        outs = []
        for x, t, w in ((q, tq, call.wq), (k, tk, call.wk)):
            outs.append(None if x is None else st.norm_rope(x, w, call.eps, call.freqs).to(x.dtype))
            if t is not None and w is not None:  # without forward mode, which may be on around this
                r = (x.double().pow(2).mean(-1, keepdim=True) + call.eps).rsqrt()
                t = r * (t.double() - x * r * (x * r * t).mean(-1, keepdim=True)) * w
            outs.append(None if t is None else st.rotate(t.double(), call.freqs).to(x.dtype))
        return (*outs, q, k)

    def gradients(call, q, k, gq, gk, wq, wk, need_wq, need_wk):
        values(q, k, gq, gk, wq, wk, call.wq, call.wk, call.freqs)
        dx, dw = [], []
        for x, g, w, need in ((q, gq, wq, need_wq), (k, gk, wk, need_wk)):
            if g is None:
                dx.append(None), dw.append(None)
                continue
            a = st.rotate(g.double(), None if call.freqs is None else -call.freqs)
            if w is not None:
                r = (x.double().pow(2).mean(-1, keepdim=True) + call.eps).rsqrt()
                n, u = x * r, a
                a = u * w
                a = r * (a - n * (a * n).mean(-1, keepdim=True))
            dx.append(a.to(x.dtype))
            dw.append((u * n).sum((0, 1, 2)).to(w.dtype) if need and w is not None else None)
        return (*dx, *dw)

    monkeypatch.setattr(prologue, "_check_same_device", lambda op, *ts: None)
    monkeypatch.setattr(prologue, "_qk_forward", forward)
    monkeypatch.setattr(prologue, "_qk_gradients", gradients)


def _small(device="cpu", grad=False, dtype=torch.float32):
    g = torch.Generator().manual_seed(3)
    x = dict(q=torch.randn(2, 5, 4, 16, generator=g), k=torch.randn(2, 5, 2, 16, generator=g), tq=torch.randn(2, 5, 4, 16, generator=g),
             tk=torch.randn(2, 5, 2, 16, generator=g), wq=torch.rand(16, generator=g) + 0.5, wk=torch.rand(16, generator=g) + 0.5)
    x = {n: t.to(device, dtype) for n, t in x.items()}
    x["freqs"] = (torch.rand(5, 8, generator=g) * 6).to(device)
    for n in ("q", "k", "wq", "wk"):
        x[n].requires_grad_(grad)
    return x


def _run(x):
    from dmad_amd import qk_norm_rope_with_tangent

    (q, tq), (k, tk) = qk_norm_rope_with_tangent((x["q"], x["tq"]), (x["k"], x["tk"]), x["wq"], x["wk"], 1e-6, x["freqs"])
    return q, tq, k, tk


OPERANDS = ("q", "tq", "k", "tk", "wq", "wk", "freqs")


@pytest.mark.parametrize("device", ["cpu", pytest.param("gpu", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("name", OPERANDS)
def test_forward_mode_is_refused(request, monkeypatch, device, name):
    """torch's forward-mode tangents are not the operator's: they would be lost, so they are refused, whichever
    operand carries them, by torch.autograd.forward_ad and by torch.func.jvp."""
    if device == "cpu":
        _mock_kernels(monkeypatch)
    x = _small(request.getfixturevalue("gpu") if device == "gpu" else device)
    with torch.no_grad(), torch.autograd.forward_ad.dual_level():
        _run(x)  # none of them
        dual = torch.autograd.forward_ad.make_dual(x[name], torch.ones_like(x[name]))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            _run({**x, name: dual})
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(lambda t: _run({**x, name: t})[0], (x[name],), (torch.ones_like(x[name]),))


@pytest.mark.parametrize("device", ["cpu", pytest.param("gpu", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("name", OPERANDS)
def test_negated_views_have_their_sign(request, monkeypatch, device, name):
    if device == "cpu":
        _mock_kernels(monkeypatch)
    x = _small(request.getfixturevalue("gpu") if device == "gpu" else device)
    want = _run({**x, name: -x[name]})
    odd = torch._neg_view(x[name])
    assert odd.is_neg()
    for a, b in zip(_run({**x, name: odd}), want):
        assert torch.equal(a, b)
    # and a cotangent
    x = {**x, **{n: x[n].clone().requires_grad_(True) for n in ("q", "wk")}}
    q, _, k, _ = _run(x)
    g = torch.ones_like(q)
    assert torch.equal(torch.autograd.grad(q, x["q"], torch._neg_view(g), retain_graph=True)[0], torch.autograd.grad(q, x["q"], -g)[0])


@pytest.mark.parametrize("device", ["cpu", pytest.param("gpu", marks=pytest.mark.gpu)])
def test_angles_that_want_a_gradient_are_refused(request, monkeypatch, device):
    if device == "cpu":
        _mock_kernels(monkeypatch)
    x = _small(request.getfixturevalue("gpu") if device == "gpu" else device)
    x["freqs"].requires_grad_(True)
    with pytest.raises(RuntimeError, match="gradient of the angles"):
        _run(x)
    with torch.no_grad():
        _run(x)


def test_meta_tensors_give_shapes():
    x = _small("meta", grad=True)
    outs = _run(x)
    assert [tuple(o.shape) for o in outs] == [(2, 5, 4, 16)] * 2 + [(2, 5, 2, 16)] * 2 and all(o.is_meta for o in outs)
    assert outs[0].requires_grad and not outs[1].requires_grad
    leaves = [x[n] for n in ("q", "k", "wq", "wk")]
    for t, g in zip(leaves, torch.autograd.grad(outs[0].sum() + outs[2].sum(), leaves)):
        assert g.is_meta and g.shape == t.shape
    with pytest.raises(ValueError, match="freqs"):
        _run({**x, "freqs": x["freqs"][:4]})


def test_batched_cotangents(monkeypatch):
    _mock_kernels(monkeypatch)
    x = _small(grad=True)
    q, _, k, _ = _run(x)
    leaves = [x[n] for n in ("q", "k", "wq", "wk")]
    cts = [torch.randn(3, *o.shape) for o in (q, k)]
    got = torch.autograd.grad((q, k), leaves, cts, is_grads_batched=True, retain_graph=True)
    for i in range(3):
        for a, b in zip(got, torch.autograd.grad((q, k), leaves, [c[i] for c in cts], retain_graph=True)):
            torch.testing.assert_close(a[i], b)


def test_fake_trace_has_one_node_per_pass():
    from torch.fx.experimental.proxy_tensor import make_fx

    def step(*ts):
        x = dict(zip(OPERANDS, ts))
        outs = _run(x)
        return torch.autograd.grad(outs[0].square().sum() + outs[2].sum(), [x[n] for n in ("q", "k", "wq", "wk")])

    x = _small("meta", grad=True)
    gm = make_fx(step, tracing_mode="fake")(*(x[n] for n in OPERANDS))
    ops = [n.target for n in gm.graph.nodes if n.op == "call_function" and "dmad" in str(n.target)]
    assert ops == [torch.ops.dmad.qk_norm_rope_fwd.default, torch.ops.dmad.qk_norm_rope_bwd.default]


def _watched(x, leaves, how):
    from torch.utils._python_dispatch import TorchDispatchMode

    class Names(TorchDispatchMode):
        names = []

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            self.names.append(str(func))
            return func(*args, **(kwargs or {}))

    def step(*ls):
        y = {**x, **dict(zip(leaves, ls))}
        outs = _run(y)
        loss = sum(o.float().square().sum() for o in (outs[0], outs[2]) if o is not None)
        return [o for o in outs if o is not None] + list(torch.autograd.grad(loss, ls))

    args = [x[n] for n in leaves]
    if how == "direct":
        return step(*args)
    if how == "compiled":
        def forward(*ls):
            return [o for o in _run({**x, **dict(zip(leaves, ls))}) if o is not None]

        outs = torch.compile(forward, fullgraph=True, backend="aot_eager")(*args)
        primal = [o for o in outs if o.requires_grad]
        return list(outs) + list(torch.autograd.grad(sum(o.float().square().sum() for o in primal), args))
    if how == "profiled":
        with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CPU]) as p:
            out = step(*args)
        assert {"dmad::qk_norm_rope_fwd", "dmad::qk_norm_rope_bwd"} <= {e.key for e in p.key_averages()}
        return out
    with Names() as m:
        out = step(*args)
    assert [n for n in m.names if "dmad" in n] == ["dmad.qk_norm_rope_fwd.default", "dmad.qk_norm_rope_bwd.default"]
    return out


@pytest.mark.parametrize("device", ["cpu", pytest.param("gpu", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("how", ["dispatch mode", "profiled", "compiled"])
@pytest.mark.parametrize("absent", [(), ("k", "tk", "wk"), ("wq",), ("tq", "tk", "freqs")])
def test_op_and_direct_calls_agree_bitwise(request, monkeypatch, device, how, absent):
    if device == "cpu":
        _mock_kernels(monkeypatch)
    x = _small(request.getfixturevalue("gpu") if device == "gpu" else device, grad=True)
    x.update({n: None for n in absent})
    leaves = [n for n in ("q", "k", "wq", "wk") if x[n] is not None]
    want = _watched(x, leaves, "direct")
    got = _watched(x, leaves, how)
    assert len(got) == len(want)
    for a, b in zip(got, want):
        assert a.requires_grad == b.requires_grad and torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("empty", ["q", "k"])
def test_an_operand_without_heads(gpu, empty):
    """q or k of no heads beside the other: empty results and a zero gradient of its weight, the other as alone."""
    from dmad_amd import qk_norm_rope_with_tangent

    x = _small(gpu, dtype=torch.bfloat16)
    other = "k" if empty == "q" else "q"
    for n in ("q", "k", "wq", "wk"):
        x[n] = (x[n][:, :, :0] if n == empty else x[n]).detach().requires_grad_(True)
    (q, _), (k, _) = qk_norm_rope_with_tangent((x["q"], None), (x["k"], None), x["wq"], x["wk"], 1e-6, x["freqs"])
    y, none = (k, q) if empty == "q" else (q, k)
    assert none.shape == (2, 5, 0, 16)
    gx, gw = torch.autograd.grad(y.float().square().sum(), (x[other], x["w" + other]), retain_graph=True)
    both = torch.autograd.grad(y.float().square().sum() + none.float().sum(), (x[other], x["w" + other], x[empty], x["w" + empty]))
    assert torch.equal(both[0], gx) and torch.equal(both[1], gw)
    assert both[2].shape == (2, 5, 0, 16) and torch.equal(both[3], torch.zeros_like(both[3])) and both[3].shape == (16,)
    # the empty one alone
    (q, _), (k, _) = qk_norm_rope_with_tangent((x["q"], None), (x["k"], None), x["wq"], x["wk"], 1e-6, x["freqs"])
    none = q if empty == "q" else k
    ge, gw = torch.autograd.grad(none.float().sum(), (x[empty], x["w" + empty]))
    assert ge.shape == (2, 5, 0, 16) and torch.equal(gw, torch.zeros_like(gw))


# ---------------------------------------------------------------- sizes whose waves take several passes, past the caches


LARGE = [
    # S, Hq, Hk, D, dtype: odd numbers of wave passes per token, q's and k's within one wave's share
    (12701, 20, 8, 128, "bf16"),
    (17001, 33, 9, 64, "fp16"),
    (8001, 20, 8, 128, "fp32"),
    (15001, 9, 4, 256, "bf16"),
    (8803, 5, 12, 256, "fp32"),
]


@pytest.mark.gpu
@pytest.mark.parametrize("S,Hq,Hk,D,dtype", LARGE)
def test_large_calls(gpu, S, Hq, Hk, D, dtype):
    """What the large calls do and small ones do not: more than two passes per wave (from three rounds of 16384
    waves on) and, with tangents and backwards, more bytes than the caches hold, which go past them."""
    from dmad_amd import qk_norm_rope_with_tangent

    t = DTYPES[dtype]
    passes = -(-Hq * D // 512) + -(-Hk * D // 512)
    assert S * passes >= 3 * 16384 and passes % 2 and 3 * S * (Hq + Hk) * D * t.itemsize > 256 << 20
    print(f"case large norm S={S} Hq={Hq} Hk={Hk} D={D} {dtype}", flush=True)
    g = torch.Generator(device=gpu).manual_seed(S)

    def r(*shape, sd=1.0):
        return (torch.randn(shape, generator=g, device=gpu) * sd).to(t)

    x = dict(q=r(1, S, Hq, D), k=r(1, S, Hk, D), tq=r(1, S, Hq, D, sd=0.1), tk=r(1, S, Hk, D, sd=0.1), gq=r(1, S, Hq, D), gk=r(1, S, Hk, D),
             wq=1 + 0.3 * r(D).float(), wk=1 + 0.3 * r(D).float())
    f = torch.rand(S, D // 2, generator=g, device=gpu) * 200 - 100
    leaves = [x[n].requires_grad_(True) for n in ("q", "k", "wq", "wk")]
    (q, tq), (k, tk) = qk_norm_rope_with_tangent((x["q"], x["tq"]), (x["k"], x["tk"]), x["wq"], x["wk"], 1e-6, f)
    grads = torch.autograd.grad((q, k), leaves, (x["gq"], x["gk"]))
    torch.cuda.synchronize()
    for n, y, ty, dx, dw in (("q", q, tq, grads[0], grads[2]), ("k", k, tk, grads[1], grads[3])):
        z, w, d = x[n].detach().double(), x["w" + n].detach().double(), x["t" + n].double()
        root = (z.pow(2).mean(-1, keepdim=True) + 1e-6).rsqrt()
        m = z * root
        _check_there(n, y, st.rotate(m * w, f), None)
        mean = (m * d).mean(-1, keepdim=True)
        size = _pair_size((d.abs() + m.abs() * (m * d).abs().mean(-1, keepdim=True)) * root * w.abs())
        _check_there("t" + n, ty, st.rotate((d - m * mean) * root * w, f), size)
        u = st.rotate(x["g" + n].double(), -f)
        _check_there("dw" + n, dw, (u * m).sum((0, 1, 2)), (u * m).abs().sum((0, 1, 2)))
        a = u * w
        size = root * (_pair_size(a) + m.abs() * (a * m).abs().mean(-1, keepdim=True))
        _check_there("d" + n, dx, root * (a - m * (a * m).mean(-1, keepdim=True)), size)


def _check_there(name, got, ref, size):
    """_check on the device, a part at a time."""
    size = _pair_size(ref) if size is None else size
    if got.dim() == 4:
        for i in range(0, got.shape[1], 2000):
            _check(name, *(t[:, i:i + 2000].cpu() for t in (got.detach(), ref, size)))
    else:
        _check(name, got.detach().cpu(), ref.cpu(), size.cpu())


@pytest.mark.gpu
def test_registered_ops_do_what_they_declare(gpu):
    x = _small(gpu, grad=True)
    torch.library.opcheck(torch.ops.dmad.qk_norm_rope_fwd.default, (*(x[n] for n in OPERANDS), 1e-6))
    torch.library.opcheck(torch.ops.dmad.qk_norm_rope_fwd.default, (x["q"], None, None, None, x["wq"], None, None, 1e-6))
    y = {n: t.detach() for n, t in x.items()}
    torch.library.opcheck(torch.ops.dmad.qk_norm_rope_bwd.default, (y["q"], y["k"], y["tq"], y["tk"], y["wq"], y["wk"], y["freqs"], 1e-6, True, False))


HOOKS = {"type": lambda t: t.to(torch.bfloat16), "shape": lambda t: t[:, :3], "place": lambda t: t.to("meta")}


@pytest.mark.parametrize("kind", [*HOOKS, "a copy"])
def test_saved_operands_are_checked(kind):
    """What a saved-tensor hook brings back in another shape, type or place is refused before a kernel reads it as
    what it was."""
    from dmad_amd.prologue import _check_saved

    x, g = torch.zeros(2, 5, 4, 16), torch.zeros(2, 5, 4, 16)
    if kind == "a copy":
        _check_saved(x.clone(), g)
        _check_saved(None, None)
        return
    with pytest.raises(RuntimeError, match="as the forward read it"):
        _check_saved(HOOKS[kind](x), g)
    with pytest.raises(RuntimeError, match="nothing"):
        _check_saved(None, g)


@pytest.mark.gpu
def test_saved_tensor_hooks(gpu):
    """Through autograd: a hook that offloads and brings back works, one that changes what it brings back raises."""
    x = _small(gpu, grad=True)
    leaves = [x[n] for n in ("q", "k", "wq", "wk")]

    def grads(pack, unpack):
        with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
            q, _, k, _ = _run(x)
        return torch.autograd.grad(q.square().sum() + k.sum(), leaves)

    same = lambda t: t  # noqa: E731
    want = grads(same, same)
    for a, b in zip(grads(lambda t: t.cpu(), lambda t: t.to(gpu)), want):
        assert torch.equal(a, b)
    for unpack in (lambda t: t.to(torch.bfloat16), lambda t: t[:1], lambda t: t.cpu()):
        with pytest.raises(RuntimeError):
            (_run_hooked(x, unpack)).backward()


def _run_hooked(x, unpack):
    def only_operands(t):
        return unpack(t) if t.dim() == 4 else t

    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, only_operands):
        q, _, k, _ = _run(x)
    return q.sum() + k.sum()


@pytest.mark.parametrize("device", ["cpu", pytest.param("gpu", marks=pytest.mark.gpu)])
def test_registered_ops_refuse_what_the_calls_refuse(request, monkeypatch, device):
    if device == "cpu":
        _mock_kernels(monkeypatch)
    x = _small(request.getfixturevalue("gpu") if device == "gpu" else device)
    t = [x[n] for n in OPERANDS]
    fwd, bwd = torch.ops.dmad.qk_norm_rope_fwd, torch.ops.dmad.qk_norm_rope_bwd
    for i, bad in ((0, x["q"][:, :3]), (1, x["tq"][:1]), (2, x["k"].half()), (4, x["wq"][:8]), (6, x["freqs"][:4])):
        with pytest.raises(ValueError):
            fwd(*t[:i], bad, *t[i + 1:], 1e-6)
    if device == "gpu":  # (the check is part of the launch)
        with pytest.raises(RuntimeError, match="as the forward read it"):
            bwd(x["q"], x["k"], x["q"][:1], x["k"], x["wq"], x["wk"], x["freqs"], 1e-6, True, True)
        with pytest.raises(RuntimeError, match="nothing"):
            bwd(x["q"], None, x["q"], x["k"], x["wq"], None, x["freqs"], 1e-6, True, True)
