"""Rotations of queries and keys by their positions (qk_rotary_with_tangent, rotary_frequencies).

CPU: the oracle (oracle/block.py) against loops, the frequencies against their definitions, refusals, what watches
operators. GPU: the kernel against the oracle on the same inputs.

The kernel reduces angles in float64 and rounds a part of a turn to float32 (off by 2^-25 turns: pi 2^-24 radians), sine
and cosine come within 2 units in the last place, the factor and the two products and their sum round once each: an
element is off by half a step of its type plus less than STEPS = 16 half steps of float32 of |factor| times the larger
element of its pair. Elements behind the turned part are copied.
"""
import contextlib
import ctypes
import math
import weakref

import pytest
import torch

from oracle import block as ob

F32 = 2.0 ** -24
STEPS = 16
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _pair_size(x, R, half):
    """The larger magnitude of each element's pair; 0 behind the turned part."""
    a = x.abs().double().clone()
    a[..., R:] = 0
    t = a[..., :R].unflatten(-1, (2, R // 2) if half else (R // 2, 2))
    t = t.amax(-2 if half else -1, keepdim=True).expand_as(t)
    a[..., :R] = t.flatten(-2)
    return a


def _check(name, got, ref, size):
    u, tiny = torch.finfo(got.dtype).eps / 2, torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps
    tol = u * ref.abs() * (1 + 1e-3) + STEPS * F32 * size + tiny
    got = got.detach().cpu().double()
    assert torch.isfinite(got).all(), name
    worst = float(((got - ref).abs() / tol).max()) if got.numel() else 0.0
    print(f"  {name}: worst error {worst:.2f} of its bound", flush=True)
    assert worst <= 1.0, name


# ---------------------------------------------------------------- the oracle and the frequencies


def test_oracle_matches_loops():
    g = torch.Generator().manual_seed(0)
    x = torch.randn(2, 3, 2, 10, generator=g, dtype=torch.float64)
    f, pos = torch.rand(3, generator=g, dtype=torch.float64), torch.tensor([[0, 5, 9], [7, 7, 100]])
    for half in (False, True):
        y = ob.turn(x, pos, f, half, 1.5)
        for b in range(2):
            for s in range(3):
                for h in range(2):
                    want = x[b, s, h].tolist()
                    for i in range(3):
                        lo, hi = (i, i + 3) if half else (2 * i, 2 * i + 1)
                        a = float(pos[b, s]) * float(f[i])
                        u, v = float(x[b, s, h, lo]), float(x[b, s, h, hi])
                        want[lo], want[hi] = 1.5 * (u * math.cos(a) - v * math.sin(a)), 1.5 * (v * math.cos(a) + u * math.sin(a))
                    assert torch.allclose(y[b, s, h], torch.tensor(want, dtype=torch.float64), atol=1e-12)
        back = ob.turn(y, pos, f, half, 1 / 1.5, back=True)
        assert torch.allclose(back, x, atol=1e-12)


def test_frequencies():
    from dmad_amd import rotary_frequencies

    f, m = rotary_frequencies(8, 100.0, device="cpu")
    assert m == 1.0 and f.dtype == torch.float64
    assert torch.allclose(f, torch.tensor([1.0, 100 ** -0.25, 0.1, 100 ** -0.75], dtype=torch.float64), rtol=1e-15)
    lin, m = rotary_frequencies(8, 100.0, "linear", 4.0, device="cpu")
    assert m == 1.0 and torch.allclose(lin, f / 4)
    ntk, m = rotary_frequencies(8, 100.0, "ntk", 4.0, device="cpu")
    assert m == 1.0 and float(ntk[0]) == 1.0 and math.isclose(float(ntk[-1]), float(f[-1]) / 4, rel_tol=1e-12)
    yarn, m = rotary_frequencies(128, 10000.0, "yarn", 8.0, trained_length=4096, device="cpu")
    plain, _ = rotary_frequencies(128, 10000.0, device="cpu")
    turns = 4096 * plain / (2 * math.pi)
    assert math.isclose(m, 0.1 * math.log(8.0) + 1)
    assert torch.equal(yarn[turns >= 32], plain[turns >= 32])
    assert torch.allclose(yarn[turns <= 1], plain[turns <= 1] / 8, rtol=1e-15)
    mid = (turns > 1) & (turns < 32)
    assert mid.any() and ((yarn / plain)[mid] > 1 / 8).all() and ((yarn / plain)[mid] < 1).all()
    for bad in (dict(dim=7), dict(dim=0), dict(dim=8, theta=0.0), dict(dim=8, factor=math.inf), dict(dim=2, scaling="ntk"),
                dict(dim=8, scaling="yarn"), dict(dim=8, scaling="dynamic"), dict(dim=8, scaling="yarn", trained_length=10, fast=1.0)):
        with pytest.raises(ValueError, match="rotary_frequencies"):
            rotary_frequencies(device="cpu", **bad)


# ---------------------------------------------------------------- on the GPU


def _inputs(B, S, Hq, Hk, D, R, dtype, seed, layout="plain", far=131072):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g).to(dtype)  # noqa: E731
    if layout == "fused":
        qkv = r(B, S, Hq + 2 * Hk, D)
        q, k = qkv[:, :, :Hq], qkv[:, :, Hq:Hq + Hk]
    elif layout == "bhsd":
        q, k = r(B, Hq, S, D).transpose(1, 2), r(B, Hk, S, D).transpose(1, 2)
    elif layout == "odd":  # rows that start anywhere
        q, k = r(B, S, Hq, D + 3)[..., 1:D + 1], r(B, S, Hk, D + 5)[..., 2:D + 2]
    else:
        q, k = r(B, S, Hq, D), r(B, S, Hk, D)
    x = dict(q=q, k=k, tq=r(B, S, Hq, D), tk=r(B, Hk, S, D).transpose(1, 2), gq=r(B, S, Hq, D), gk=r(B, S, Hk, D))
    x["positions"] = torch.randint(0, far, (B, S), generator=g)
    x["frequencies"] = 10000.0 ** (-torch.arange(R // 2, dtype=torch.float64) * 2 / R)
    return x


def _to(t, dev):
    # (views keep their offset from an aligned start, so that their rows start where they did)
    if t.is_contiguous() or t.dtype == torch.float64:
        return t.to(dev)
    base = torch.empty_strided((t.untyped_storage().nbytes() // t.element_size(),), (1,), dtype=t.dtype, device=dev)
    return base.as_strided(t.shape, t.stride(), t.storage_offset()).copy_(t)


CASES = [
    # B, S, Hq, Hk, D, R, dtype, half, layout, positions, factor
    (1, 1, 1, 1, 2, 2, "fp32", False, "plain", "int64", 1.0),
    (2, 7, 3, 1, 9, 6, "bf16", True, "plain", "int32", 1.0),
    (1, 5, 2, 2, 16, 2, "fp16", False, "plain", "int64", 1.0),
    (32, 1, 32, 8, 128, 128, "bf16", True, "plain", "int32", 1.21),
    (1, 1, 40, 40, 128, 128, "bf16", False, "plain", "shared", 1.0),
    (3, 99, 32, 8, 64, 32, "fp16", True, "fused", "int32", 1.0),
    (2, 130, 12, 12, 128, 128, "bf16", False, "bhsd", "int32", 1.0),
    (1, 77, 9, 3, 80, 80, "fp32", True, "plain", "shared", 0.5),
    (1, 64, 4, 4, 80, 40, "bf16", True, "plain", "int64", 1.0),
    (2, 33, 7, 1, 96, 24, "fp16", False, "fused", "int32", 1.0),
    (1, 50, 4, 2, 256, 256, "bf16", True, "plain", "int64", 1.0),
    (1, 50, 4, 2, 256, 64, "fp32", False, "plain", "int32", -1.0),
    (2, 40, 6, 2, 128, 128, "bf16", True, "odd", "int32", 1.0),
    (1, 40, 1, 1, 20, 20, "fp16", True, "plain", "int32", 1.0),
    (1, 3, 1, 1, 8192, 8192, "bf16", True, "plain", "int32", 1.0),
    (1, 999, 40, 8, 32, 8, "bf16", True, "plain", "int32", 1.0),
    (1, 3000, 5, 1, 128, 128, "bf16", False, "plain", "int32", 1.0),
]


def _call(x, half, factor=1.0, tangents=True, **over):
    from dmad_amd import qk_rotary_with_tangent

    x = {**x, **over}
    t = (lambda n: x.get(n)) if tangents else (lambda n: None)
    return qk_rotary_with_tangent((x["q"], t("tq")), (x["k"], t("tk")), x["positions"], x["frequencies"],
                                  "half" if half else "interleaved", factor)


@pytest.mark.gpu
@pytest.mark.parametrize("B,S,Hq,Hk,D,R,dtype,half,layout,pos,factor", CASES)
def test_forward_tangent_backward(gpu, B, S, Hq, Hk, D, R, dtype, half, layout, pos, factor):
    print(f"case rotary B={B} S={S} Hq={Hq} Hk={Hk} D={D} R={R} {dtype} half={half} {layout} {pos}", flush=True)
    x = _inputs(B, S, Hq, Hk, D, R, DTYPES[dtype], D + S, layout)
    x["positions"] = x["positions"][0] if pos == "shared" else x["positions"].int() if pos == "int32" else x["positions"]
    d = {n: _to(t, gpu) for n, t in x.items()}
    for n in ("q", "k"):
        assert d[n].stride() == x[n].stride()
        d[n].requires_grad_(True)
    (q, tq), (k, tk) = _call(d, half, factor)
    assert q.requires_grad and not tq.requires_grad and q.is_contiguous() and q.dtype == DTYPES[dtype]
    grads = torch.autograd.grad((q, k), (d["q"], d["k"]), (d["gq"], d["gk"]))
    torch.cuda.synchronize()
    f = torch.tensor(factor).float().double()  # as the kernel takes it
    for n, y, ty, g in (("q", q, tq, grads[0]), ("k", k, tk, grads[1])):
        for name, got, src, back in ((n, y, x[n], False), ("t" + n, ty, x["t" + n], False), ("d" + n, g, x["g" + n], True)):
            ref = ob.turn(src.double(), x["positions"], x["frequencies"], half, f, back)
            _check(name, got, ref, abs(factor) * _pair_size(src, R, half))
            assert torch.equal(got.detach()[..., R:].cpu(), src[..., R:])
    with torch.no_grad():
        (q2, t2), (k2, _) = _call(d, half, factor, tangents=False)
    assert t2 is None and torch.equal(q2, q) and torch.equal(k2, k)


@pytest.mark.gpu
@pytest.mark.parametrize("half,R", [(False, 128), (True, 128), (False, 64)])
def test_calls_past_the_caches(gpu, half, R):
    """Calls of more than the caches hold (256 MB): bit for bit what their chunks of tokens give, forwards and backwards."""
    n, parts, H, D = 1500, 4, 40, 128
    S = parts * n
    assert 4 * S * 2 * H * D * 2 > 256e6 > 4 * n * 2 * H * D * 2 and 2 * 2 * S * 2 * H * D * 2 > 256e6
    g = torch.Generator(device=gpu).manual_seed(4)
    x = {k: torch.randn(1, S, H, D, generator=g, device=gpu).to(torch.bfloat16) for k in ("q", "tq", "k", "tk")}
    x["positions"] = torch.arange(S, device=gpu, dtype=torch.int32) + 7
    x["frequencies"] = 10000.0 ** (torch.arange(R // 2, device=gpu, dtype=torch.float64) * (-2.0 / R))
    whole = _call(x, half)
    q = x["q"].expand(2, S, H, D).detach().requires_grad_()  # two sequences: past the caches without tangents too
    k = x["k"].expand(2, S, H, D).detach().requires_grad_()
    (qo, _), (ko, _) = _call(x, half, tangents=False, q=q, k=k)
    torch.autograd.backward((qo, ko), (x["tq"].expand(2, S, H, D), x["tk"].expand(2, S, H, D)))
    for i in range(parts):
        rows = slice(i * n, (i + 1) * n)
        part = {m: t[:, rows] for m, t in x.items() if t.dim() == 4}
        part["positions"], part["frequencies"] = x["positions"][rows], x["frequencies"]
        some = _call(part, half)
        for a, b in zip((*whole[0], *whole[1]), (*some[0], *some[1])):
            assert torch.equal(a[:, rows], b)
        sq, sk = (part[m].detach().requires_grad_() for m in "qk")
        (oq, _), (ok, _) = _call(part, half, tangents=False, q=sq, k=sk)
        torch.autograd.backward((oq, ok), (part["tq"], part["tk"]))
        for b in range(2):
            for a, c in ((qo, oq), (ko, ok), (q.grad, sq.grad), (k.grad, sk.grad)):
                assert torch.equal(a[b:b + 1, rows], c)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("D,R", [(16, 16), (128, 128), (80, 40)])
def test_bits_do_not_depend_on_tangents_or_alignment(gpu, dtype, half, D, R):
    """Over a million elements: with tangents, without, and from rows that start anywhere, where the accesses are single."""
    S, H = 2 ** 20 // (5 * D), 3
    print(f"case bits {dtype} half={half} D={D} R={R}", flush=True)
    x = {n: _to(t, gpu) for n, t in _inputs(1, S, H, 2, D, R, DTYPES[dtype], 41).items()}

    def off(t):
        return torch.empty(t.numel() + 1, device=gpu, dtype=t.dtype)[1:].view(t.shape).copy_(t)

    with torch.no_grad():
        (q, tq), (k, tk) = _call(x, half, 1.25)
        for y in ({**x, "tq": None, "tk": None}, {n: off(t) if n in ("q", "k", "tq", "tk") else t for n, t in x.items()}):
            (q2, tq2), (k2, tk2) = _call(y, half, 1.25)
            assert torch.equal(q2, q) and torch.equal(k2, k)
            if tq2 is not None:
                assert torch.equal(tq2, tq) and torch.equal(tk2, tk)


@pytest.mark.gpu
@pytest.mark.parametrize("half", [False, True])
def test_more_elements_than_32_bits_count(gpu, half):
    """The last tokens of a call of more than 2^31 elements: bit for bit what a call of them alone gives."""
    S, H, D, n = 420000, 40, 128, 500
    assert S * H * D > 2 ** 31
    print(f"case beyond 32 bits half={half}", flush=True)
    x = {k: torch.empty(1, S, H, D, device=gpu, dtype=torch.bfloat16) for k in ("q", "tq")}
    for t in x.values():
        t.view(-1, 1000 * H * D)[:] = torch.randn(1000 * H * D, device=gpu).to(torch.bfloat16)
    x["positions"], x["frequencies"] = torch.arange(S, device=gpu), 10000.0 ** (-torch.arange(64, dtype=torch.float64, device=gpu) / 64)
    x["k"] = x["tk"] = None
    outs = _call(x, half)[0]
    last = {k: t if k in ("k", "tk", "frequencies") else t[-n:] if k == "positions" else t[:, -n:] for k, t in x.items()}
    for a, b in zip(outs, _call(last, half)[0]):
        assert torch.equal(a[:, -n:], b)


@pytest.mark.gpu
def test_far_and_negative_positions(gpu):
    """Angles of many turns are as exact as near ones; positions are any whole numbers."""
    x = _inputs(1, 6, 2, 1, 64, 64, torch.float32, 3)
    x["positions"] = torch.tensor([[0, -1, 1 << 20, -(1 << 30), (1 << 31) - 1, 1 << 40]])
    # the product of a position of 2^40 and a frequency up to 1 is off by 2^-13 turns of float64 there: compare those
    # where it is below 2^-24, all but the last
    d = {n: t.to(gpu) for n, t in x.items()}
    for half in (False, True):
        (q, _), (k, _) = _call(d, half, tangents=False)
        for n, y in (("q", q), ("k", k)):
            ref = ob.turn(x[n].double(), x["positions"], x["frequencies"], half)
            _check(n, y[:, :5], ref[:, :5], _pair_size(x[n], 64, half)[:, :5])
            assert torch.isfinite(y[:, 5]).all()


@pytest.mark.gpu
def test_equals_the_rotation_by_a_table(gpu):
    """Neighbours, the whole head: what apply_rope_with_tangent gives for the table of angles, within one rounding each."""
    from dmad_amd import apply_rope_with_tangent

    x = _inputs(2, 50, 4, 4, 128, 128, torch.bfloat16, 4, far=500)
    d = {n: t.to(gpu) for n, t in x.items()}
    d["positions"] = d["positions"][0]
    (q, tq), _ = _call(d, False)
    freqs = (d["positions"].double()[:, None] * d["frequencies"]).float()
    r, tr = apply_rope_with_tangent(d["q"], d["tq"], freqs)
    # a table in float32 holds 500 radians to 2^-16: 2^-15 of the pair, and one half step of bf16 each
    for a, b, src in ((q, r, "q"), (tq, tr, "tq")):
        size = _pair_size(x[src], 128, False).to(gpu)
        assert ((a.double() - b.double()).abs() <= 2 * 2.0 ** -8 * b.double().abs() + 2.0 ** -14 * size).all()


@pytest.mark.gpu
def test_one_operand_partial_gradients_and_no_heads(gpu):
    x = _inputs(2, 19, 4, 2, 64, 32, torch.bfloat16, 7)
    d = {n: t.to(gpu) for n, t in x.items()}
    both = _call(d, True)
    (q, tq), none = _call(d, True, k=None, tk=None)
    assert none == (None, None) and torch.equal(q, both[0][0]) and torch.equal(tq, both[0][1])
    none, (k, _) = _call(d, True, q=None, tq=None)
    assert none == (None, None) and torch.equal(k, both[1][0])
    y = {n: d[n].clone().requires_grad_(True) for n in ("q", "k")}
    (_, _), (k, _) = _call({**d, **y}, True)
    k.float().square().sum().backward()
    assert y["q"].grad is None and y["k"].grad is not None
    # a summed output's gradient is an expanded scalar
    (q, _), (k, _) = _call({**d, **y}, True)
    (g,) = torch.autograd.grad(q.sum(), y["q"])
    (q, _), (k, _) = _call({**d, **y}, True)
    (h,) = torch.autograd.grad(q, y["q"], torch.ones_like(q))
    assert torch.equal(g, h)
    empty = {"k": d["k"][:, :, :0].detach().requires_grad_(True), "tk": d["tk"][:, :, :0]}
    (q, _), (k, _) = _call({**d, **empty}, True)
    assert k.shape == (2, 19, 0, 64) and torch.equal(q, both[0][0])
    (g,) = torch.autograd.grad(k.float().sum(), empty["k"])
    assert g.shape == (2, 19, 0, 64)
    e = torch.zeros(0, 4, 3, 32, device=gpu, requires_grad=True)
    (y, _), _ = _call(dict(q=e, k=None, positions=torch.zeros(0, 4, device=gpu, dtype=torch.int32), frequencies=d["frequencies"]), True)
    assert y.shape == e.shape and torch.autograd.grad(y.sum(), e)[0].shape == e.shape


@pytest.mark.gpu
def test_nan_and_infinity_stay_with_their_pair(gpu):
    x = _inputs(1, 4, 3, 1, 64, 32, torch.bfloat16, 8)
    d = {n: t.to(gpu) for n, t in x.items()}
    for half, mate in ((False, 7), (True, 22)):
        clean = _call(d, half, tangents=False)[0][0]
        q = d["q"].clone()
        q[0, 1, 2, 6] = math.nan
        q[0, 2, 0, 40] = math.inf  # behind the turned part
        got = _call(d, half, tangents=False, q=q)[0][0]
        assert torch.isnan(got[0, 1, 2, [6, mate]]).all() and got[0, 2, 0, 40] == math.inf
        got[0, 1, 2, [6, mate]], got[0, 2, 0, 40] = clean[0, 1, 2, [6, mate]], clean[0, 2, 0, 40]
        assert torch.equal(got, clean)


@pytest.mark.gpu
def test_captured_and_on_another_stream(gpu):
    """Positions are read on the device: a replay turns by what stands there."""
    x = _inputs(2, 300, 6, 2, 128, 128, torch.bfloat16, 15)
    d = {n: t.to(gpu) for n, t in x.items()}

    def step():
        y = {n: d[n].detach().requires_grad_(True) for n in ("q", "k")}
        (q, tq), (k, tk) = _call({**d, **y}, True)
        return [q.detach(), tq, k.detach(), tk, *torch.autograd.grad((q, k), (y["q"], y["k"]), (d["gq"], d["gk"]))]

    ref = [t.clone() for t in step()]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(other, ref))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(3):
        d["positions"].add_(i)
        want = [t.clone() for t in step()]
        junk = torch.randn(1024, 1024, device=gpu)
        (junk @ junk).sum().item()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


@pytest.mark.gpu
def test_no_second_derivative(gpu):
    x = _inputs(1, 4, 2, 1, 32, 32, torch.float32, 9)
    d = {n: t.to(gpu) for n, t in x.items()}
    d["q"].requires_grad_(True)

    def grad(create_graph):
        (q, _), _ = _call(d, False, tangents=False)
        return torch.autograd.grad(q.square().sum(), d["q"], create_graph=create_graph)[0]

    g = grad(True)
    assert torch.equal(g.detach(), grad(False))
    with pytest.raises(RuntimeError, match="differentiate twice"):
        g.sum().backward()


# ---------------------------------------------------------------- refusals


def test_refusals_on_the_cpu():
    from dmad_amd import qk_rotary_with_tangent

    with pytest.raises(RuntimeError, match="GPU only"):
        qk_rotary_with_tangent((torch.randn(1, 2, 3, 32), None), (None, None), torch.arange(2), torch.ones(16).double())


@pytest.mark.parametrize("error,match,over", [
    (ValueError, "neither q nor k", dict(q=None, k=None, tq=None, tk=None)),
    (ValueError, r"\[B, S, H, D\]", dict(q=(5, 4, 16))),
    (ValueError, "heads", dict(k=(2, 4, 2, 16))),
    (ValueError, "heads", dict(k=(2, 5, 2, 18))),
    (ValueError, "and k", dict(k=torch.float16)),
    (NotImplementedError, "dtype", dict(q=torch.float64, k=torch.float64, tq=None, tk=None)),
    (ValueError, "tangents of both", dict(tk=None)),
    (ValueError, "shape and type", dict(tq=(2, 5, 3, 16))),
    (ValueError, "positions", dict(positions=None)),
    (ValueError, "positions", dict(positions=(2, 4))),
    (ValueError, "positions", dict(positions=torch.float32)),
    (ValueError, "frequencies", dict(frequencies=torch.float32)),
    (ValueError, "frequencies", dict(frequencies=(0,))),
    (ValueError, "frequencies", dict(frequencies=(9,))),
    (ValueError, "layout", dict(layout="quarter")),
    (ValueError, "factor", dict(factor=math.nan)),
])
def test_refusals(monkeypatch, error, match, over):
    from dmad_amd import qk_rotary_with_tangent

    _mock_kernels(monkeypatch)
    x = _small()
    how = {k: over[k] for k in ("layout", "factor") if k in over}
    for n, v in over.items():
        if n not in how:
            x[n] = None if v is None else torch.zeros(v, dtype=x[n].dtype) if isinstance(v, tuple) else x[n].to(v)
    with pytest.raises(error, match=match):
        qk_rotary_with_tangent((x["q"], x["tq"]), (x["k"], x["tk"]), x["positions"], x["frequencies"], **how)


def _strides(*v):
    return (ctypes.c_int64 * len(v))(*v)


@pytest.mark.parametrize("over,code,needle", [
    (dict(dtype=9), 2, "dtype"),
    (dict(D=0), 1, "sizes"),
    (dict(Hq=0, Hk=0), 1, "sizes"),
    (dict(S=-1), 1, "sizes"),
    (dict(R=0), 1, "turned part"),
    (dict(R=7), 1, "turned part"),
    (dict(R=66), 1, "turned part"),
    (dict(layout=2), 1, "layout"),
    (dict(factor=math.inf), 1, "factor"),
    (dict(q=0), 1, "q: null"),
    (dict(Hk=0), 1, "no heads"),
    (dict(tq=256), 1, "neither"),
    (dict(q=257), 1, "element"),
    (dict(qs=_strides(512, 256, 64, 2)), 1, "head dim must be 1"),
    (dict(ks=_strides(512, -256, 64, 1)), 1, "negative"),
    (dict(oq=0), 1, "output"),
    (dict(positions=0), 1, "positions"),
    (dict(frequencies=0), 1, "positions and frequencies"),
    (dict(B=1 << 20, S=1 << 20), 2, "too many"),
    (dict(D=16384, R=2), 2, "too many"),
    (dict(Hq=1 << 19, D=128, R=2), 2, "too many"),
])
def test_c_entry_rejects_bad_arguments(over, code, needle):
    from dmad_amd import _native as nat

    a = dict(dtype=0, B=1, S=2, Hq=4, Hk=2, D=64, R=64, q=256, tq=0, k=256, tk=0, qs=_strides(512, 256, 64, 1),
             ks=_strides(256, 128, 64, 1), positions=256, frequencies=256, layout=1, factor=1.0, oq=256, ok=256)
    a.update(over)
    p = ctypes.c_void_p
    rc = nat.lib().dmad_qk_rotary(a["dtype"], a["B"], a["S"], a["Hq"], a["Hk"], a["D"], a["R"], p(a["q"]), p(a["tq"]), p(a["k"]),
                                  p(a["tk"]), a["qs"], a["qs"], a["ks"], a["ks"], p(a["positions"]), 0, _strides(2, 1),
                                  p(a["frequencies"]), a["layout"], 0, a["factor"], p(a["oq"]), p(0), p(a["ok"]), p(0), p(0))
    assert rc == code, nat.lib().dmad_last_error()
    assert needle in nat.lib().dmad_last_error().decode()


def test_the_walk_covers_every_element_once(tmp_path):
    """The host's plan (access width, units, tile, multipliers) and the kernel's walk over it, on the CPU: every element of
    the outputs is written once and every pair turned by its own angle, inside the tile's sines."""
    import subprocess

    src = tmp_path / "walk.cpp"
    src.write_text(WALK)
    from dmad_amd import build as b

    exe = tmp_path / "walk"
    subprocess.run([b._hipcc(), "-x", "hip", "--offload-arch=gfx950", "-std=c++17", "-O1", "-Xclang", "-target-feature", "-Xclang",
                    "-packed-fp32-ops", "-I", b.CSRC, str(src), "-o", str(exe)], check=True, capture_output=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True)
    assert out.returncode == 0, out.stdout + out.stderr


WALK = r"""
#include <cstdio>
#include <vector>
#include "rotary.hip"
using namespace dmad;
static uint32_t hi(uint32_t a, uint32_t b) { return (uint32_t)(((uint64_t)a * b) >> 32); }
static int quot(int x, uint32_t m) { return m == 0 ? x : (int)hi((uint32_t)x, m); }
int main() {
  const int shapes[][6] = {{1, 1, 1, 0, 2, 2}, {2, 7, 3, 1, 9, 6}, {1, 5, 2, 2, 16, 2}, {32, 1, 32, 8, 128, 128}, {3, 99, 32, 8, 64, 32},
                           {1, 77, 9, 3, 80, 80}, {1, 64, 4, 4, 80, 40}, {2, 33, 7, 1, 96, 24}, {1, 50, 4, 2, 256, 64}, {1, 40, 1, 1, 20, 20},
                           {1, 3, 1, 1, 8192, 8192}, {1, 3000, 1, 0, 16, 4}, {1, 40, 1, 1, 3, 2}, {1, 9, 1000, 24, 128, 128}};
  for (auto& z : shapes)
    for (int esz : {2, 4})
      for (int align : {1, 2, 4, 8})
        for (int inter : {0, 1}) {
          RotaryParams p{};
          p.B = z[0]; p.S = z[1]; p.op[0].H = z[2]; p.op[1].H = z[3]; p.D = z[4]; p.R = z[5];
          p.tokens = (int64_t)p.B * p.S;
          p.interleaved = inter;
          if (!rotary_plan(p, esz, align)) { printf("no plan\n"); return 1; }
          const int V = p.vec, pairs = p.R / 2, heads = z[2] + z[3];
          if (V * esz > 16 || V > align || p.tile < 1 || p.tile > kRotaryMaxTile || p.tile * pairs > kRotaryLdsPairs) { printf("bad plan\n"); return 1; }
          // one tile is like another: the first and the last
          for (int64_t token0 : {(int64_t)0, (p.tokens - 1) / p.tile * p.tile}) {
            const int tokens = (int)(p.tokens - token0 < p.tile ? p.tokens - token0 : p.tile);
            std::vector<int> wrote((size_t)tokens * heads * p.D, 0);
            for (int i = 0; i < tokens * p.per_token; ++i) {
              const int k = quot(i, p.token_mul), in = i - k * p.per_token;
              const int h = quot(in, p.head_mul), unit = in - h * p.per_head, turned = pairs / V;
              if (k != i / p.per_token || h != in / p.per_head || k >= tokens || h >= heads) { printf("bad quotient\n"); return 1; }
              const bool turns = unit < turned;
              const bool pair = inter && V == 1;
              const int first = turns ? (pair ? 2 * unit : V * unit) : p.R + 2 * V * (unit - turned);
              const int second = turns ? (pair ? first + 1 : first + pairs) : first + V;
              const int angle = (inter && V > 1 ? V / 2 : V) * unit;
              if (turns && inter && V > 1 && (pairs % 2 || angle != first / 2 || angle + pairs / 2 != second / 2 || angle + pairs / 2 + V / 2 > pairs)) {
                printf("angles of neighbours\n");
                return 1;
              }
              if (turns && V * unit + V > pairs) { printf("angles beyond the row\n"); return 1; }
              for (int f : {first, second}) {
                if (f == second && second >= p.D) continue;
                if (f % V || f + V > p.D) { printf("access beyond the row %d %d %d\n", f, V, p.D); return 1; }
                for (int e = 0; e < V; ++e) ++wrote[((size_t)k * heads + h) * p.D + f + e];
              }
            }
            for (int w : wrote) if (w != 1) { printf("D %d R %d V %d: written %d times\n", p.D, p.R, V, w); return 1; }
          }
        }
  return 0;
}
"""


# ---------------------------------------------------------------- what watches operators, and tensors that are not their memory


def _mock_kernels(monkeypatch):
    """The oracle in place of the launch, on CPU tensors, which it takes as the kernel does: by their memory."""
    from dmad_amd import block_ops

    def launch(call, q, tq, k, tk, transposed):
        for t in (q, tq, k, tk, call.positions, call.frequencies):
            assert t is None or (t.data_ptr() and not t.is_neg()), "a tensor whose memory does not hold its values"
        return [None if t is None else ob.turn(t.detach().double(), call.positions, call.frequencies, call.layout == 1, call.factor,
                                               bool(transposed)).to(t.dtype) for t in (q, tq, k, tk)]

    monkeypatch.setattr(block_ops, "_check_same_device", lambda op, *ts: None)
    monkeypatch.setattr(block_ops, "_rotary_launch", launch)


BOTH = pytest.mark.parametrize("device", ["cpu", pytest.param("gpu", marks=pytest.mark.gpu)])
OPERANDS = ("q", "tq", "k", "tk", "positions", "frequencies")


def _small(device="cpu", grad=False):
    x = {n: t.to(device).clone() for n, t in _inputs(2, 5, 4, 2, 16, 8, torch.float32, 3).items()}
    for n in ("q", "k"):
        x[n].requires_grad_(grad)
    return x


def _set_up(request, monkeypatch, device, **how):
    if device == "cpu":
        _mock_kernels(monkeypatch)
    return _small(request.getfixturevalue("gpu") if device == "gpu" else device, **how)


def _run(x):
    (q, tq), (k, tk) = _call(x, True, 1.25)
    return q, tq, k, tk


@BOTH
@pytest.mark.parametrize("name", ("q", "tq", "k", "tk", "frequencies"))
def test_forward_mode_is_refused(request, monkeypatch, device, name):
    x = _set_up(request, monkeypatch, device)
    with torch.no_grad(), torch.autograd.forward_ad.dual_level():
        _run(x)
        dual = torch.autograd.forward_ad.make_dual(x[name], torch.ones_like(x[name]))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            _run({**x, name: dual})
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(lambda t: _run({**x, name: t})[0], (x[name],), (torch.ones_like(x[name]),))


@BOTH
@pytest.mark.parametrize("name", OPERANDS)
def test_negated_views_have_their_sign(request, monkeypatch, device, name):
    x = _set_up(request, monkeypatch, device)
    want = _run({**x, name: -x[name]})
    odd = torch._neg_view(x[name])
    assert odd.is_neg()
    for a, b in zip(_run({**x, name: odd}), want):
        assert torch.equal(a, b)
    x["q"] = x["q"].clone().requires_grad_(True)
    q = _run(x)[0]
    g = torch.ones_like(q)
    assert torch.equal(torch.autograd.grad(q, x["q"], torch._neg_view(g), retain_graph=True)[0], torch.autograd.grad(q, x["q"], -g)[0])


@BOTH
def test_frequencies_that_want_a_gradient_are_refused(request, monkeypatch, device):
    x = _set_up(request, monkeypatch, device)
    x["frequencies"].requires_grad_(True)
    with pytest.raises(RuntimeError, match="gradient of the frequencies"):
        _run(x)
    with torch.no_grad():
        _run(x)


def test_meta_tensors_give_shapes():
    x = _small("meta", grad=True)
    outs = _run(x)
    assert [tuple(o.shape) for o in outs] == [(2, 5, 4, 16)] * 2 + [(2, 5, 2, 16)] * 2 and all(o.is_meta for o in outs)
    assert outs[0].requires_grad and not outs[1].requires_grad
    for n, g in zip(("q", "k"), torch.autograd.grad(outs[0].sum() + outs[2].sum(), (x["q"], x["k"]))):
        assert g.is_meta and g.shape == x[n].shape


def test_batched_cotangents(monkeypatch):
    _mock_kernels(monkeypatch)
    x = _small(grad=True)
    q, _, k, _ = _run(x)
    cts = [torch.randn(3, *o.shape) for o in (q, k)]
    got = torch.autograd.grad((q, k), (x["q"], x["k"]), cts, is_grads_batched=True, retain_graph=True)
    for i in range(3):
        for a, b in zip(got, torch.autograd.grad((q, k), (x["q"], x["k"]), [c[i] for c in cts], retain_graph=True)):
            torch.testing.assert_close(a[i], b)


@BOTH
@pytest.mark.parametrize("how", ["dispatch mode", "profiled", "compiled"])
@pytest.mark.parametrize("absent", [(), ("k", "tk"), ("q", "tq"), ("tq", "tk")])
def test_op_and_direct_calls_agree_bitwise(request, monkeypatch, device, how, absent):
    from torch.utils._python_dispatch import TorchDispatchMode

    x = _set_up(request, monkeypatch, device, grad=True)
    x.update({n: None for n in absent})
    names = [n for n in ("q", "k") if x[n] is not None]
    seen = []

    class Names(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(str(func))
            return func(*args, **(kwargs or {}))

    def forward(*ls):
        return [o for o in _run({**x, **dict(zip(names, ls))}) if o is not None]

    def step(fn, *ls):
        outs = fn(*ls)
        return list(outs) + list(torch.autograd.grad(sum(o.square().sum() for o in outs if o.requires_grad), ls))

    args = [x[n] for n in names]
    want = step(forward, *args)
    if how == "compiled":
        got = step(torch.compile(forward, fullgraph=True, backend="aot_eager"), *args)
    elif how == "profiled":
        with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CPU]) as p:
            got = step(forward, *args)
        assert {"dmad::qk_rotary_fwd", "dmad::qk_rotary_bwd"} <= {e.key for e in p.key_averages()}
    else:
        with Names():
            got = step(forward, *args)
        assert [n for n in seen if "dmad" in n] == ["dmad.qk_rotary_fwd.default", "dmad.qk_rotary_bwd.default"]
    assert len(got) == len(want)
    for a, b in zip(got, want):
        assert a.requires_grad == b.requires_grad and torch.equal(a, b)


@pytest.mark.gpu
def test_registered_ops_do_what_they_declare(gpu):
    x = _small(gpu, grad=True)
    torch.library.opcheck(torch.ops.dmad.qk_rotary_fwd.default, (*(x[n] for n in OPERANDS), True, 1.5))
    torch.library.opcheck(torch.ops.dmad.qk_rotary_fwd.default, (None, None, x["k"], None, x["positions"], x["frequencies"], False, 1.0))
    torch.library.opcheck(torch.ops.dmad.qk_rotary_bwd.default, (x["gq"], None, x["positions"], x["frequencies"], True, 1.5))


@BOTH
@pytest.mark.parametrize("when", ["packed", "after the backward"])
def test_angles_are_kept_by_their_saved_tensors_alone(request, monkeypatch, device, when):
    """Hooks that move what is saved move all of it, and a graph that lives on after its backward holds nothing."""
    leaves = _set_up(request, monkeypatch, device, grad=True)
    x = {n: t * 1 for n, t in leaves.items()}
    there = {n: weakref.ref(t) for n, t in x.items()}
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.clone(), lambda t: t) if when == "packed" else contextlib.nullcontext():
        q, _, k, _ = _run(x)
    if when != "packed":
        torch.autograd.grad(q.sum() + k.sum(), (leaves["q"], leaves["k"]))
    del x
    assert [n for n, r in there.items() if r() is not None] == []
    assert q.requires_grad


@BOTH
@pytest.mark.parametrize("shared", [False, True])
def test_angles_from_hooks(request, monkeypatch, device, shared):
    """What comes back from hooks may lie otherwise than it did; in another shape, type or place it is refused."""
    x = _set_up(request, monkeypatch, device, grad=True)
    if shared:
        x["positions"], x["frequencies"] = x["positions"][:1].expand(2, -1), torch.stack((x["frequencies"],) * 2, -1)[:, 0]

    def grads(pack, unpack):
        with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
            q, _, k, _ = _run(x)
        return torch.autograd.grad(q.square().sum() + k.sum(), (x["q"], x["k"]))

    want = grads(lambda t: t, lambda t: t)
    for unpack in (lambda t: t.clone(memory_format=torch.contiguous_format), lambda t: torch.stack((t, t), -1)[..., 0]):
        for a, b in zip(grads(lambda t: t, unpack), want):
            assert torch.equal(a, b)
    wrong = [lambda t: t[..., :-1], lambda t: t.to(torch.int16), lambda t: t[None, None]]
    for change in wrong + ([lambda t: t.cpu()] if device == "gpu" else []):
        for dtype in (x["positions"].dtype, torch.float64):
            with pytest.raises((RuntimeError, ValueError), match="as the forward read them"):
                grads(lambda t: t, lambda t: change(t) if t.dtype == dtype else t)


@BOTH
def test_registered_ops_refuse_what_the_calls_refuse(request, monkeypatch, device):
    x = _set_up(request, monkeypatch, device)
    t = [x[n] for n in OPERANDS]
    for i, bad in ((1, x["tq"][:1]), (2, x["k"].half()), (4, x["positions"][:, :3]), (5, x["frequencies"].float())):
        with pytest.raises(ValueError):
            torch.ops.dmad.qk_rotary_fwd(*t[:i], bad, *t[i + 1:], True, 1.0)
    with pytest.raises(ValueError, match="positions"):
        torch.ops.dmad.qk_rotary_bwd(x["gq"][:, :3], None, x["positions"], x["frequencies"], True, 1.0)


@BOTH
def test_a_change_in_place_is_noticed(request, monkeypatch, device):
    x = _set_up(request, monkeypatch, device, grad=True)
    q = _run(x)[0]
    x["positions"].add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        q.sum().backward()
