"""The operators around the attention together, as a block uses them: a training step with tangents, and the decoding of
continuations that share a prefix, against the same blocks in float64.

Rounding between the operators is the operands' type's in both; errors then pass through a few products, so results are
compared by relative L2 norm: each of the about 8 roundings on the way to an output is off by at most half a step u of
its type (u / sqrt(3) rms), projections average them, and the softmax's scores (about 1) turn a relative error e of q and k
into one of the same size in the weights: 16 u bounds the lot."""
import pytest
import torch

from oracle import block as ob

EPS = 1e-6


def _rel(a, b):
    a, b = a.detach().cpu().double(), b.detach().cpu().double()
    return float((a - b).norm() / b.norm())


def _weights(C, H, D, F, seed):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s, sd=1.0: torch.randn(s, generator=g) * sd  # noqa: E731
    w = {n: r(C, H * D, sd=C ** -0.5) for n in ("wq", "wk", "wv")}
    w["wo"] = r(H * D, C, sd=C ** -0.5)
    w["mods"] = r(1, F, 5 * C, sd=0.3)  # shift, scale of the first norm; gate; shift, scale of the second
    return {n: t.bfloat16() for n, t in w.items()}


def _mods(m, C):
    return [m[..., i * C:(i + 1) * C] for i in range(5)]


@pytest.mark.gpu
def test_a_block_with_tangents_and_gradients(gpu):
    """x -> norm, modulate -> q, k, v -> rotate -> attention with tangents -> project -> gate, residual, norm, modulate."""
    from dmad_amd import (gated_residual_norm_with_tangent, qk_rotary_with_tangent, rotary_frequencies, torch_attention_op_withT)

    B, S, H, D, F = 2, 96, 4, 64, 3
    C = H * D
    g = torch.Generator().manual_seed(1)
    w = _weights(C, H, D, F, 2)
    x = torch.randn(B, S, C, generator=g).bfloat16()
    tx = (torch.randn(B, S, C, generator=g) * 0.1).bfloat16()
    mods = w["mods"].expand(B, F, 5 * C).contiguous()
    tmods = (torch.randn(mods.shape, generator=g) * 0.1).bfloat16()
    gx, gn = (torch.randn(B, S, C, generator=g).bfloat16() for _ in range(2))
    pos = torch.arange(S)
    freqs, by = rotary_frequencies(32, 10000.0, "yarn", 4.0, trained_length=64, device="cpu")

    def ours(x, tx, mods, tmods, w):
        m, tm = _mods(mods, C), _mods(tmods, C)
        _, (n, tn) = gated_residual_norm_with_tangent((x, tx), scale_withT=(m[1], tm[1]), shift_withT=(m[0], tm[0]), eps=EPS)
        q, k, v = ((n @ w[i]).view(B, S, H, D) for i in ("wq", "wk", "wv"))
        tq, tk, tv = ((tn @ w[i]).detach().view(B, S, H, D) for i in ("wq", "wk", "wv"))
        qT, kT = qk_rotary_with_tangent((q, tq), (k, tk), pos.to(x.device), freqs.to(x.device), "half", by)
        o, to = torch_attention_op_withT(qT, kT, (v, tv))
        y, ty = o.reshape(B, S, C) @ w["wo"], to.reshape(B, S, C) @ w["wo"]
        return gated_residual_norm_with_tangent((x, tx), (y, ty.detach()), (m[2], tm[2]), (m[4], tm[4]), (m[3], tm[3]), eps=EPS)

    def plain(x, mods):
        """The primal in float64; its tangent is torch's."""
        m = _mods(mods, C)
        _, n = ob.gated_norm(x, scale=m[1], shift=m[0], eps=EPS)
        q, k, v = ((n @ w[i].double()).view(B, S, H, D) for i in ("wq", "wk", "wv"))
        q, k = (_turn(t, by).transpose(1, 2) for t in (q, k))
        p = torch.softmax(q @ k.transpose(2, 3) * D ** -0.5, -1)
        y = (p @ v.transpose(1, 2)).transpose(1, 2).reshape(B, S, C) @ w["wo"].double()
        return ob.gated_norm(x, y, m[2], m[4], m[3], eps=EPS)

    def _turn(t, by):
        angle = (pos.double()[:, None] * freqs)[None, :, None]
        c, s = angle.cos() * by, angle.sin() * by
        a, b = t[..., :16], t[..., 16:32]
        return torch.cat((a * c - b * s, b * c + a * s, t[..., 32:]), -1)

    d = {n: t.to(gpu) for n, t in w.items()}
    xs, ms = x.to(gpu).requires_grad_(True), mods.to(gpu).requires_grad_(True)
    (xo, txo), (n, tn) = ours(xs, tx.to(gpu), ms, tmods.to(gpu), d)
    dx, dm = torch.autograd.grad((xo, n), (xs, ms), (gx.to(gpu), gn.to(gpu)))

    xr, mr = x.double().requires_grad_(True), mods.double().requires_grad_(True)
    rx, rn = plain(xr, mr)
    rdx, rdm = torch.autograd.grad((rx, rn), (xr, mr), (gx.double(), gn.double()))
    _, (rtx, rtn) = torch.func.jvp(plain, (x.double(), mods.double()), (tx.double(), tmods.double()))
    bound = 16 * 2.0 ** -8
    for name, a, b in (("x'", xo, rx), ("n", n, rn), ("tx'", txo, rtx), ("tn", tn, rtn), ("dx", dx, rdx), ("dmods", dm, rdm)):
        e = _rel(a, b)
        print(f"  {name}: {e:.2e} of {bound:.2e}", flush=True)
        assert e <= bound, name


@pytest.mark.gpu
@pytest.mark.parametrize("captured", [False, True])
def test_decoding_continuations_of_one_prefix(gpu, captured):
    """Steps of 6 continuations: norm, rotate by the cache's own positions, append, attend behind the shared prefix, gate,
    residual, norm; eager and as one captured graph replayed step by step."""
    from dmad_amd import (PagedKVCache, append_kv, gated_residual_norm_with_tangent, qk_rotary_with_tangent, rotary_frequencies,
                          shared_prefix_attention)

    B, H, Hk, D, L, steps = 6, 8, 2, 64, 150, 5
    C = H * D
    g = torch.Generator().manual_seed(5)
    r = lambda *s, sd=1.0: (torch.randn(s, generator=g) * sd).bfloat16()  # noqa: E731
    w = {"wq": r(C, C, sd=C ** -0.5), "wk": r(C, Hk * D, sd=C ** -0.5), "wv": r(C, Hk * D, sd=C ** -0.5), "wo": r(C, C, sd=C ** -0.5)}
    norm_w = torch.rand(C, generator=g) + 0.5
    past, xs = r(1, L, C), [r(B, 1, C) for _ in range(steps)]
    freqs, by = rotary_frequencies(D, device="cpu")

    # float64: all tokens of a sequence at once, the prefix first
    def reference(b):
        x = torch.cat([past[0]] + [x[b] for x in xs]).double()
        n = ob.gated_norm(x[None], weight=norm_w.double(), kind="rms", eps=EPS)[1]
        T = L + steps
        q, k, v = ((n[0] @ w[i].double()).view(T, -1, D) for i in ("wq", "wk", "wv"))
        q, k = (ob.turn(t[None], torch.arange(T), freqs, True)[0] for t in (q, k))
        k, v = (t.repeat_interleave(H // Hk, 1) for t in (k, v))
        s = torch.einsum("qhd,khd->hqk", q, k) * D ** -0.5
        s = s.masked_fill(torch.arange(T) > torch.arange(T)[:, None], -float("inf"))
        o = torch.einsum("hqk,khd->qhd", torch.softmax(s, -1), v).reshape(T, C)[L:]
        return ob.gated_norm(x[None, L:], (o @ w["wo"].double())[None], weight=norm_w.double(), kind="rms", eps=EPS)

    d = {n: t.to(gpu) for n, t in w.items()}
    nw, f = norm_w.to(gpu), freqs.to(gpu)
    prefix = PagedKVCache.allocate(1, L, Hk, D, device=gpu, page_size=16, track_weights=False)
    cache = PagedKVCache.allocate(B, 16, Hk, D, device=gpu, page_size=16, track_weights=False)
    cache.seen.fill_(L)  # the next token's position

    def qkv(x, positions):
        _, (n, _) = gated_residual_norm_with_tangent((x, None), weight=nw, eps=EPS, norm="rms")
        q, k, v = ((n @ d[i]).view(*x.shape[:2], -1, D) for i in ("wq", "wk", "wv"))
        (q, _), (k, _) = qk_rotary_with_tangent((q, None), (k, None), positions, f, "half", by)
        return q, k, v

    def step(x):
        q, k, v = qkv(x, cache.seen[:, None])
        append_kv(k, v, cache)
        o = shared_prefix_attention(q, prefix, cache, causal=True)
        (xo, _), (n, _) = gated_residual_norm_with_tangent((x, None), (o.view(B, 1, C) @ d["wo"], None), weight=nw, eps=EPS, norm="rms")
        return xo, n

    with torch.no_grad():
        _, k, v = qkv(past.to(gpu), torch.arange(L, device=gpu))
        append_kv(k, v, prefix)
        if captured:
            x = xs[0].to(gpu)
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                step(x)
            torch.cuda.current_stream().wait_stream(side)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = step(x)
            cache.lengths.zero_()
            cache.seen.fill_(L)
            got = []
            for new in xs:
                x.copy_(new)
                graph.replay()
                got.append([t.clone() for t in out])
        else:
            got = [step(x.to(gpu)) for x in xs]
    torch.cuda.synchronize()
    assert cache.lengths.tolist() == [steps] * B and cache.seen.tolist() == [L + steps] * B
    bound = 16 * 2.0 ** -8
    for b in range(B):
        rx, rn = reference(b)
        for i, (xo, n) in enumerate(got):
            assert _rel(xo[b, 0], rx[0, i]) <= bound and _rel(n[b, 0], rn[0, i]) <= bound, (b, i)
