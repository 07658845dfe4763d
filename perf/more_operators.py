"""Calls of the operators around a block's attention, as plain data with a way to run each in two forms.

Three kinds of call, told apart by a case's ``op``:

    "norm"    gate, residual and the next norm in one pass: x' = x + gate y (y first normed where there is a norm after
              the block), n = norm(x') scaled and shifted; forward, with tangents, or trained through
    "rotary"  positions turned into rotations of queries and keys: pairs of neighbours or of halves, part of the head,
              frequencies scaled for long contexts; forward, with tangents, or trained through
    "prefix"  attention of new tokens of many sequences that share a long prefix, and of their own caches

``own`` says which form ``run`` takes: elementary torch operations in 32 bits, or this package's entry points.

    listed()            the named cases
    draw(rng)           one more case of the ranges they stand for
    prepare(case, seed) inputs on the GPU
    run(state)          one pass; returns its outputs whole
    work(case)          bytes and flops a pass cannot do without
    exact(case, seed)   the outputs in float64 from the definitions

Sizes are those of the Wan2.1 students (1536 and 5120 channels, 12 and 40 heads of 128, 1560 tokens per latent frame at
480p, 21 frames and 32760 tokens per clip), of this repository's tests (999 tokens, 64-wide heads, two fp32 heads of 256
tokens), and generic ones for shared key heads (32 or 64 query heads over 8 key heads).
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
TANGENT_STD = 0.1
EPS = 1e-6


def listed():
    return [
        # The plumbing configuration's width, forward and backward: launches and latency alone.
        dict(name="norm_train_plumbing_fp32", op="norm", B=1, S=256, C=128, dtype="fp32", mods="fp32", mode="train",
             kind="layer", branch=True, gate=True, mod=True, F=1, affine=False, post=False),
        # One decoding step of 32 sequences at 14B's width, each with its own modulation.
        dict(name="norm_token_14b", op="norm", B=32, S=1, C=5120, dtype="bf16", mods="bf16", mode="plain", kind="layer",
             branch=True, gate=True, mod=True, F=1, affine=False, post=False),
        # Training with norms before and after each block (weights, no modulation), odd lengths in half precision.
        dict(name="norm_train_sandwich_fp16", op="norm", B=3, S=999, C=1536, dtype="fp16", mods="fp32", mode="train",
             kind="rms", branch=True, gate=False, mod=False, F=1, affine=True, post=True),
        # One 1.3B block boundary over a 480p clip, forward and backward, modulated for each latent frame.
        dict(name="norm_train_clip_1p3b", op="norm", B=1, S=32760, C=1536, dtype="bf16", mods="fp32", mode="train",
             kind="layer", branch=True, gate=True, mod=True, F=21, affine=False, post=False),
        # One 14B block boundary over a 480p clip with tangents, of the modulation too: a tangent evaluation's forward.
        dict(name="norm_jvp_clip_14b", op="norm", B=1, S=32760, C=5120, dtype="bf16", mods="fp32", mode="jvp",
             kind="layer", branch=True, gate=True, mod=True, F=1, affine=False, post=False),
        # One new token for each of 32 sequences at far positions, halves paired, frequencies stretched eightfold.
        dict(name="rotary_token", op="rotary", B=32, S=1, Hq=32, Hk=8, D=128, R=128, dtype="bf16", mode="plain",
             layout="half", scaling="yarn", first=1, last=131072),
        # Training a batch of odd-length sequences, half of each 64-wide head turned, in half precision.
        dict(name="rotary_train_part_fp16", op="rotary", B=3, S=999, Hq=32, Hk=8, D=64, R=32, dtype="fp16", mode="train",
             layout="half", scaling="none", first=0, last=0),
        # Queries and keys of one 14B self-attention over a 480p clip, with tangents.
        dict(name="rotary_jvp_clip_14b", op="rotary", B=1, S=32760, Hq=40, Hk=40, D=128, R=128, dtype="bf16", mode="jvp",
             layout="interleaved", scaling="linear", first=0, last=0),
        # Four short sequences behind a short prefix, in half precision: the call whose latency counts.
        dict(name="prefix_short_fp16", op="prefix", P=1, n=4, S=1, Hq=12, Hk=12, D=64, dtype="fp16", page=16, prefix=257,
             shortest=1, longest=64, causal=False),
        # Eight continuations of one 480p clip at 14B: few rows, the prefix's bytes count.
        dict(name="prefix_clip_14b", op="prefix", P=1, n=8, S=1, Hq=40, Hk=40, D=128, dtype="bf16", page=64, prefix=32760,
             shortest=1, longest=1560, causal=False),
        # Two prompts with 48 samples each, of very different lengths.
        dict(name="prefix_samples", op="prefix", P=2, n=48, S=1, Hq=32, Hk=8, D=128, dtype="bf16", page=16, prefix=16000,
             shortest=1, longest=4001, causal=False),
        # 48 sequences behind a very long prefix, four new tokens each (a draft checked in one step): the arithmetic counts.
        dict(name="prefix_draft_long", op="prefix", P=1, n=48, S=4, Hq=64, Hk=8, D=128, dtype="bf16", page=64,
             prefix=131072, shortest=4, longest=2000, causal=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


# A drawn case moves and computes at most this much (the largest listed ones: 2.7e9 bytes, 8.3e11 flops).
MAX_BYTES = 2.7e9
MAX_FLOPS = 8.0e11


def draw(rng):
    while True:
        case = _draw_any(rng)
        w = work(case)
        if w["bytes"] <= MAX_BYTES and w["flops"] <= MAX_FLOPS:
            return case


def _draw_any(rng):
    op = rng.choice(["norm", "norm", "rotary", "rotary", "prefix", "prefix"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp16"])
    if op == "norm":
        dtype = rng.choice([dtype, dtype, dtype, "fp32"])
        C = rng.choice([1536, 1536, 5120, 5120, 8 * _log_int(rng, 8, 1024)])
        B = rng.choice([1, 1, 2, 3, 32])
        F = rng.choice([1, 1, 1, 3, 21])
        S = F * max(1, _log_int(rng, 1, 32760) // F)
        case = dict(op=op, B=B, S=S, C=C, dtype=dtype, mods=rng.choice([dtype, "fp32"]),
                    mode=rng.choice(["train", "train", "jvp", "plain"]), kind=rng.choice(["layer", "layer", "rms"]),
                    branch=rng.random() < 0.8, gate=False, mod=rng.random() < 0.7, F=F, affine=False, post=False)
        case["gate"] = case["branch"] and rng.random() < 0.7
        case["affine"] = not case["mod"] or rng.random() < 0.2
        case["post"] = case["branch"] and case["kind"] == "rms" and rng.random() < 0.5
        if not (case["gate"] or case["mod"]):
            case["F"] = 1
        return case
    D = rng.choice([128, 128, 128, 64, 64, 32, 256])
    Hk = rng.choice([1, 2, 4, 5, 8, 12, 40])
    group = rng.choice([1, 1, 2, 4, 5, 8]) if Hk <= 8 else 1
    if op == "rotary":
        D = rng.choice([D, D, D, 80, 96])
        R = rng.choice([D, D, D // 2, D // 4])
        S = _log_int(rng, 1, 32760)
        first = rng.choice([0, _log_int(rng, 1, 100000)])
        return dict(op=op, B=rng.choice([1, 1, 2, 3, 32]), S=S, Hq=Hk * group, Hk=Hk, D=D, R=R,
                    dtype=rng.choice([dtype, dtype, dtype, "fp32"]), mode=rng.choice(["train", "jvp", "plain"]),
                    layout=rng.choice(["half", "half", "interleaved"]), scaling=rng.choice(["none", "linear", "ntk", "yarn"]),
                    first=first, last=rng.choice([first, 2 * first]))
    S = rng.choice([1, 1, 1, 2, 4, 7])
    a, b = sorted((_log_int(rng, S, 4001), _log_int(rng, S, 4001)))
    return dict(op=op, P=rng.choice([1, 1, 1, 2, 3]), n=_log_int(rng, 1, 64), S=S, Hq=Hk * group, Hk=Hk, D=D, dtype=dtype,
                page=rng.choice([16, 16, 32, 48, 64, 128]), prefix=_log_int(rng, 17, 131072), shortest=a, longest=b,
                causal=rng.random() < 0.5)


# ---------------------------------------------------------------- sizes


def _lengths(case):
    """Slots of each sequence's own cache: from the shortest to the longest in equal ratios, in a fixed mixed order."""
    B, lo, hi = case["P"] * case["n"], case["shortest"], case["longest"]
    ratio = [lo * (hi / lo) ** (i / max(B - 1, 1)) for i in range(B)]
    ratio[-1] = hi if B > 1 else lo
    step = next(s for s in (7, 11, 13, 1) if math.gcd(s, B) == 1)
    return [int(round(ratio[(i * step) % B])) for i in range(B)]


def _prefixes(case):
    """Slots of each prefix: the case's, the further ones a little shorter."""
    return [max(1, case["prefix"] - 37 * i) for i in range(case["P"])]


def work(case):
    size = DTYPES[case["dtype"]].itemsize
    if case["op"] == "norm":
        rows, C = case["B"] * case["S"], case["C"]
        streams = {"plain": 1, "jvp": 2, "train": 2}[case["mode"]]  # values, and their tangents or gradients
        tensors = 4 if case["branch"] else 2
        small = case["B"] * case["F"] * C * DTYPES[case["mods"]].itemsize * (case["gate"] + 2 * case["mod"]) * streams
        return {"bytes": streams * tensors * rows * C * size + small, "flops": streams * 16 * rows * C}
    if case["op"] == "rotary":
        elems = case["B"] * case["S"] * (case["Hq"] + case["Hk"]) * case["D"]
        streams = 1 if case["mode"] == "plain" else 2
        return {"bytes": streams * 2 * elems * size + 8 * case["B"] * case["S"], "flops": streams * 3 * elems}
    rows, Hk, D = case["S"] * case["Hq"], case["Hk"], case["D"]
    shared, lengths = _prefixes(case), _lengths(case)
    slots = sum(shared) + sum(lengths)
    q = 2 * case["P"] * case["n"] * rows * D * size + 4 * case["P"] * case["n"] * rows
    pairs = rows * (case["n"] * sum(shared) + sum(lengths))
    return {"bytes": 2 * slots * Hk * D * size + q + 4 * slots // case["page"], "flops": 4 * D * pairs}


# ---------------------------------------------------------------- inputs


def _norm_inputs(case, draw_, g):
    B, S, C, F = case["B"], case["S"], case["C"], case["F"]
    mods = DTYPES[case["mods"]]
    # a residual stream: channels of different size and an offset of their own, a few of them large
    scale = torch.rand(C, generator=g, device="cuda") + 0.5
    scale[torch.randint(0, C, (max(1, C // 256),), generator=g, device="cuda")] *= 8.0
    offset = torch.randn(C, generator=g, device="cuda") * 0.3
    x = {"x": draw_(B, S, C, by=scale, plus=offset)}
    if case["branch"]:
        x["y"] = draw_(B, S, C, by=0.7)
    for n, there, mean in (("gate", case["gate"], 0.5), ("scale", case["mod"], 0.0), ("shift", case["mod"], 0.0)):
        if there:
            x[n] = (mean + 0.3 * torch.randn(B, F, C, generator=g, device="cuda")).to(mods)
    if case["affine"]:
        x["weight"] = (1 + 0.2 * torch.randn(C, generator=g, device="cuda")).to(mods)
        if case["kind"] == "layer":
            x["bias"] = (0.1 * torch.randn(C, generator=g, device="cuda")).to(mods)
    if case["post"]:
        x["post_weight"] = (1 + 0.2 * torch.randn(C, generator=g, device="cuda")).to(mods)
    if case["mode"] == "jvp":
        for n in ("x", "y", "gate", "scale", "shift"):
            if n in x:
                x["t" + n] = (torch.randn(x[n].shape, generator=g, device="cuda") * TANGENT_STD).to(x[n].dtype)
    if case["mode"] == "train":
        if case["branch"]:
            x["gx"] = draw_(B, S, C)
        x["gn"] = draw_(B, S, C)
    return x


# Where a prefix of the trained length ends and stretched frequencies begin to matter.
TRAINED = 16384
FACTOR = 8.0


def _rotary_inputs(case, draw_, g):
    B, S, D = case["B"], case["S"], case["D"]
    scale = torch.rand(D, generator=g, device="cuda") + 0.5
    x = {"q": draw_(B, S, case["Hq"], D, by=scale), "k": draw_(B, S, case["Hk"], D, by=scale)}
    lo, hi = case["first"], case["last"]
    start = torch.tensor([round(lo + (hi - lo) * i / max(B - 1, 1)) for i in range(B)], device="cuda", dtype=torch.int64)
    x["positions"] = (start[:, None] + torch.arange(S, device="cuda")).to(torch.int32)
    for n in ("q", "k"):
        if case["mode"] == "jvp":
            x["t" + n] = draw_(*x[n].shape, by=TANGENT_STD)
        if case["mode"] == "train":
            x["g" + n] = draw_(*x[n].shape)
    x["frequencies"], x["factor"] = _frequencies(case)
    return x


def _frequencies(case):
    """(radians per position [R/2] float64, what sines and cosines are multiplied by)."""
    R, i = case["R"], torch.arange(case["R"] // 2, device="cuda", dtype=torch.float64)
    plain = 10000.0 ** (-2 * i / R)
    if case["scaling"] == "linear":
        return plain / FACTOR, 1.0
    if case["scaling"] == "ntk":
        return (10000.0 * FACTOR ** (R / (R - 2))) ** (-2 * i / R), 1.0
    if case["scaling"] == "yarn":  # full turns over the trained length: from 32 on as they are, up to 1 stretched
        keep = ((TRAINED * plain / (2 * math.pi) - 1) / 31).clamp(0, 1)
        return plain * (keep + (1 - keep) / FACTOR), 0.1 * math.log(FACTOR) + 1
    return plain, 1.0


def _prefix_inputs(case, draw_, g):
    P, n, Hk, D, page = case["P"], case["n"], case["Hk"], case["D"], case["page"]
    B, shared, lengths = P * n, _prefixes(case), _lengths(case)
    Mp, M = -(-max(shared) // page), -(-max(lengths) // page)
    N = P * Mp + B * M + 1
    at = torch.randperm(N, generator=g, device="cuda").to(torch.int32)
    x = {"k_pages": draw_(N, Hk, page, D, by=1.5), "v_pages": draw_(N, Hk, page, D),
         "prefix_table": at[:P * Mp].view(P, Mp).contiguous(), "page_table": at[P * Mp:P * Mp + B * M].view(B, M).contiguous(),
         "prefix_lengths": torch.tensor(shared, device="cuda", dtype=torch.int32),
         "lengths": torch.tensor(lengths, device="cuda", dtype=torch.int32)}
    x["prefix_seen"], x["seen"] = x["prefix_lengths"].clone(), x["lengths"].clone()
    x["q"] = draw_(B, case["S"], case["Hq"], D, by=1.5)
    return x


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def draw_(*shape, by=1.0, plus=None):
        t = torch.randn(shape, generator=g, device="cuda").mul_(by)
        return (t if plus is None else t.add_(plus)).to(dtype)

    return {"norm": _norm_inputs, "rotary": _rotary_inputs, "prefix": _prefix_inputs}[case["op"]](case, draw_, g)


LEAVES = ("x", "y", "gate", "scale", "shift", "weight", "bias", "post_weight")


def prepare(case, seed):
    x = _inputs(case, seed)
    x["case"] = case
    if case.get("mode") == "train":
        for n in LEAVES if case["op"] == "norm" else ("q", "k"):
            if n in x:
                x[n].requires_grad_(True)
    if own and case["op"] == "prefix":
        from dmad_amd import PagedKVCache

        x["shared"] = PagedKVCache(x["k_pages"], x["v_pages"], x["prefix_table"], x["prefix_lengths"], x["prefix_seen"])
        x["cache"] = PagedKVCache(x["k_pages"], x["v_pages"], x["page_table"], x["lengths"], x["seen"])
    return x


# ---------------------------------------------------------------- one pass


def run(x):
    case = x["case"]
    if case["op"] == "norm":
        return _own_norm(case, x) if own else _plain_norm(case, x)
    if case["op"] == "rotary":
        return _own_rotary(case, x) if own else _plain_rotary(case, x)
    return _own_prefix(case, x) if own else _plain_prefix(case, x)


def _own_norm(case, x):
    from dmad_amd import gated_residual_norm_with_tangent

    def call():
        return gated_residual_norm_with_tangent(
            *((x.get(n), x.get("t" + n)) for n in ("x", "y", "gate", "scale", "shift")), weight=x.get("weight"),
            bias=x.get("bias"), post_weight=x.get("post_weight"), eps=EPS, norm=case["kind"])

    if case["mode"] != "train":
        with torch.no_grad():
            (r, tr), (n, tn) = call()
        return [t for t in ((r, tr) if case["branch"] else ()) + (n, tn) if t is not None]
    (r, _), (n, _) = call()
    outs, into = ((r, n), (x["gx"], x["gn"])) if case["branch"] else ((n,), (x["gn"],))
    grads = torch.autograd.grad(outs, [x[k] for k in LEAVES if k in x], into)
    return [t.detach() for t in outs] + list(grads)


def _unit(x, kind):
    """x normed, and the reciprocal root that did it."""
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    r = torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + EPS)
    return x * r, r


def _unit_back(a, n, r, kind):
    """The transposed derivative of the norm, on a; by symmetry its derivative too."""
    a = a - n * (a * n).mean(-1, keepdim=True)
    if kind == "layer":
        a = a - a.mean(-1, keepdim=True)
    return a * r


def _plain_norm(case, x):
    kind, dtype = case["kind"], x["x"].dtype
    B, S, C = x["x"].shape
    with torch.no_grad():
        f = {n: t.float() for n, t in x.items() if torch.is_tensor(t)}
        for n in ("gate", "scale", "shift", "tgate", "tscale", "tshift"):  # a row for every token
            if n in f:
                f[n] = f[n].repeat_interleave(S // case["F"], dim=1)
        s = f["x"]
        if case["branch"]:
            y = f["y"]
            if case["post"]:
                yn, yr = _unit(y, "rms")
                y = yn * f["post_weight"]
            s = s + (f["gate"] * y if case["gate"] else y)
        n, r = _unit(s, kind)
        by = f["weight"] if case["affine"] else torch.ones((), device=s.device)
        plus = f["bias"] if "bias" in f else torch.zeros((), device=s.device)
        gain = by * (1 + f["scale"]) if case["mod"] else by
        out = n * gain + (plus * (1 + f["scale"]) + f["shift"] if case["mod"] else plus)
        outs = ([s.to(dtype)] if case["branch"] else []) + [out.to(dtype)]
        if case["mode"] == "plain":
            return outs
        if case["mode"] == "jvp":
            t = f["tx"]
            if case["branch"]:
                ty = _unit_back(f["ty"], yn, yr, "rms") * f["post_weight"] if case["post"] else f["ty"]
                t = t + (f["tgate"] * y + f["gate"] * ty if case["gate"] else ty)
            to = _unit_back(t, n, r, kind) * gain
            if case["mod"]:
                to = to + (n * by + plus) * f["tscale"] + f["tshift"]
            return [outs[0], t.to(dtype), outs[1], to.to(dtype)] if case["branch"] else [outs[0], to.to(dtype)]
        gn = f["gn"]
        ds = _unit_back(gn * gain, n, r, kind)
        if case["branch"]:
            ds = ds + f["gx"]
        per = lambda z: z.view(B, case["F"], -1, C).sum(2, dtype=torch.float64)  # noqa: E731
        all_ = lambda z: z.sum((0, 1), dtype=torch.float64)  # noqa: E731
        grads = {"x": ds}
        if case["branch"]:
            dy = ds * f["gate"] if case["gate"] else ds
            if case["gate"]:
                grads["gate"] = per(ds * y)
            if case["post"]:
                grads["post_weight"] = all_(dy * yn)
                dy = _unit_back(dy * f["post_weight"], yn, yr, "rms")
            grads["y"] = dy
        if case["mod"]:
            grads["scale"], grads["shift"] = per(gn * (n * by + plus)), per(gn)
        if case["affine"]:
            one = gn * (1 + f["scale"]) if case["mod"] else gn
            grads["weight"], grads["bias"] = all_(one * n), all_(one)
        return outs + [grads[k].to(x[k].dtype) for k in LEAVES if k in x]


def _own_rotary(case, x):
    from dmad_amd import qk_rotary_with_tangent

    def call():
        return qk_rotary_with_tangent((x["q"], x.get("tq")), (x["k"], x.get("tk")), x["positions"], x["frequencies"],
                                      layout=case["layout"], factor=x["factor"])

    if case["mode"] != "train":
        with torch.no_grad():
            (q, tq), (k, tk) = call()
        return [t for t in (q, tq, k, tk) if t is not None]
    (q, _), (k, _) = call()
    return [q.detach(), k.detach(), *torch.autograd.grad((q, k), (x["q"], x["k"]), (x["gq"], x["gk"]))]


def _plain_turn(x, cos, sin, layout):
    R = 2 * cos.shape[-1]
    xf, rest = x[..., :R].float(), x[..., R:]
    a, b = (xf[..., 0::2], xf[..., 1::2]) if layout == "interleaved" else (xf[..., :R // 2], xf[..., R // 2:])
    u, v = a * cos - b * sin, b * cos + a * sin
    y = torch.stack((u, v), dim=-1).flatten(-2) if layout == "interleaved" else torch.cat((u, v), dim=-1)
    return torch.cat((y.to(x.dtype), rest), dim=-1)


def _plain_rotary(case, x):
    with torch.no_grad():
        angle = (x["positions"].double()[..., None] * x["frequencies"])[:, :, None]
        cos, sin = (torch.cos(angle) * x["factor"]).float(), (torch.sin(angle) * x["factor"]).float()
        if case["mode"] == "jvp":
            return [_plain_turn(x[n], cos, sin, case["layout"]) for n in ("q", "tq", "k", "tk")]
        outs = [_plain_turn(x[n], cos, sin, case["layout"]) for n in ("q", "k")]
        if case["mode"] == "train":
            outs += [_plain_turn(x[n], cos, -sin, case["layout"]) for n in ("gq", "gk")]
        return outs


def _own_prefix(case, x):
    from dmad_amd import shared_prefix_attention

    return shared_prefix_attention(x["q"], x["shared"], x["cache"], causal=case["causal"], return_lse=True)


def _plain_prefix(case, x):
    q, n = x["q"], case["n"]
    B, S, Hq, D = q.shape
    Hk, page = case["Hk"], case["page"]
    P, G = case["P"], Hq // case["Hk"]

    def flat(table):
        return (x[name][table.long()].transpose(1, 2).reshape(table.shape[0], Hk, -1, D).float() for name in ("k_pages", "v_pages"))

    qf = q.float().view(P, n, S, Hk, G, D) * D ** -0.5
    # scores over the prefix, rows of all its sequences together, and over each sequence's own slots
    kp, vp = flat(x["prefix_table"])
    sp = (qf.permute(0, 3, 1, 2, 4, 5).reshape(P, Hk, -1, D) @ kp.transpose(2, 3).contiguous())
    sp.masked_fill_((torch.arange(kp.shape[2], device="cuda") >= x["prefix_lengths"][:, None])[:, None, None], -math.inf)
    ko, vo = flat(x["page_table"])
    so = (qf.view(B, S, Hk, G, D).transpose(1, 2).reshape(B, Hk, -1, D) @ ko.transpose(2, 3).contiguous()).view(B, Hk, S, G, -1)
    seen = x["lengths"][:, None].expand(B, S).long()
    if case["causal"]:
        seen = seen - (S - 1) + torch.arange(S, device="cuda")
    so.masked_fill_((torch.arange(ko.shape[2], device="cuda") >= seen[..., None])[:, None, :, None], -math.inf)
    # one softmax over both
    sp = sp.view(P, Hk, n, S * G, -1)
    so = so.view(P, n, Hk, S * G, -1).transpose(1, 2)
    top = torch.maximum(sp.amax(-1, keepdim=True), so.amax(-1, keepdim=True))
    sp, so = sp.sub_(top).exp_(), torch.exp(so - top)
    total = sp.sum(-1, keepdim=True) + so.sum(-1, keepdim=True)
    o = (sp.view(P, Hk, n * S * G, -1) @ vp).view(P, Hk, n, S * G, D)
    o = o + (so.transpose(1, 2).reshape(B, Hk, S * G, -1) @ vo).view(P, n, Hk, S * G, D).transpose(1, 2)
    o = (o / total).view(P, Hk, n, S, G, D).permute(0, 2, 3, 1, 4, 5).reshape(B, S, Hq, D).to(q.dtype)
    lse = (top + torch.log(total)).view(P, Hk, n, S, G).permute(0, 2, 1, 4, 3).reshape(B, Hq, S)
    return o, lse


# ---------------------------------------------------------------- float64 references


def _exact_norm(case, x):
    names = [n for n in LEAVES if n in x]
    group = torch.arange(case["S"], device="cuda") // (case["S"] // case["F"])

    def outs(*ts):
        v = dict(zip(names, ts))
        s = v["x"]
        if case["branch"]:
            y = v["y"]
            if case["post"]:
                y = y / ((y * y).sum(-1, keepdim=True) / case["C"] + EPS).sqrt() * v["post_weight"]
            s = s + (y * v["gate"][:, group] if case["gate"] else y)
        z = s - s.mean(-1, keepdim=True) if case["kind"] == "layer" else s
        z = z / ((z * z).sum(-1, keepdim=True) / case["C"] + EPS).sqrt()
        if case["affine"]:
            z = z * v["weight"]
            if "bias" in v:
                z = z + v["bias"]
        if case["mod"]:
            z = z * (1 + v["scale"][:, group]) + v["shift"][:, group]
        return (s, z) if case["branch"] else (z,)

    values = [x[n].double() for n in names]
    if case["mode"] == "plain":
        return list(outs(*values))
    if case["mode"] == "jvp":
        along = [x["t" + n].double() if "t" + n in x else torch.zeros_like(v) for n, v in zip(names, values)]
        primal, tangent = torch.func.jvp(outs, tuple(values), tuple(along))
        return [t for pair in zip(primal, tangent) for t in pair]
    for v in values:
        v.requires_grad_(True)
    with torch.enable_grad():
        y = outs(*values)
        grads = torch.autograd.grad(y, values, [x[n].double() for n in (("gx", "gn") if case["branch"] else ("gn",))])
    return [t.detach() for t in y] + list(grads)


def _exact_turn(z, turn, layout):
    """Pairs as complex numbers, times `turn`."""
    R = 2 * turn.shape[-1]
    z = z.double()
    pairs = z[..., :R].unflatten(-1, (R // 2, 2) if layout == "interleaved" else (2, R // 2))
    if layout == "half":
        pairs = pairs.transpose(-1, -2)
    y = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
    if layout == "half":
        y = y.transpose(-1, -2)
    return torch.cat((y.flatten(-2), z[..., R:]), dim=-1)


def _exact_rotary(case, x):
    angle = x["positions"].double()[:, :, None, None] * x["frequencies"]
    turn = torch.polar(torch.full_like(angle, x["factor"]), angle)
    names = {"plain": ("q", "k"), "jvp": ("q", "tq", "k", "tk"), "train": ("q", "k", "gq", "gk")}[case["mode"]]
    return [_exact_turn(x[n], turn.conj() if n.startswith("g") else turn, case["layout"]) for n in names]


def _exact_prefix(case, x):
    B, S, Hq, D = x["q"].shape
    n, G = case["n"], Hq // case["Hk"]
    o = torch.empty(B, S, Hq, D, dtype=torch.float64, device="cuda")
    lse = torch.empty(B, Hq, S, dtype=torch.float64, device="cuda")
    shared, lengths = _prefixes(case), _lengths(case)

    def rows(table, head, count):
        used = table[:-(-count // case["page"])].long()
        return (x[name][used, head].reshape(-1, D)[:count].double() for name in ("k_pages", "v_pages"))

    for p in range(case["P"]):
        for h in range(case["Hk"]):
            heads = slice(h * G, (h + 1) * G)
            k, v = rows(x["prefix_table"][p], h, shared[p])
            q = x["q"][p * n:(p + 1) * n, :, heads].double() / math.sqrt(D)
            s = q.reshape(-1, D) @ k.t().contiguous()
            first = torch.logsumexp(s, dim=-1)
            behind = (torch.exp(s.sub_(first[:, None])) @ v).view(n, S * G, D)
            first = first.view(n, S * G)
            for i in range(n):
                b = p * n + i
                k, v = rows(x["page_table"][b], h, lengths[b])
                t = q[i].reshape(-1, D) @ k.t().contiguous()
                if case["causal"]:
                    last = torch.arange(S, device="cuda").repeat_interleave(G)[:, None] + (lengths[b] - S)
                    t = t.masked_fill(torch.arange(lengths[b], device="cuda") > last, -math.inf)
                both = torch.logaddexp(first[i], torch.logsumexp(t, dim=-1))
                y = torch.exp(first[i] - both)[:, None] * behind[i] + torch.exp(t - both[:, None]) @ v
                o[b, :, heads], lse[b, heads] = y.view(S, G, D), both.view(S, G).t()
    return o, lse


def exact(case, seed):
    with torch.no_grad():
        x = _inputs(case, seed)
        return {"norm": _exact_norm, "rotary": _exact_rotary, "prefix": _exact_prefix}[case["op"]](case, x)
