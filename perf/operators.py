"""Calls of the streaming operators, as plain data with a way to run each in two forms.

Four kinds of call, told apart by a case's ``op``:

    "norm"    RMSNorm of queries and keys for each head and their rotation in one pass; with tangents (forward only)
              or trained through (outputs and gradients of inputs and weights)
    "append"  the same for new tokens, whose keys and values go into the pages of a cache
    "attend"  attention of one or a few new tokens over the cache, with or without each slot's share added up
    "evict"   the cache cut to its heaviest slots

``own`` says which form ``run`` takes: elementary torch operations in 32 bits, or this package's entry points.

    listed()            the named cases
    draw(rng)           one more case of the ranges they stand for
    prepare(case, seed) inputs on the GPU
    run(state)          one pass; returns its outputs whole
    work(case)          bytes and flops a pass cannot do without
    exact(case, seed)   the outputs in float64 from the definitions

Sizes are those of the Wan2.1 students (128-wide heads, 12 of them at 1.3B and 40 at 14B, 1560 tokens per latent frame
at 480p, 32760 per clip), of this repository's tests (999 tokens, 64-wide heads, two fp32 heads of 256 tokens), and
generic ones for shared key heads (32 or 64 query heads over 8 key heads).
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
TANGENT_STD = 0.1
EPS = 1e-6


def listed():
    return [
        # The plumbing configuration, forward and backward: launches and latency alone.
        dict(name="norm_train_plumbing_fp32", op="norm", B=1, S=256, Hq=2, Hk=2, D=64, dtype="fp32", mode="train"),
        # Training a batch of odd-length sequences with shared key heads in half precision.
        dict(name="norm_train_shared_fp16", op="norm", B=3, S=999, Hq=32, Hk=8, D=64, dtype="fp16", mode="train"),
        # Inputs of one 1.3B self-attention over a 480p clip, forward and backward.
        dict(name="norm_train_clip_1p3b", op="norm", B=1, S=32760, Hq=12, Hk=12, D=128, dtype="bf16", mode="train"),
        # Inputs of one 14B self-attention over a 480p clip, with tangents: a tangent evaluation's forward.
        dict(name="norm_jvp_clip_14b", op="norm", B=1, S=32760, Hq=40, Hk=40, D=128, dtype="bf16", mode="jvp"),
        # One new token for each of 32 sequences on their way into the cache: what every decoding step does.
        dict(name="append_token", op="append", B=32, S=1, Hq=32, Hk=8, D=128, dtype="bf16", page=16, shortest=17,
             longest=4001),
        # One 480p latent frame of the 14B student on its way into the cache.
        dict(name="append_frame_14b", op="append", B=1, S=1560, Hq=40, Hk=40, D=128, dtype="bf16", page=64,
             shortest=3120, longest=3120),
        # One token against a short history of one sequence, in half precision: the call whose latency counts.
        dict(name="attend_short_fp16", op="attend", B=1, S=1, Hq=12, Hk=12, D=64, dtype="fp16", page=16, shortest=257,
             longest=257, causal=False, weights=False),
        # One token of the 14B student against a whole 480p clip: a single sequence, split over its length.
        dict(name="attend_clip_14b", op="attend", B=1, S=1, Hq=40, Hk=40, D=128, dtype="bf16", page=64, shortest=32760,
             longest=32760, causal=False, weights=False),
        # One token for each of 48 sequences of very different lengths, whose slots' shares are added up for eviction.
        dict(name="attend_ragged_weights", op="attend", B=48, S=1, Hq=32, Hk=8, D=128, dtype="bf16", page=16,
             shortest=1, longest=16000, causal=False, weights=True),
        # Four new tokens at once (a draft checked in one step) for 16 long sequences: the pool passes 32-bit offsets.
        dict(name="attend_draft_long", op="attend", B=16, S=4, Hq=64, Hk=8, D=128, dtype="bf16", page=64,
             shortest=120001, longest=131072, causal=True, weights=False),
        # A short cache cut by a few slots: eviction at nearly every step.
        dict(name="evict_few_fp16", op="evict", B=2, Hk=12, D=64, dtype="fp16", page=16, shortest=270, longest=273,
             keep=256, recent=32, sink=4),
        # Long caches of several sequences cut to half: eviction once in a while.
        dict(name="evict_half", op="evict", B=8, Hk=8, D=128, dtype="bf16", page=64, shortest=20001, longest=32760,
             keep=16384, recent=1024, sink=4),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


# A drawn case moves at most MAX_BYTES and has a pool of at most MAX_POOL (the largest listed one: 8.2e9, 8.6e9).
MAX_BYTES = 8.0e9
MAX_POOL = 8.6e9


def draw(rng):
    while True:
        case = _draw_any(rng)
        if work(case)["bytes"] <= MAX_BYTES and _pool_bytes(case) <= MAX_POOL:
            return case


def _draw_any(rng):
    op = rng.choice(["norm", "norm", "append", "attend", "attend", "attend", "evict"])
    D = rng.choice([128, 128, 128, 64, 64, 32, 256])
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp16"])
    Hk = rng.choice([1, 2, 4, 5, 8, 12, 40])
    group = rng.choice([1, 1, 2, 4, 5, 8]) if Hk <= 8 else 1
    if op == "norm":
        return dict(op=op, B=rng.choice([1, 1, 2, 3]), S=_log_int(rng, 1, 32760), Hq=Hk * group, Hk=Hk, D=D,
                    dtype=rng.choice([dtype, dtype, dtype, "fp32"]), mode=rng.choice(["train", "train", "jvp"]))
    page = rng.choice([16, 16, 32, 48, 64, 128])
    if op == "append":
        long = rng.random() < 0.3
        B, S = (rng.choice([1, 2]), _log_int(rng, 16, 6240)) if long else (_log_int(rng, 1, 128), rng.choice([1, 1, 2, 5]))
        a, b = sorted((_log_int(rng, 1, 8000), _log_int(rng, 1, 8000)))
        return dict(op=op, B=B, S=S, Hq=Hk * group, Hk=Hk, D=D, dtype=dtype, page=page, shortest=a, longest=b)
    if op == "attend":
        B = _log_int(rng, 1, 64)
        top = 131072 if B * Hk * D <= 16384 else 16000
        S = rng.choice([1, 1, 1, 2, 4, 7])
        a, b = sorted((_log_int(rng, S, top), _log_int(rng, S, top)))
        return dict(op=op, B=B, S=S, Hq=Hk * group, Hk=Hk, D=D, dtype=dtype, page=page, shortest=a, longest=b,
                    causal=rng.random() < 0.5, weights=rng.random() < 0.4)
    B = _log_int(rng, 1, 16)
    b = _log_int(rng, 64, 32760)
    a = rng.randint(max(1, b // 2), b)
    keep = max(1, int(b * rng.uniform(0.3, 0.98)))
    recent = rng.choice([0, keep // 16, keep // 4])
    return dict(op=op, B=B, Hk=Hk, D=D, dtype=dtype, page=page, shortest=a, longest=b, keep=keep, recent=recent,
                sink=min(rng.choice([0, 1, 4]), keep - recent))


# ---------------------------------------------------------------- sizes


def _lengths(case):
    """Slots in use per sequence: from the shortest to the longest in equal ratios, dealt in a fixed mixed order."""
    B, lo, hi = case["B"], case["shortest"], case["longest"]
    ratio = [lo * (hi / lo) ** (i / max(B - 1, 1)) for i in range(B)]
    ratio[-1] = hi if B > 1 else lo
    step = next(s for s in (7, 11, 13, 1) if math.gcd(s, B) == 1)
    return [int(round(ratio[(i * step) % B])) for i in range(B)]


def _pages_per_sequence(case):
    room = case["longest"] + (case["S"] if case["op"] == "append" else 0)
    return -(-room // case["page"])


def _pool_bytes(case):
    if case["op"] == "norm":
        return 0
    slots = case["B"] * _pages_per_sequence(case) * case["page"]
    return 2 * slots * case["Hk"] * case["D"] * DTYPES[case["dtype"]].itemsize


def work(case):
    size, D, Hk = DTYPES[case["dtype"]].itemsize, case["D"], case["Hk"]
    if case["op"] == "norm":
        elems = case["B"] * case["S"] * (case["Hq"] + Hk) * D
        angles = case["S"] * D // 2 * 4
        if case["mode"] == "jvp":  # primal and tangent, in and out
            return {"bytes": 4 * elems * size + angles, "flops": 24 * elems}
        # inputs and the outputs' gradients in, outputs and the inputs' gradients out
        return {"bytes": 4 * elems * size + angles, "flops": 30 * elems}
    if case["op"] == "append":
        new = case["B"] * case["S"]
        elems = new * (case["Hq"] + 2 * Hk) * D
        return {"bytes": 2 * elems * size + new * D // 2 * 4 + new * Hk * 8 + 16 * case["B"],
                "flops": 12 * new * (case["Hq"] + Hk) * D}
    if case["op"] == "attend":
        rows, slots = case["S"] * case["Hq"], sum(_lengths(case))
        cache = 2 * slots * Hk * D * size + (8 * slots * Hk if case["weights"] else 0)
        return {"bytes": cache + 2 * case["B"] * rows * D * size + 4 * case["B"] * rows + 4 * slots // case["page"],
                "flops": 4 * rows * D * slots + (rows * slots if case["weights"] else 0)}
    total, flops = 0, 0
    keep, recent = case["keep"], case["recent"]
    for n in _lengths(case):
        if n <= keep:
            continue
        old = n - recent  # the heaviest of the old slots stay wherever they are; the rest of the tail moves
        moved = min(recent, n - keep) + max(0, n - keep - recent) * (keep - recent) / max(old, 1)
        total += Hk * (8 * n + 2 * moved * (2 * D * size + 8))
        flops += Hk * n
    return {"bytes": int(total) + 8 * case["B"], "flops": flops}


# ---------------------------------------------------------------- inputs


def _norm_inputs(case, draw_, g):
    Hq, Hk, D = case["Hq"], case["Hk"], case["D"]
    # Linear outputs: channels of different size, as trained projections give
    scale = torch.rand(D, generator=g, device="cuda") + 0.5
    x = {"q": draw_(case["B"], case["S"], Hq, D, by=scale), "k": draw_(case["B"], case["S"], Hk, D, by=scale)}
    for n in ("q", "k"):
        x["w" + n] = (1 + 0.2 * torch.randn(D, generator=g, device="cuda")).to(DTYPES[case["dtype"]])
    return x


def _angles(rows, D):
    """[rows, D/2] rotation angles of consecutive positions (theta 10000)."""
    i = torch.arange(D // 2, device="cuda", dtype=torch.float64)
    t = torch.arange(rows, device="cuda", dtype=torch.float64)
    return (t[:, None] * 10000.0 ** (-i / (D // 2))).float()


def _pool(case, draw_, g):
    """Pages of a cache in mixed order, each sequence's in its row of the table, and what its slots hold."""
    B, Hk, D, P = case["B"], case["Hk"], case["D"], case["page"]
    M = _pages_per_sequence(case)
    N = B * M + 1
    lengths = torch.tensor(_lengths(case), device="cuda", dtype=torch.int32)
    x = {"k_pages": draw_(N, Hk, P, D, by=1.5), "v_pages": draw_(N, Hk, P, D),
         "page_table": torch.randperm(N, generator=g, device="cuda")[:B * M].view(B, M).to(torch.int32)}
    # a sequence has seen more tokens than it holds once some were evicted
    extra = torch.randint(0, 50, (B,), generator=g, device="cuda", dtype=torch.int32)
    x["counts0"] = torch.stack([lengths, lengths + extra])
    x["counts"] = x["counts0"].clone()
    # attention weight so far: a few heavy slots, many light ones, some never looked at
    w = torch.rand(N, Hk, P, generator=g, device="cuda")
    x["weight0"] = torch.where(w < 0.05, torch.zeros_like(w), w ** 6 * 8)
    x["weight"] = x["weight0"].clone()
    slot = torch.zeros(N, P, device="cuda", dtype=torch.int32)
    slot[x["page_table"].view(-1).long()] = torch.arange(M * P, device="cuda", dtype=torch.int32).view(M, P).repeat(B, 1)
    x["position0"] = slot[:, None].expand(N, Hk, P).contiguous()
    if case["op"] == "evict":  # holes of an earlier eviction filled from the tail: positions follow no order
        far = torch.zeros(N, device="cuda", dtype=torch.int32)
        far[x["page_table"].view(-1).long()] = extra.repeat_interleave(M)
        mixed = (slot % 5 == 3) & (slot > 4)
        x["position0"] = (slot + torch.where(mixed, far[:, None], torch.zeros_like(slot)))[:, None].expand(N, Hk, P).contiguous()
    x["position"] = x["position0"].clone()
    return x


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def draw_(*shape, by=1.0):
        return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32 if math.prod(shape) < 1 << 28 else dtype
                           ).mul_(by).to(dtype)

    if case["op"] == "norm":
        x = _norm_inputs(case, draw_, g)
        x["freqs"] = _angles(case["S"], case["D"])
        for n in ("q", "k"):
            if case["mode"] == "jvp":
                x["t" + n] = draw_(*x[n].shape, by=TANGENT_STD)
            else:
                x["g" + n] = draw_(*x[n].shape)
        return x
    x = _pool(case, draw_, g)
    if case["op"] == "append":
        x.update(_norm_inputs(case, draw_, g))
        x["v"] = draw_(case["B"], case["S"], case["Hk"], case["D"])
        x["freqs"] = _angles(case["longest"] + 50 + case["S"], case["D"])
    if case["op"] == "attend":
        x["q"] = draw_(case["B"], case["S"], case["Hq"], case["D"], by=1.5)
    return x


def prepare(case, seed):
    x = _inputs(case, seed)
    x["case"] = case
    if case["op"] == "norm" and case["mode"] == "train":
        for n in ("q", "k", "wq", "wk"):
            x[n].requires_grad_(True)
    if own and case["op"] != "norm":
        from dmad_amd import PagedKVCache

        x["cache"] = PagedKVCache(k_pages=x["k_pages"], v_pages=x["v_pages"], page_table=x["page_table"],
                                  lengths=x["counts"][0], seen=x["counts"][1], weight=x["weight"],
                                  position=x["position"])
    return x


# ---------------------------------------------------------------- one pass


def run(x):
    case = x["case"]
    if case["op"] == "norm":
        return _run_norm(case, x)
    # the state is put back first, so that every pass does the same
    if case["op"] in ("append", "evict"):
        x["counts"].copy_(x["counts0"])
    if case["op"] == "evict":
        x["position"].copy_(x["position0"])
    if case["op"] == "evict" or case.get("weights"):
        x["weight"].copy_(x["weight0"])
    if case["op"] == "append":
        return _run_append(x)
    if case["op"] == "attend":
        return _run_attend(case, x)
    return _run_evict(case, x)


def _run_norm(case, x):
    if own:
        from dmad_amd import qk_norm_rope_with_tangent

        if case["mode"] == "jvp":
            with torch.no_grad():
                (q, tq), (k, tk) = qk_norm_rope_with_tangent((x["q"], x["tq"]), (x["k"], x["tk"]), x["wq"], x["wk"], EPS,
                                                             x["freqs"])
            return q, tq, k, tk
        (q, _), (k, _) = qk_norm_rope_with_tangent((x["q"], None), (x["k"], None), x["wq"], x["wk"], EPS, x["freqs"])
        return (q.detach(), k.detach()) + torch.autograd.grad((q, k), (x["q"], x["k"], x["wq"], x["wk"]), (x["gq"], x["gk"]))
    with torch.no_grad():
        cos, sin = torch.cos(x["freqs"])[:, None], torch.sin(x["freqs"])[:, None]
        if case["mode"] == "jvp":
            return sum((_plain_norm(x[n], x["w" + n], cos, sin, x["t" + n]) for n in ("q", "k")), ())
        outs = [_plain_norm(x[n], x["w" + n], cos, sin)[0] for n in ("q", "k")]
        grads = [_plain_norm_grad(x[n], x["w" + n], cos, sin, x["g" + n]) for n in ("q", "k")]
        return outs[0], outs[1], grads[0][0], grads[1][0], grads[0][1], grads[1][1]


def _rotated(x, cos, sin):
    even, odd = x[..., 0::2], x[..., 1::2]
    return torch.stack((even * cos - odd * sin, odd * cos + even * sin), dim=-1).flatten(-2)


def _plain_norm(x, w, cos, sin, t=None):
    xf, wf = x.float(), w.float()
    r = torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + EPS)
    y = _rotated(xf * r * wf, cos, sin).to(x.dtype)
    if t is None:
        return (y,)
    tf = t.float()
    rd = -r.pow(3) * (xf * tf).mean(-1, keepdim=True)
    return y, _rotated((tf * r + xf * rd) * wf, cos, sin).to(x.dtype)


def _plain_norm_grad(x, w, cos, sin, g):
    xf, wf = x.float(), w.float()
    r = torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + EPS)
    n = xf * r
    back = _rotated(g.float(), cos, -sin)
    dw = (back * n).sum((0, 1, 2), dtype=torch.float64)  # up to millions of rows
    a = back * wf
    return (r * (a - n * (a * n).mean(-1, keepdim=True))).to(x.dtype), dw.to(w.dtype)


def _run_append(x):
    if own:
        from dmad_amd import qk_norm_rope_append

        q = qk_norm_rope_append(x["q"], x["k"], x["v"], x["wq"], x["wk"], EPS, x["freqs"], x["cache"])
        return q, x["k_pages"], x["v_pages"], x["weight"], x["position"], x["counts"]
    B, S, Hk, _ = x["k"].shape
    P = x["k_pages"].shape[2]
    i = torch.arange(S, device="cuda")
    at = x["counts"][1].long()[:, None] + i  # [B, S] positions
    f = x["freqs"][at][:, :, None]
    cos, sin = torch.cos(f), torch.sin(f)
    q = _plain_norm(x["q"], x["wq"], cos, sin)[0]
    k = _plain_norm(x["k"], x["wk"], cos, sin)[0]
    slot = x["counts"][0].long()[:, None] + i
    page = torch.gather(x["page_table"].long(), 1, slot // P)
    x["k_pages"][page, :, slot % P] = k
    x["v_pages"][page, :, slot % P] = x["v"]
    x["weight"][page, :, slot % P] = 0.0
    x["position"][page, :, slot % P] = at.to(torch.int32)[:, :, None].expand(B, S, Hk)
    x["counts"].add_(S)
    return q, x["k_pages"], x["v_pages"], x["weight"], x["position"], x["counts"]


def _run_attend(case, x):
    if own:
        from dmad_amd import paged_attention

        o, lse = paged_attention(x["q"], x["cache"], causal=case["causal"], accumulate=case["weights"], return_lse=True)
        return (o, lse, x["weight"]) if case["weights"] else (o, lse)
    q, table = x["q"], x["page_table"].long()
    B, S, Hq, D = q.shape
    _, Hk, P, _ = x["k_pages"].shape
    M = table.shape[1]
    slot = torch.arange(M * P, device="cuda")
    seen = x["counts"][0][:, None].expand(B, S).long()
    if case["causal"]:
        seen = seen - (S - 1) + torch.arange(S, device="cuda")
    visible = (slot < seen[..., None])[:, None, :, None]  # [B, 1, S, 1, M P]
    k, v = (x[n][table].transpose(1, 2).reshape(B, Hk, M * P, D).float() for n in ("k_pages", "v_pages"))
    qf = q.float().view(B, S, Hk, Hq // Hk, D).permute(0, 2, 1, 3, 4).reshape(B, Hk, -1, D)
    s = (qf @ k.transpose(2, 3) * D ** -0.5).view(B, Hk, S, Hq // Hk, M * P).masked_fill(~visible, -math.inf)
    top = s.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = torch.exp(s - top)
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, torch.ones_like(total), total)
    o = (p.view(B, Hk, -1, M * P) @ v).view(B, Hk, S, Hq // Hk, D).permute(0, 2, 1, 3, 4).reshape(B, S, Hq, D).to(q.dtype)
    lse = (top + torch.log(total)).squeeze(-1).permute(0, 1, 3, 2).reshape(B, Hq, S)
    if not case["weights"]:
        return o, lse
    share = p.sum((2, 3)).view(B, Hk, M, P).transpose(1, 2)  # [B, M, Hk, P]
    x["weight"][table] += share
    return o, lse, x["weight"]


def _run_evict(case, x):
    if own:
        from dmad_amd import evict_low_weight

        evict_low_weight(x["cache"], case["keep"], recent=case["recent"], sink=case["sink"])
        return x["k_pages"], x["v_pages"], x["weight"], x["position"], x["counts"]
    table, keep = x["page_table"].long(), case["keep"]
    B, M = table.shape
    _, Hk, P, _ = x["k_pages"].shape
    n, seen = x["counts"][0].long(), x["counts"][1].long()
    slot = torch.arange(M * P, device="cuda").expand(B, Hk, M * P)
    w, at = (x[name][table].transpose(1, 2).reshape(B, Hk, M * P) for name in ("weight", "position"))
    forced = (at < case["sink"]) | (at >= (seen - case["recent"])[:, None, None])
    key = w.masked_fill(forced, math.inf).masked_fill(slot >= n[:, None, None], -math.inf)
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices
    stays = torch.zeros_like(key, dtype=torch.bool).scatter_(2, order[..., :keep], True)
    hole, moves = ~stays & (slot < keep), stays & (slot >= keep)
    cut = (n > keep)[:, None, None]
    hole, moves = hole & cut, moves & cut
    # the i-th hole takes the i-th slot that moves
    rank = (moves.cumsum(-1) - 1).masked_fill(~moves, M * P)
    source = torch.zeros(B, Hk, M * P + 1, device="cuda", dtype=torch.long).scatter_(2, rank, slot)
    source = torch.where(hole, torch.gather(source, 2, (hole.cumsum(-1) - 1).clamp(min=0)), slot)[..., :keep]
    head = torch.arange(Hk, device="cuda")[None, :, None]
    page = torch.gather(table[:, None].expand(B, Hk, M), 2, source // P)
    to = torch.gather(table[:, None].expand(B, Hk, M), 2, slot[..., :keep] // P)
    for name in ("k_pages", "v_pages", "weight", "position"):
        x[name][to, head, slot[..., :keep] % P] = x[name][page, head, source % P]
    x["counts"][0].clamp_(max=keep)
    return x["k_pages"], x["v_pages"], x["weight"], x["position"], x["counts"]


# ---------------------------------------------------------------- float64 references


def _turn(z, angle):
    """Pairs as complex numbers, turned by the angle."""
    pair = torch.view_as_complex(z.reshape(*z.shape[:-1], -1, 2).contiguous())
    return torch.view_as_real(pair * torch.polar(torch.ones_like(angle), angle)).reshape(z.shape)


def _exact_norm(case, x):
    angle = x["freqs"].double()[None, :, None]
    outs, grads, sums = [], [], []
    for n in ("q", "k"):
        z, w = x[n].double(), x["w" + n].double()
        root = (z.square().sum(-1, keepdim=True) / z.shape[-1] + EPS).sqrt()
        unit = z / root
        outs.append(_turn(unit * w, angle))
        if case["mode"] == "jvp":
            t = x["t" + n].double()
            outs.append(_turn((t - unit * (unit * t).mean(-1, keepdim=True)) / root * w, angle))
        else:
            back = _turn(x["g" + n].double(), -angle)
            sums.append((back * unit).sum((0, 1, 2)))
            back = back * w
            grads.append((back - unit * (unit * back).mean(-1, keepdim=True)) / root)
    return tuple(outs + grads + sums)


def _exact_append(case, x):
    n, seen = x["counts0"].tolist()
    k_pages, v_pages = x["k_pages"].double(), x["v_pages"].double()
    weight, position = x["weight0"].double(), x["position0"].clone()
    table, P, S = x["page_table"].tolist(), case["page"], case["S"]
    qs = []
    for b in range(case["B"]):
        angle = x["freqs"][seen[b]:seen[b] + S].double()[:, None]
        turned = []
        for name in ("q", "k"):
            z = x[name][b].double()
            z = z / (z.square().mean(-1, keepdim=True) + EPS).sqrt() * x["w" + name].double()
            turned.append(_turn(z, angle))
        qs.append(turned[0])
        first = 0
        while first < S:  # the tokens that fall into one page
            page, inside = table[b][(n[b] + first) // P], (n[b] + first) % P
            some = min(S - first, P - inside)
            k_pages[page, :, inside:inside + some] = turned[1][first:first + some].transpose(0, 1)
            v_pages[page, :, inside:inside + some] = x["v"][b, first:first + some].double().transpose(0, 1)
            weight[page, :, inside:inside + some] = 0
            position[page, :, inside:inside + some] = torch.arange(seen[b] + first, seen[b] + first + some, device="cuda",
                                                                   dtype=torch.int32)
            first += some
    return torch.stack(qs), k_pages, v_pages, weight, position, x["counts0"] + S


def _exact_attend(case, x):
    B, S, Hq, D = x["q"].shape
    Hk, group = case["Hk"], Hq // case["Hk"]
    o = torch.zeros(B, S, Hq, D, dtype=torch.float64, device="cuda")
    lse = torch.full((B, Hq, S), -math.inf, dtype=torch.float64, device="cuda")
    weight = x["weight0"].double()
    for b, n in enumerate(_lengths(case)):
        used = x["page_table"][b, :-(-n // case["page"])].long()
        for h in range(Hk):
            k, v = (x[name][used, h].reshape(-1, D)[:n].double() for name in ("k_pages", "v_pages"))
            share = torch.zeros(len(used) * case["page"], dtype=torch.float64, device="cuda")
            for i in range(S):
                m = n - (S - 1 - i) if case["causal"] else n
                if m <= 0:
                    continue
                heads = slice(h * group, (h + 1) * group)
                s = (k[:m] @ x["q"][b, i, heads].double().t()).t() / math.sqrt(D)
                p = torch.softmax(s, dim=-1)
                o[b, i, heads] = p @ v[:m]
                lse[b, heads, i] = torch.logsumexp(s, dim=-1)
                share[:m] += p.sum(0)
            weight[used, h] += share.view(-1, case["page"])
    return (o, lse, weight) if case["weights"] else (o, lse)


def _exact_evict(case, x):
    counts = x["counts0"].cpu().numpy()
    table = x["page_table"].cpu().numpy().astype(np.int64)
    weight0, position0 = x["weight0"].cpu().numpy(), x["position0"].cpu().numpy()
    P, keep = case["page"], case["keep"]
    to, source = [], []  # (page, head, slot in the page)
    for b in range(case["B"]):
        n, seen = int(counts[0, b]), int(counts[1, b])
        if n <= keep:
            continue
        s = np.arange(n)
        for h in range(case["Hk"]):
            w, at = weight0[table[b, s // P], h, s % P], position0[table[b, s // P], h, s % P]
            safe = (at < case["sink"]) | (at >= seen - case["recent"])
            best = np.lexsort((s, -w.astype(np.float64), ~safe))[:keep]
            gone = np.setdiff1d(s[:keep], best)
            tail = np.sort(best[best >= keep])
            to += [(table[b, d // P], h, d % P) for d in gone]
            source += [(table[b, d // P], h, d % P) for d in tail]
    outs = [x["k_pages"].double(), x["v_pages"].double(), x["weight0"].double(), x["position0"].clone()]
    if to:
        to, source = (torch.tensor(np.array(z), device="cuda").unbind(1) for z in (to, source))
        for z in outs:
            z[to] = z[source].clone()
    after = x["counts0"].clone()
    after[0] = after[0].clamp(max=keep)
    return (*outs, after)


def exact(case, seed):
    with torch.no_grad():
        x = _inputs(case, seed)
        return {"norm": _exact_norm, "append": _exact_append, "attend": _exact_attend, "evict": _exact_evict}[case["op"]](case, x)
