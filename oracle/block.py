"""CPU oracle of the operators around a block's attention and of the attention behind shared prefixes.

Plain float64 torch, written from the definitions.
"""
from __future__ import annotations

import math

import torch

from oracle import streaming as st


def normed(x, kind, eps):
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    return x / (x.pow(2).mean(-1, keepdim=True) + eps).sqrt()


def rows_of(v, S):
    """A vector per group of tokens [B, F, C] as one per token [B, S, C]."""
    return v.repeat_interleave(S // v.shape[1], dim=1) if v.shape[1] else v


OPERANDS = ("x", "y", "gate", "scale", "shift", "weight", "bias", "post_weight")


def gated_norm(x, y=None, gate=None, scale=None, shift=None, weight=None, bias=None, post_weight=None, eps=1e-6, kind="layer",
               rs=1.0):
    """(x', n), differentiable."""
    S = x.shape[1]
    if y is not None:
        if post_weight is not None:
            y = normed(y, "rms", eps) * post_weight
        x = x + rs * (y if gate is None else rows_of(gate, S) * y)
    n = normed(x, kind, eps)
    if weight is not None:
        n = n * weight
    if bias is not None:
        n = n + bias
    if scale is not None:
        n = n * (1 + rows_of(scale, S))
    if shift is not None:
        n = n + rows_of(shift, S)
    return x, n


def gated_norm_tangent(ops, tangents, **how):
    """(tx', tn) of gated_norm at ``ops`` along ``tangents`` (both by name; what is missing is zero), by forward mode."""
    names = list(ops)
    along = tuple(tangents[n].double() if n in tangents else torch.zeros_like(ops[n].double()) for n in names)
    return torch.func.jvp(lambda *ts: gated_norm(**dict(zip(names, ts)), **how), tuple(ops[n].double() for n in names), along)[1]


def turn(x, positions, frequencies, half, factor=1.0, back=False):
    """x [B, S, H, D] float64 with the pairs of its first 2 len(frequencies) elements turned, one element at a time where
    that is clearer: pair i by positions [S] or [B, S] times frequencies[i]."""
    R = 2 * frequencies.shape[0]
    angle = positions.double()[..., None] * frequencies.double()
    angle = (angle if angle.dim() == 3 else angle[None])[:, :, None]
    if back:
        angle = -angle
    c, s = angle.cos() * factor, angle.sin() * factor
    y = x.clone()
    lo = torch.arange(R // 2) * (1 if half else 2)
    hi = lo + (R // 2 if half else 1)
    y[..., lo] = x[..., lo] * c - x[..., hi] * s
    y[..., hi] = x[..., hi] * c + x[..., lo] * s
    return y


def prefix_attend(p, c, q, scale=None, causal=False):
    """(o, lse, bound) as streaming.attend, each sequence's slots behind those of its prefix; caches as dicts of tensors."""
    B, S, Hq, D = q.shape
    Hk = c["k_pages"].shape[1]
    G, n = Hq // Hk, B // p["page_table"].shape[0]
    scale = D ** -0.5 if scale is None else scale
    dev = q.device
    o = torch.zeros(B, S, Hq, D, dtype=torch.float64, device=dev)
    lse = torch.full((B, Hq, S), -math.inf, dtype=torch.float64, device=dev)
    pv, sv = torch.zeros_like(o), torch.zeros_like(o)
    size = torch.zeros(B, S, Hq, 1, dtype=torch.float64, device=dev)

    def held(c, b):
        """k, v [slots, Hk, D] float64 of the slots that a page holds, and their numbers."""
        N, _, P, _ = c["k_pages"].shape
        slot = torch.arange(st.length(c, b), device=dev)
        page = c["page_table"][b].long()[slot // P] if slot.numel() else slot
        there = (page >= 0) & (page < N)
        slot, page = slot[there], page[there]
        return c["k_pages"][page, :, slot % P].double(), c["v_pages"][page, :, slot % P].double(), slot

    for b in range(B):
        pk, pv_, pslot = held(p, b // n)
        ok, ov, oslot = held(c, b)
        length = st.length(c, b)
        k, v = torch.cat((pk, ok)), torch.cat((pv_, ov))
        for i in range(S):
            see = length - (S - 1 - i) if causal else length
            seen = torch.cat((torch.ones_like(pslot, dtype=torch.bool), oslot < see))
            if not bool(seen.any()):
                continue
            for h in range(Hk):
                at = (b, i, slice(h * G, (h + 1) * G))
                rows = q[at].double()
                kk, vv = k[seen, h], v[seen, h]
                s = rows @ kk.t().contiguous() * scale
                w = torch.softmax(s, -1)
                o[at], pv[at], sv[at] = w @ vv, w @ vv.abs(), vv.abs().sum(0)
                lse[b, h * G:(h + 1) * G, i] = torch.logsumexp(s, -1)
                size[at] = (rows.abs() @ kk.abs().t().contiguous() * scale).amax(-1, keepdim=True)
    return o, lse, (pv, sv, size)
