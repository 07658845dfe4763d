"""CPU oracle of the per-head norm and rotation, the paged cache, its attention and its eviction.

Plain float64 torch, written from the definitions, one token, slot or head at a time where that is
clearer. A cache is a dict of CPU tensors with the fields of ``dmad_amd.PagedKVCache``.
"""
from __future__ import annotations

import math

import torch

FIELDS = ("k_pages", "v_pages", "page_table", "lengths", "seen", "weight", "position")


def rotate(x, freqs):
    """x [B, S, H, D] float64, pairs turned by freqs [S, D/2] or [B, S, D/2]; None: as it is."""
    if freqs is None:
        return x
    a = freqs.double()
    a = (a if a.dim() == 3 else a[None])[:, :, None]
    e, o = x[..., 0::2], x[..., 1::2]
    return torch.stack((e * a.cos() - o * a.sin(), e * a.sin() + o * a.cos()), -1).reshape(x.shape)


def norm_rope(x, w, eps, freqs):
    """The operator on one operand, differentiable, in float64."""
    x = x.double()
    if w is not None:
        x = x / (x.pow(2).mean(-1, keepdim=True) + eps).sqrt() * w.double()
    return rotate(x, freqs)


def norm_rope_tangent(x, t, w, eps, freqs):
    """Its derivative along t, by torch's forward mode."""
    return torch.func.jvp(lambda z: norm_rope(z, w, eps, freqs), (x.double(),), (t.double(),))[1]


def cache_of(cache):
    """CPU copies of a PagedKVCache's tensors."""
    return {n: None if getattr(cache, n) is None else getattr(cache, n).detach().cpu().clone() for n in FIELDS}


def capacity(c):
    return c["page_table"].shape[1] * c["k_pages"].shape[2]


def length(c, b):
    return min(max(int(c["lengths"][b]), 0), capacity(c))


def locate(c, b, s):
    """(page, slot in it) of slot s of sequence b, or None where no page holds it."""
    P = c["k_pages"].shape[2]
    page = int(c["page_table"][b, s // P])
    return (page, s % P) if 0 <= page < c["k_pages"].shape[0] else None


def append(c, q, k, v, wq, wk, eps, freqs):
    """Appends in place; (q', k' [B, S, Hk, D] float64 as they should be). Pages get k' in their type."""
    B, S = k.shape[:2]
    cap = capacity(c)
    pos = c["seen"].long()[:, None] + torch.arange(S)
    a = None
    if freqs is not None:
        a = torch.full((B, S, freqs.shape[1]), math.nan, dtype=torch.float64)
        ok = (pos >= 0) & (pos < freqs.shape[0])
        a[ok] = freqs.double()[pos[ok]]
    kn = norm_rope(k, wk, eps, a)
    for b in range(B):
        n = length(c, b)
        for i in range(S):
            if n + i >= cap:
                continue
            at = locate(c, b, n + i)
            if at is None:
                continue
            c["k_pages"][at[0], :, at[1]] = kn[b, i].to(c["k_pages"].dtype)
            c["v_pages"][at[0], :, at[1]] = v[b, i]
            if c["weight"] is not None:
                c["weight"][at[0], :, at[1]] = 0
                c["position"][at[0], :, at[1]] = int(pos[b, i])
        c["lengths"][b] = min(n + S, cap)
    c["seen"] += S
    return None if q is None else norm_rope(q, wq, eps, a), kn


def attend(c, q, scale=None, causal=False, accumulate=False):
    """(o, lse, bound): bound[b, i, h] = sum_j p_j |v_j|, and per row the largest scaled sum |q k| and
    sum |v|, for error bounds. With accumulate, adds to c["weight"] (made float64)."""
    B, S, Hq, D = q.shape
    Hk = c["k_pages"].shape[1]
    G = Hq // Hk
    scale = D ** -0.5 if scale is None else scale
    o = torch.zeros(B, S, Hq, D, dtype=torch.float64)
    lse = torch.full((B, Hq, S), -math.inf, dtype=torch.float64)
    pv, sv = torch.zeros_like(o), torch.zeros_like(o)
    size = torch.zeros(B, S, Hq, 1, dtype=torch.float64)
    if accumulate:
        c["weight"] = c["weight"].double()
    for b in range(B):
        n = length(c, b)
        where = [(s, at) for s in range(n) if (at := locate(c, b, s)) is not None]
        for i in range(S):
            see = n - (S - 1 - i) if causal else n
            at = [w for s, w in where if s < see]
            if not at:
                continue
            page, slot = torch.tensor(at).unbind(1)
            for h in range(Hq):
                k, v = c["k_pages"][page, h // G, slot].double(), c["v_pages"][page, h // G, slot].double()
                s = (k @ q[b, i, h].double()) * scale
                p = torch.softmax(s, 0)
                o[b, i, h] = p @ v
                lse[b, h, i] = torch.logsumexp(s, 0)
                pv[b, i, h] = p @ v.abs()
                sv[b, i, h] = v.abs().sum(0)
                size[b, i, h] = ((k.abs() @ q[b, i, h].double().abs()) * scale).max()
                if accumulate:
                    c["weight"][page, h // G, slot] += p
    return o, lse, (pv, sv, size)


def attend_long(c, q, scale=None, causal=False, accumulate=False):
    """``attend`` a key head at a time, for long caches, on whichever device the cache lies."""
    B, S, Hq, D = q.shape
    N, Hk, P, _ = c["k_pages"].shape
    G, dev = Hq // Hk, c["k_pages"].device
    scale = D ** -0.5 if scale is None else scale
    o = torch.zeros(B, S, Hq, D, dtype=torch.float64, device=dev)
    lse = torch.full((B, Hq, S), -math.inf, dtype=torch.float64, device=dev)
    pv, sv = torch.zeros_like(o), torch.zeros_like(o)
    size = torch.zeros(B, S, Hq, 1, dtype=torch.float64, device=dev)
    if accumulate:
        c["weight"] = c["weight"].double()
    for b in range(B):
        n = length(c, b)
        slot = torch.arange(n, device=dev)
        page = c["page_table"][b].long()[slot // P]
        there = (page >= 0) & (page < N)
        slot, page = slot[there], page[there]
        see = torch.arange(S, device=dev).repeat_interleave(G) + (n - S + 1) if causal else torch.full((S * G,), n, device=dev)
        seen = slot[None] < see[:, None]
        some = seen.any(1)
        if not bool(some.any()):
            continue
        for h in range(Hk):
            k, v = (c[x][page, h, slot % P].double() for x in ("k_pages", "v_pages"))
            rows = q[b, :, h * G:(h + 1) * G].reshape(S * G, D).double()
            s = (rows @ k.T.contiguous() * scale).masked_fill(~seen, -math.inf)
            p = torch.where(some[:, None], torch.softmax(s, 1), torch.zeros((), dtype=torch.float64, device=dev))
            at = (b, slice(None), slice(h * G, (h + 1) * G))
            o[at], pv[at], sv[at] = (x.view(S, G, D) for x in (p @ v, p @ v.abs(), seen.double() @ v.abs()))
            lse[b, h * G:(h + 1) * G] = torch.logsumexp(s, 1).view(S, G).T
            size[at] = ((rows.abs() @ k.abs().T.contiguous() * scale) * seen).amax(1).view(S, G, 1)
            if accumulate:
                c["weight"].index_put_((page, torch.tensor(h, device=dev), slot % P), p.sum(0), accumulate=True)
    return o, lse, (pv, sv, size)


def evict(c, keep, recent=0, sink=0):
    """Cuts the cache in place. Only slots that a page holds count: the sequence then ends behind the
    keep-th of them."""
    Hk = c["k_pages"].shape[1]
    for b in range(c["page_table"].shape[0]):
        n = length(c, b)
        held = [s for s in range(n) if locate(c, b, s) is not None]
        end = n
        if len(held) > keep:
            end = held[keep - 1] + 1
            for h in range(Hk):
                rank = []
                for s in held:
                    at = locate(c, b, s)
                    w, p = float(c["weight"][at[0], h, at[1]]), int(c["position"][at[0], h, at[1]])
                    stays = p < sink or p >= int(c["seen"][b]) - recent
                    rank.append((0, 0.0, s) if stays else (1, 0.0, s) if math.isnan(w) else (2, -w, s))
                kept = {s for _, _, s in sorted(rank)[:keep]}
                holes = [s for s in held if s < end and s not in kept]
                tail = [s for s in held if s >= end and s in kept]
                assert len(holes) == len(tail)
                for to, source in zip(holes, tail):
                    (tp, ts), (fp, fs) = locate(c, b, to), locate(c, b, source)
                    for name in ("k_pages", "v_pages", "weight", "position"):
                        c[name][tp, h, ts] = c[name][fp, h, fs]
        c["lengths"][b] = end
