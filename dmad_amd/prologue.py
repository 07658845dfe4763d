"""Fused attention-input prologue for gfx950: RMSNorm(+JVP) and RoPE-with-tangent.

In the reference the tensors handed to the JVP attention op are produced by two
separate steps, each a ``torch.func.jvp`` over float32 round trips:
  * ``WanRMSNorm._forward`` under ``torch.func.jvp`` inside
    ``WanSelfAttention._forward_jvp`` (train/wan/rcm/networks/wan2pt1_jvp.py:207-216,
    312-317), applied to the q and k Linear outputs and their tangents;
  * ``apply_rope_with_tangent`` (train/wan/rcm/utils/rope.py:106-114) inside
    ``MinimalA2AAttnOpWithT.forward`` (train/wan/rcm/utils/jvp_helper.py:180-196).
``rmsnorm_rope_with_tangent`` does both in one HIP kernel (one HBM read of the
Linear output and its tangent, one write of the rotated pair), with the
reference's rounding points. ``apply_rope_with_tangent`` is the rotation alone
(the reference function of that name), with a backward: the rotation's
transpose is the rotation by the negated angles, run on the same kernel.
Device work only: tensors off the GPU raise.
"""
from __future__ import annotations

import torch

from . import _native as nat


def rmsnorm_rope_with_tangent(x_with_t, weight, eps, freqs, num_heads):
    """((y, ty), weight [C], eps, freqs [L, D/2] or None, H) -> (q, q_dot) as [B, L, H, D].

    ``y`` is the [B, L, C] Linear output (C = H*D) and ``ty`` its tangent (or None
    for the primal only). The tangent output is detached, as both reference steps
    detach it (wan2pt1_jvp.py:212, jvp_helper.py:194).
    """
    y, ty = x_with_t
    if y.device.type != "cuda":
        raise RuntimeError("dmad_amd prologue runs on the GPU only (HIP kernel); got a tensor on " + str(y.device))
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (y, ty, weight)):
        raise RuntimeError("rmsnorm_rope_with_tangent has no backward: call it under torch.no_grad() "
                           "(the JVP evaluations it serves run without gradients)")
    B, L, C = y.shape
    if C % num_heads:
        raise ValueError(f"model dim {C} is not a multiple of num_heads {num_heads}")
    D = C // num_heads
    code = nat.dtype_code(y.dtype)
    if weight.dtype != y.dtype:
        weight = weight.to(y.dtype)
    y = y.reshape(B * L, C)
    if y.stride(-1) != 1 or y.stride(0) % 8 or y.data_ptr() % 16:
        y = y.contiguous()
    if ty is not None:
        ty = ty.reshape(B * L, C)
        if ty.stride() != y.stride() or ty.data_ptr() % 16:
            y, ty = y.contiguous(), ty.contiguous()
    weight = weight.contiguous()
    if freqs is not None:
        freqs = freqs.reshape(L, D // 2).to(device=y.device, dtype=torch.float32).contiguous()
    out = torch.empty((B * L, C), device=y.device, dtype=y.dtype)
    tout = torch.empty_like(out) if ty is not None else None
    nat.check(
        nat.lib().dmad_rmsnorm_rope_jvp(
            code, B * L, L, num_heads, D, nat.ptr(y), nat.ptr(ty), y.stride(0), nat.ptr(weight),
            nat.ctypes.cast(nat.ptr(freqs), nat._FP), float(eps), nat.ptr(out), nat.ptr(tout), out.stride(0),
            nat.stream_ptr(y.device),
        )
    )
    q = out.view(B, L, num_heads, D)
    return q, (None if tout is None else tout.view(B, L, num_heads, D).detach())


def _rope_launch(x, t_x, freqs):
    """Rotation of [B, S, H, D] x (and t_x) by freqs [S, D/2]; returns [B, S, H, D] outputs."""
    if x.device.type != "cuda":
        raise RuntimeError("dmad_amd RoPE runs on the GPU only (HIP kernel); got a tensor on " + str(x.device))
    B, S, H, D = x.shape
    code = nat.dtype_code(x.dtype)

    def rows(t):
        if t.stride(3) != 1 or t.stride(2) != D or t.stride(1) % 8 or t.data_ptr() % 16 or (B > 1 and t.stride(0) != S * t.stride(1)):
            t = t.contiguous()
        return t

    x = rows(x)
    if t_x is not None:
        t_x = rows(t_x)
        if t_x.stride() != x.stride():
            x, t_x = x.contiguous(), t_x.contiguous()
    f = freqs.reshape(S, D // 2).to(device=x.device, dtype=torch.float32).contiguous()
    out = torch.empty((B, S, H, D), device=x.device, dtype=x.dtype)
    tout = torch.empty_like(out) if t_x is not None else None
    nat.check(
        nat.lib().dmad_rmsnorm_rope_jvp(
            code, B * S, S, H, D, nat.ptr(x), nat.ptr(t_x), x.stride(1), nat.ptr(None),
            nat.ctypes.cast(nat.ptr(f), nat._FP), 0.0, nat.ptr(out), nat.ptr(tout), out.stride(1),
            nat.stream_ptr(x.device),
        )
    )
    return out, tout


class _RopeWithTangent(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, t_x, freqs):
        ctx.save_for_backward(freqs)
        return _rope_launch(x, t_x, freqs)

    @staticmethod
    def backward(ctx, g_out, g_tout):
        (freqs,) = ctx.saved_tensors
        neg = -freqs
        gx = gtx = None
        if g_out is not None and g_tout is not None and g_out.dtype == g_tout.dtype:
            gx, gtx = _rope_launch(g_out, g_tout, neg)
        else:
            if g_out is not None:
                gx = _rope_launch(g_out, None, neg)[0]
            if g_tout is not None:
                gtx = _rope_launch(g_tout, None, neg)[0]
        return gx, gtx, None


def apply_rope_with_tangent(x, t_x, freqs, fused: bool = False):
    """Interleaved rotary embedding of x [B, S, H, D] and of its tangent t_x by
    freqs [S, D/2] (train/wan/rcm/utils/rope.py:106-114, apply_rope :56-70):
    pairs (x[2i], x[2i+1]) rotated by freqs[s, i] in float32, cast back to the
    input type. ``freqs is None`` returns the inputs. ``fused`` is accepted for
    the reference's signature and ignored (one kernel either way). Differentiable:
    the gradient is the rotation by -freqs.
    """
    del fused
    if freqs is None:
        return x, t_x
    if t_x is None:
        return _RopeWithTangent.apply(x, None, freqs)[0], None
    return _RopeWithTangent.apply(x, t_x, freqs)


# ---------------------------------------------------------------- norm of each head, and rotation

HEAD_DIMS = (16, 32, 64, 128, 256)


def _check_same_device(op, *ts):
    dev = None
    for t in ts:
        if t is None:
            continue
        if t.device.type != "cuda":
            raise RuntimeError(f"{op} runs on the GPU only (HIP kernel); got a tensor on {t.device}")
        if dev is not None and t.device != dev:
            raise ValueError(f"{op}: tensors on {dev} and on {t.device}")
        dev = t.device
    return dev


def row_strides(t):
    """Strides the kernels take for a [.., D] operand (an axis of one element counts as 0), or None
    where rows are not contiguous and 16-byte aligned."""
    if t.shape[-1] != 1 and t.stride(-1) != 1 or t.data_ptr() % 16:
        return None
    st = [0 if n == 1 else s for n, s in zip(t.shape[:-1], t.stride()[:-1])]
    step = 16 // t.element_size()
    return None if any(s % step for s in st) else (*st, 1)


def readable_rows(t):
    """(tensor, ctypes strides): ``t`` itself or a contiguous copy the kernels can read."""
    st = row_strides(t)
    if st is None:
        # a contiguous tensor may still start unaligned
        t = t.contiguous() if not t.is_contiguous() else t.clone(memory_format=torch.contiguous_format)
        st = row_strides(t)
    return t, nat.int64_array(st)


def _norm_weights(op, x, D, wq, wk):
    """(wq, wk, their type code): one type for both, the operands' own or float32."""
    for w in (wq, wk):
        if w is not None and (w.shape != (D,) or not w.is_floating_point() or w.dtype == torch.float64):
            raise ValueError(f"{op}: weights must be [{D}] in the operands' type or float32, "
                             f"got {tuple(w.shape)} {w.dtype}")
    given = [w for w in (wq, wk) if w is not None]
    dtype = x.dtype if all(w.dtype == x.dtype for w in given) else torch.float32
    aligned = [None if w is None else w.to(dtype).contiguous() for w in (wq, wk)]
    aligned = [w.clone() if w is not None and w.data_ptr() % 16 else w for w in aligned]
    return aligned[0], aligned[1], nat.dtype_code(dtype)


def _angle_table(op, freqs, B, S, D):
    """(float32 table, batch stride) of [S, D/2] or [B, S, D/2] angles."""
    if freqs is None:
        return None, 0
    if freqs.shape[-1] != D // 2 or freqs.dim() not in (2, 3) or freqs.shape[-2] != S or \
            (freqs.dim() == 3 and freqs.shape[0] not in (1, B)):
        raise ValueError(f"{op}: freqs must be [{S}, {D // 2}] or [{B}, {S}, {D // 2}], got {tuple(freqs.shape)}")
    f = freqs.to(torch.float32).contiguous()
    return f, (S * (D // 2) if f.dim() == 3 and f.shape[0] == B and B > 1 else 0)


def _qk_shapes(op, q, k):
    given = [x for x in (q, k) if x is not None]
    if not given:
        raise ValueError(f"{op}: neither q nor k")
    for x in given:
        if x.dim() != 4:
            raise ValueError(f"{op}: q and k must be [B, S, H, D], got {tuple(x.shape)}")
    B, S, _, D = given[0].shape
    if len(given) == 2 and (k.shape[0], k.shape[1], k.shape[3]) != (B, S, D):
        raise ValueError(f"{op}: q {tuple(q.shape)} and k {tuple(k.shape)} differ in more than their heads")
    if len(given) == 2 and q.dtype != k.dtype:
        raise ValueError(f"{op}: q is {q.dtype} and k {k.dtype}")
    if D not in HEAD_DIMS:
        raise NotImplementedError(f"{op}: head dim {D} is not one of {HEAD_DIMS}")
    return B, S, 0 if q is None else q.shape[2], 0 if k is None else k.shape[2], D


class _QkNormRope(torch.autograd.Function):
    """(q, tq, k, tk, wq, wk, freqs, eps) -> (q', tq', k', tk'); gradients of the primal outputs."""

    @staticmethod
    def forward(ctx, q, tq, k, tk, wq, wk, freqs, eps):
        op = "qk_norm_rope_with_tangent"
        B, S, Hq, Hk, D = _qk_shapes(op, q, k)
        x = q if q is not None else k
        cq, ck, wcode = _norm_weights(op, x, D, wq, wk)
        f, fb = _angle_table(op, freqs, B, S, D)
        ops, outs = [], []
        for t in (q, tq, k, tk):
            ops.append((None, None) if t is None else readable_rows(t))
            outs.append(None if t is None else torch.empty(t.shape, device=t.device, dtype=t.dtype))
        with nat.on_device(x.device):
            nat.check(nat.lib().dmad_qk_norm_rope(
                nat.dtype_code(x.dtype), wcode, B, S, Hq, Hk, D, *(nat.ptr(t) for t, _ in ops), *(s for _, s in ops),
                nat.ptr(cq), nat.ptr(ck), nat.ptr(f), fb, float(eps), *(nat.ptr(t) for t in outs),
                nat.stream_ptr(x.device)))
        ctx.save_for_backward(q, k, wq, wk, freqs)
        ctx.eps = float(eps)
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(*(t for t in (outs[1], outs[3]) if t is not None))
        return tuple(outs)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, gq, _gtq, gk, _gtk):
        q, k, wq, wk, freqs = ctx.saved_tensors
        need = ctx.needs_input_grad
        # an output whose gradient did not arrive adds nothing
        q, k = (q if gq is not None else None), (k if gk is not None else None)
        if q is None and k is None:
            return (None,) * 8
        op = "qk_norm_rope_with_tangent"
        B, S, Hq, Hk, D = _qk_shapes(op, q, k)
        x = q if q is not None else k
        cq, ck, wcode = _norm_weights(op, x, D, wq, wk)
        f, fb = _angle_table(op, freqs, B, S, D)
        grads = [None if g is None else g.to(x.dtype) for g in (gq, gk)]
        ops = [(None, None) if t is None else readable_rows(t) for t in (q, grads[0], k, grads[1])]
        dx = [None if t is None else torch.empty(t.shape, device=t.device, dtype=t.dtype) for t in (q, k)]
        dw = [torch.empty_like(w) if w is not None and t is not None and need[i] else None
              for w, t, i in ((cq, q, 4), (ck, k, 5))]
        if x.numel() == 0:
            dw = [None if w is None else w.zero_() for w in dw]
        else:
            size = nat.qk_norm_rope_bwd_workspace_bytes(B, S, Hq, Hk, D) if any(w is not None for w in dw) else 0
            ws_ptr, ws_size, ws = nat.workspace(size, x.device)
            with nat.on_device(x.device):
                nat.check(nat.lib().dmad_qk_norm_rope_bwd(
                    nat.dtype_code(x.dtype), wcode, B, S, Hq, Hk, D, *(nat.ptr(t) for t, _ in ops),
                    *(s for _, s in ops), nat.ptr(cq if q is not None else None),
                    nat.ptr(ck if k is not None else None), nat.ptr(f), fb, ctx.eps,
                    *(nat.ptr(t) for t in dx), *(nat.ptr(t) for t in dw), ws_ptr, ws_size, nat.stream_ptr(x.device)))
        dw = [None if g is None else g.to(w.dtype) for g, w in zip(dw, (wq, wk))]
        return dx[0], None, dx[1], None, dw[0], dw[1], None, None


def qk_norm_rope_with_tangent(q_withT, k_withT, q_weight, k_weight, eps, freqs):
    """RMSNorm of queries and keys for each head and their rotation, in one pass over both.

    ``((q, tq), (k, tk), wq [D], wk [D], eps, freqs) -> ((q', tq'), (k', tk'))`` for q [B, S, Hq, D]
    and k [B, S, Hk, D] (any head counts; bf16, fp16 or fp32; D in 16, 32, 64, 128, 256; any strides
    with contiguous 16-byte-aligned rows are read in place). Each head's row x becomes
    R(x / sqrt(mean(x^2) + eps) * w), R turning the pairs (x[2i], x[2i+1]) by freqs[s, i] as
    ``apply_rope_with_tangent`` does; float32 throughout, rounded once at the end. This is the
    norm per head; ``rmsnorm_rope_with_tangent`` is the one over the whole model width.

    ``tq``/``tk``: tangents, given for both or for neither; their outputs are detached. ``k_withT``
    (or ``q_withT``) may be ``(None, None)``: the other alone. A weight of None skips that norm,
    ``freqs`` None the rotation; freqs are [S, D/2], or [B, S, D/2] for angles per sequence.
    Weights have the operands' type or float32. Differentiable in q, k and the weights.
    """
    op = "qk_norm_rope_with_tangent"
    (q, tq), (k, tk) = q_withT, k_withT
    _check_same_device(op, q, tq, k, tk, q_weight, k_weight, freqs)
    _qk_shapes(op, q, k)
    nat.dtype_code((q if q is not None else k).dtype)
    if not eps >= 0:
        raise ValueError(f"{op}: eps must be non-negative, got {eps}")
    for x, t in ((q, tq), (k, tk)):
        if t is not None and (x is None or t.shape != x.shape or t.dtype != x.dtype):
            raise ValueError(f"{op}: a tangent has its operand's shape and type")
    if (tq is not None or tk is not None) and any(x is not None and t is None for x, t in ((q, tq), (k, tk))):
        raise ValueError(f"{op}: tangents of both q and k, or of neither")
    q, tq, k, tk = _QkNormRope.apply(q, tq, k, tk, q_weight, k_weight, freqs, eps)
    return (q, tq), (k, tk)
