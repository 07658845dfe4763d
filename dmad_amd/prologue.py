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
``qk_norm_rope_with_tangent`` is the norm per head of queries and keys with the
rotation in the same pass, tangents and a backward (no counterpart there).
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
        if not t.is_cuda:
            raise RuntimeError(f"{op} runs on the GPU only (HIP kernel); got a tensor on {t.device}")
        if dev is None:
            dev = t.device
        elif t.device != dev:
            raise ValueError(f"{op}: tensors on {dev} and on {t.device}")
    return dev


# ctypes strides by (shape, strides, element size); None where the kernels cannot read the rows in place
_row_strides: dict = {}


def _strides_of_rows(t):
    key = (t.shape, t.stride(), t.element_size())
    arr = _row_strides.get(key, 0)
    if arr == 0:
        *shape, D = t.shape
        # an axis of one element is never stepped along
        st = [0 if n == 1 else s for n, s in zip(shape, t.stride()[:-1])]
        step = 16 // t.element_size()
        bad = (D != 1 and t.stride(-1) != 1) or any(s % step for s in st)
        if len(_row_strides) > 4096:
            _row_strides.clear()
        arr = _row_strides[key] = None if bad else nat.int64_array((*st, 1))
    return arr


def readable_rows(t):
    """(tensor, ctypes strides): ``t`` itself where its rows are contiguous and 16-byte aligned, else a
    contiguous copy."""
    st = _strides_of_rows(t)
    if st is None or t.data_ptr() % 16:
        t = t.clone(memory_format=torch.contiguous_format)
        st = _strides_of_rows(t)
    return t, st


def _norm_weights(op, x, D, wq, wk):
    """(wq, wk, their type code) as the kernels take them: one type for both, the operands' own or float32."""
    dtype = x.dtype
    for w in (wq, wk):
        if w is None:
            continue
        if w.dim() != 1 or w.shape[0] != D or w.dtype not in (torch.float32, torch.bfloat16, torch.float16):
            raise ValueError(f"{op}: weights must be [{D}] in the operands' type or float32, "
                             f"got {tuple(w.shape)} {w.dtype}")
        if w.dtype != dtype:
            dtype = torch.float32

    def as_read(w):
        if w is None or w.dtype == dtype and w.is_contiguous() and not w.data_ptr() % 16:
            return w
        return torch.empty(D, device=w.device, dtype=dtype).copy_(w.detach())

    return as_read(wq), as_read(wk), nat.dtype_code(dtype)


def _angle_table(op, freqs, B, S, D):
    """(float32 table, batch stride) of [S, D/2] or [B, S, D/2] angles."""
    if freqs is None:
        return None, 0
    if freqs.shape[-1] != D // 2 or freqs.dim() not in (2, 3) or freqs.shape[-2] != S or \
            (freqs.dim() == 3 and freqs.shape[0] not in (1, B)):
        raise ValueError(f"{op}: freqs must be [{S}, {D // 2}] or [{B}, {S}, {D // 2}], got {tuple(freqs.shape)}")
    if freqs.dtype != torch.float32 or not freqs.is_contiguous():
        freqs = freqs.to(torch.float32).contiguous()
    return freqs, (S * (D // 2) if freqs.dim() == 3 and B > 1 and freqs.shape[0] == B else 0)


def _qk_shapes(op, q, k):
    x = q if q is not None else k
    if x is None:
        raise ValueError(f"{op}: neither q nor k")
    if x.dim() != 4 or (k is not None and k.dim() != 4):
        raise ValueError(f"{op}: q and k must be [B, S, H, D], got {tuple(x.shape if x.dim() != 4 else k.shape)}")
    B, S, H, D = x.shape
    if q is None:
        Hq, Hk = 0, H
    elif k is None:
        Hq, Hk = H, 0
    else:
        Bk, Sk, Hk, Dk = k.shape
        Hq = H
        if Bk != B or Sk != S or Dk != D:
            raise ValueError(f"{op}: q {tuple(q.shape)} and k {tuple(k.shape)} differ in more than their heads")
        if q.dtype != k.dtype:
            raise ValueError(f"{op}: q is {q.dtype} and k {k.dtype}")
    if D not in HEAD_DIMS:
        raise NotImplementedError(f"{op}: head dim {D} is not one of {HEAD_DIMS}")
    return x, B, S, Hq, Hk, D


_NOTHING = (None, None)


class _QkCall:
    """What forward and backward of one call share, besides its operands: sizes, the weights and the
    angles as the kernels take them."""

    __slots__ = ("device", "code", "B", "S", "Hq", "Hk", "D", "wq", "wk", "wcode", "freqs", "freqs_b", "eps")


def _qk_forward(call, q, tq, k, tk):
    """The launch: (q', tq', k', tk') and q and k as they were read."""
    q, sq = _NOTHING if q is None else readable_rows(q)
    k, sk = _NOTHING if k is None else readable_rows(k)
    tq, stq = _NOTHING if tq is None else readable_rows(tq)
    tk, stk = _NOTHING if tk is None else readable_rows(tk)
    dev = call.device
    oq, otq, ok, otk = (None if t is None else torch.empty(t.shape, device=dev, dtype=t.dtype) for t in (q, tq, k, tk))
    with nat.on_device(dev):
        nat.check(nat.lib().dmad_qk_norm_rope(
            call.code, call.wcode, call.B, call.S, call.Hq, call.Hk, call.D, nat.ptr(q), nat.ptr(tq), nat.ptr(k),
            nat.ptr(tk), sq, stq, sk, stk, nat.ptr(call.wq), nat.ptr(call.wk), nat.ptr(call.freqs), call.freqs_b,
            call.eps, nat.ptr(oq), nat.ptr(otq), nat.ptr(ok), nat.ptr(otk), nat.stream_ptr(dev)))
    return oq, otq, ok, otk, q, k


class _QkNormRope(torch.autograd.Function):
    """(call, q, tq, k, tk, wq, wk) -> (q', tq', k', tk'); gradients of the primal outputs."""

    @staticmethod
    def forward(ctx, call, q, tq, k, tk, wq, wk):
        oq, otq, ok, otk, q, k = _qk_forward(call, q, tq, k, tk)
        ctx.save_for_backward(q, k, wq, wk, call.freqs)
        ctx.call = call
        ctx.set_materialize_grads(False)
        if tq is not None or tk is not None:
            ctx.mark_non_differentiable(*(t for t in (otq, otk) if t is not None))
        return oq, otq, ok, otk

    @staticmethod
    def backward(ctx, gq, _gtq, gk, _gtk):
        # a backward that is itself recorded (create_graph) must refuse to be differentiated
        if torch.is_grad_enabled():
            return _qk_backward_once(ctx, gq, gk)
        return _qk_backward(ctx, gq, gk)


def _qk_backward(ctx, gq, gk):
    q, k, wq, wk, _ = ctx.saved_tensors  # unpacked, so that a change in place is noticed
    call, need = ctx.call, ctx.needs_input_grad
    cq, ck, Hq, Hk, dev = call.wq, call.wk, call.Hq, call.Hk, call.device
    sq = sgq = sk = sgk = dq = dk = dwq = dwk = ws = ws_ptr = None
    ws_size = 0
    # an output whose gradient did not arrive adds nothing
    if gq is not None:
        q, sq = readable_rows(q)
        gq, sgq = readable_rows(gq)
        dq = torch.empty(q.shape, device=dev, dtype=q.dtype)
        if cq is not None and need[5]:
            dwq = torch.empty_like(cq)
    else:
        q, cq, Hq = None, None, 0
    if gk is not None:
        k, sk = readable_rows(k)
        gk, sgk = readable_rows(gk)
        dk = torch.empty(k.shape, device=dev, dtype=k.dtype)
        if ck is not None and need[6]:
            dwk = torch.empty_like(ck)
    else:
        k, ck, Hk = None, None, 0
    if gq is None and gk is None:
        return (None,) * 7
    if call.B * call.S == 0:
        for dw in (dwq, dwk):
            if dw is not None:
                dw.zero_()
    else:
        if dwq is not None or dwk is not None:
            ws_ptr, ws_size, ws = nat.workspace(
                nat.qk_norm_rope_bwd_workspace_bytes(call.B, call.S, Hq, Hk, call.D), dev)
        with nat.on_device(dev):
            nat.check(nat.lib().dmad_qk_norm_rope_bwd(
                call.code, call.wcode, call.B, call.S, Hq, Hk, call.D, nat.ptr(q), nat.ptr(gq), nat.ptr(k), nat.ptr(gk),
                sq, sgq, sk, sgk, nat.ptr(cq), nat.ptr(ck), nat.ptr(call.freqs), call.freqs_b, call.eps, nat.ptr(dq),
                nat.ptr(dk), nat.ptr(dwq), nat.ptr(dwk), ws_ptr, ws_size, nat.stream_ptr(dev)))
    if dwq is not None and dwq.dtype != wq.dtype:
        dwq = dwq.to(wq.dtype)
    if dwk is not None and dwk.dtype != wk.dtype:
        dwk = dwk.to(wk.dtype)
    return None, dq, None, dk, None, dwq, dwk


_qk_backward_once = torch.autograd.function.once_differentiable(_qk_backward)


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
    Weights have the operands' type or float32. Differentiable (once) in q, k and the weights.
    """
    op = "qk_norm_rope_with_tangent"
    (q, tq), (k, tk) = q_withT, k_withT
    _check_same_device(op, q, tq, k, tk, q_weight, k_weight, freqs)
    call = _QkCall()
    x, call.B, call.S, call.Hq, call.Hk, call.D = _qk_shapes(op, q, k)
    call.code, call.device = nat.dtype_code(x.dtype), x.device
    call.eps = float(eps)
    if not call.eps >= 0:
        raise ValueError(f"{op}: eps must be non-negative, got {eps}")
    if tq is not None or tk is not None:
        for y, t in ((q, tq), (k, tk)):
            if (y is None) != (t is None):
                raise ValueError(f"{op}: tangents of both q and k, or of neither")
            if t is not None and (t.shape != y.shape or t.dtype != y.dtype):
                raise ValueError(f"{op}: a tangent has its operand's shape and type")
    if (q is None and q_weight is not None) or (k is None and k_weight is not None):
        raise ValueError(f"{op}: a weight without its operand")
    # the weights' gradients are the operator's own
    call.wq, call.wk, call.wcode = _norm_weights(op, x, call.D, q_weight, k_weight)
    call.freqs, call.freqs_b = _angle_table(op, freqs, call.B, call.S, call.D)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, q_weight, k_weight)):
        q, tq, k, tk = _QkNormRope.apply(call, q, tq, k, tk, q_weight, k_weight)
    else:
        q, tq, k, tk = _qk_forward(call, q, tq, k, tk)[:4]
    return (q, tq), (k, tk)
