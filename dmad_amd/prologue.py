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

from typing import Optional, Tuple

import torch

from . import _native as nat
from .jvp_attention import _eager_call


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


def refuse_forward_mode(op, *ts):
    """Raises where one of ``ts`` carries a forward-mode tangent, which the kernels do not see and the result
    would lack."""
    if torch.compiler.is_compiling() or torch.autograd.forward_ad._current_level < 0:
        return
    if any(t is not None and torch.autograd.forward_ad.unpack_dual(t).tangent is not None for t in ts):
        raise NotImplementedError(f"{op} has no forward-mode derivative of torch's; tangents are operands of their own")


def _check_same_device(op, *ts):
    dev = None
    for t in ts:
        if t is None:
            continue
        d = t.device
        if d != dev:
            if d.type not in ("cuda", "meta"):
                raise RuntimeError(f"{op} runs on the GPU only (HIP kernel); got a tensor on {d}")
            if dev is not None:
                raise ValueError(f"{op}: tensors on {dev} and on {d}")
            dev = d
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


def _weights_dtype(op, x, D, wq, wk):
    """The one type in which the kernels take both weights: the operands' own or float32."""
    dtype = x.dtype
    for w in (wq, wk):
        if w is None:
            continue
        if w.dim() != 1 or w.shape[0] != D or w.dtype not in (torch.float32, torch.bfloat16, torch.float16):
            raise ValueError(f"{op}: weights must be [{D}] in the operands' type or float32, "
                             f"got {tuple(w.shape)} {w.dtype}")
        if w.dtype != dtype:
            dtype = torch.float32
    return dtype


def _weight_as_read(w, dtype):
    if w is None or w.dtype == dtype and w.is_contiguous() and not w.data_ptr() % 16:
        return w
    return torch.empty(w.shape, device=w.device, dtype=dtype).copy_(w.detach())


def _norm_weights(op, x, D, wq, wk):
    """(wq, wk, their type code) as the kernels take them."""
    dtype = _weights_dtype(op, x, D, wq, wk)
    return _weight_as_read(wq, dtype), _weight_as_read(wk, dtype), nat.dtype_code(dtype)


def _check_angles(op, freqs, B, S, D):
    if freqs is not None and (freqs.dim() not in (2, 3) or freqs.shape[-1] != D // 2 or freqs.shape[-2] != S or
                              (freqs.dim() == 3 and freqs.shape[0] not in (1, B))):
        raise ValueError(f"{op}: freqs must be [{S}, {D // 2}] or [{B}, {S}, {D // 2}], got {tuple(freqs.shape)}")


def _angle_table(freqs, B, S, D):
    """(float32 table, batch stride) of [S, D/2] or [B, S, D/2] angles."""
    if freqs is None:
        return None, 0
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

    def __init__(self, sizes, wq, wk, freqs, eps):
        x, self.B, self.S, self.Hq, self.Hk, self.D, wdtype = sizes
        self.code, self.device, self.eps = nat.dtype_code(x.dtype), x.device, eps
        # the weights' gradients are the operator's own
        self.wq, self.wk, self.wcode = _weight_as_read(wq, wdtype), _weight_as_read(wk, wdtype), nat.dtype_code(wdtype)
        self.freqs, self.freqs_b = _angle_table(freqs, self.B, self.S, self.D)


_QK = "qk_norm_rope_with_tangent"


def _qk_check(q, tq, k, tk, wq, wk, freqs, eps):
    """Refuses what the operator does not take; (an operand, B, S, Hq, Hk, D, the weights' type)."""
    op = _QK
    _check_same_device(op, q, tq, k, tk, wq, wk, freqs)
    x, B, S, Hq, Hk, D = _qk_shapes(op, q, k)
    nat.dtype_code(x.dtype)
    if not eps >= 0:
        raise ValueError(f"{op}: eps must be non-negative, got {eps}")
    if tq is not None or tk is not None:
        for y, t in ((q, tq), (k, tk)):
            if (y is None) != (t is None):
                raise ValueError(f"{op}: tangents of both q and k, or of neither")
            if t is not None and (t.shape != y.shape or t.dtype != y.dtype):
                raise ValueError(f"{op}: a tangent has its operand's shape and type")
    if (q is None and wq is not None) or (k is None and wk is not None):
        raise ValueError(f"{op}: a weight without its operand")
    wdtype = _weights_dtype(op, x, D, wq, wk)
    _check_angles(op, freqs, B, S, D)
    if freqs is not None and freqs.requires_grad and torch.is_grad_enabled():
        raise RuntimeError(f"{op} has no gradient of the angles: detach freqs")
    return x, B, S, Hq, Hk, D, wdtype


def _qk_forward(call, q, tq, k, tk):
    """The launch: (q', tq', k', tk') and q and k as they were read."""
    q, sq = _NOTHING if q is None else readable_rows(q)
    k, sk = _NOTHING if k is None else readable_rows(k)
    tq, stq = _NOTHING if tq is None else readable_rows(tq)
    tk, stk = _NOTHING if tk is None else readable_rows(tk)
    dev = call.device
    # (half the host time of torch.empty with a device and a type)
    oq, otq, ok, otk = (None if t is None else torch.empty_like(t, memory_format=torch.contiguous_format)
                        for t in (q, tq, k, tk))
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
    q, k, wq, wk, freqs = ctx.saved_tensors  # unpacked, so that a change in place is noticed
    call, need = ctx.call, ctx.needs_input_grad
    # an output whose gradient did not arrive adds nothing
    if gq is None and gk is None:
        return (None,) * 7
    if _eager_call(gq, gk):  # what was saved was read by an eager forward
        dq, dk, dwq, dwk = _qk_gradients(call, q, k, gq, gk, wq, wk, need[5], need[6])
    else:
        dq, dk, dwq, dwk = _qk_gradients_op(q, k, gq, gk, wq, wk, freqs, call.eps, need[5], need[6])
    return None, dq, None, dk, None, dwq, dwk


_qk_backward_once = torch.autograd.function.once_differentiable(_qk_backward)


def _check_saved(x, g):
    """The kernels read an operand as the forward did: one that came back from a saved-tensor hook in another
    shape, type or place is refused."""
    if g is not None and (x is None or x.shape != g.shape or x.dtype != g.dtype or x.device != g.device):
        got = "nothing" if x is None else f"{tuple(x.shape)} {x.dtype} on {x.device}"
        raise RuntimeError(f"{_QK}: the backward needs the operand of a gradient {tuple(g.shape)} {g.dtype} on "
                           f"{g.device} as the forward read it, got {got}")


def _qk_gradients(call, q, k, gq, gk, wq, wk, need_wq, need_wk):
    """The launch: (dq, dk, dwq, dwk), None where there is no gradient of that output or none is asked for."""
    _check_saved(q, gq)
    _check_saved(k, gk)
    cq, ck, Hq, Hk, dev = call.wq, call.wk, call.Hq, call.Hk, call.device
    sq = sgq = sk = sgk = dq = dk = dwq = dwk = ws = ws_ptr = None
    ws_size = 0
    if gq is not None:
        q, sq = readable_rows(q)
        gq, sgq = readable_rows(gq)
        dq = torch.empty_like(q, memory_format=torch.contiguous_format)
        if cq is not None and need_wq:
            dwq = torch.empty_like(cq)
    else:
        q, cq, Hq = None, None, 0
    if gk is not None:
        k, sk = readable_rows(k)
        gk, sgk = readable_rows(gk)
        dk = torch.empty_like(k, memory_format=torch.contiguous_format)
        if ck is not None and need_wk:
            dwk = torch.empty_like(ck)
    else:
        k, ck, Hk = None, None, 0
    tokens = call.B * call.S
    # without rows a weight's gradient is zero, and the kernels are not asked for it
    ask_q, ask_k = dwq, dwk
    if dwq is not None and tokens * Hq == 0:
        ask_q, cq = None, None
        dwq.zero_()
    if dwk is not None and tokens * Hk == 0:
        ask_k, ck = None, None
        dwk.zero_()
    if tokens * (Hq + Hk):
        if ask_q is not None or ask_k is not None:
            ws_ptr, ws_size, ws = nat.workspace(
                nat.qk_norm_rope_bwd_workspace_bytes(call.B, call.S, Hq, Hk, call.D), dev)
        with nat.on_device(dev):
            nat.check(nat.lib().dmad_qk_norm_rope_bwd(
                call.code, call.wcode, call.B, call.S, Hq, Hk, call.D, nat.ptr(q), nat.ptr(gq), nat.ptr(k), nat.ptr(gk),
                sq, sgq, sk, sgk, nat.ptr(cq), nat.ptr(ck), nat.ptr(call.freqs), call.freqs_b, call.eps, nat.ptr(dq),
                nat.ptr(dk), nat.ptr(ask_q), nat.ptr(ask_k), ws_ptr, ws_size, nat.stream_ptr(dev)))
    if dwq is not None and dwq.dtype != wq.dtype:
        dwq = dwq.to(wq.dtype)
    if dwk is not None and dwk.dtype != wk.dtype:
        dwk = dwk.to(wk.dtype)
    return dq, dk, dwq, dwk


# The same as registered ops, for whatever watches or replaces operators (compilers, dispatch modes, the profiler)
# and for operands whose memory does not hold their values. What is absent comes back with 0 elements.
def _or_empty(x, ts):
    return tuple(x.new_empty((0,)) if t is None else t for t in ts)


@torch.library.custom_op("dmad::qk_norm_rope_fwd", mutates_args=())
def qk_norm_rope_fwd(q: Optional[torch.Tensor], tq: Optional[torch.Tensor], k: Optional[torch.Tensor],
                     tk: Optional[torch.Tensor], wq: Optional[torch.Tensor], wk: Optional[torch.Tensor],
                     freqs: Optional[torch.Tensor],
                     eps: float) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """(q', tq', k', tk') of ``qk_norm_rope_with_tangent``."""
    call = _QkCall(_qk_check(q, tq, k, tk, wq, wk, freqs, eps), wq, wk, freqs, eps)
    return _or_empty(k if q is None else q, _qk_forward(call, q, tq, k, tk)[:4])


@qk_norm_rope_fwd.register_fake
def _(q, tq, k, tk, wq, wk, freqs, eps):
    return _or_empty(k if q is None else q, (None if t is None else t.new_empty(t.shape) for t in (q, tq, k, tk)))


@torch.library.custom_op("dmad::qk_norm_rope_bwd", mutates_args=())
def qk_norm_rope_bwd(q: Optional[torch.Tensor], k: Optional[torch.Tensor], gq: Optional[torch.Tensor],
                     gk: Optional[torch.Tensor], wq: Optional[torch.Tensor], wk: Optional[torch.Tensor],
                     freqs: Optional[torch.Tensor], eps: float, need_wq: bool,
                     need_wk: bool) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """(dq, dk, dwq, dwk) of qk_norm_rope_fwd over its primal outputs' gradients, of which one may be absent."""
    call = _QkCall(_qk_check(q, None, k, None, wq, wk, freqs, eps), wq, wk, freqs, eps)
    return _or_empty(k if q is None else q, _qk_gradients(call, q, k, gq, gk, wq, wk, need_wq, need_wk))


@qk_norm_rope_bwd.register_fake
def _(q, k, gq, gk, wq, wk, freqs, eps, need_wq, need_wk):
    outs = [(q, gq is not None), (k, gk is not None), (wq, need_wq and gq is not None), (wk, need_wk and gk is not None)]
    return _or_empty(k if q is None else q, (t.new_empty(t.shape) if t is not None and there else None for t, there in outs))


def _qk_gradients_op(q, k, gq, gk, wq, wk, freqs, eps, need_wq, need_wk):
    """(dq, dk, dwq, dwk) by the registered op, None where there is none."""
    need_wq, need_wk = need_wq and wq is not None and gq is not None, need_wk and wk is not None and gk is not None
    outs = torch.ops.dmad.qk_norm_rope_bwd(q, k, gq, gk, wq, wk, freqs, eps, need_wq, need_wk)
    there = (gq is not None, gk is not None, need_wq, need_wk)
    return tuple(t if y else None for t, y in zip(outs, there))


def _qk_setup_context(ctx, inputs, output):
    q, _, k, _, wq, wk, freqs, ctx.eps = inputs
    ctx.save_for_backward(q, k, wq, wk, freqs)
    ctx.set_materialize_grads(False)


def _qk_op_backward(ctx, gq, _gtq, gk, _gtk):
    q, k, wq, wk, freqs = ctx.saved_tensors
    # the gradient of an absent operand's 0-element output is none
    gq, gk, need = None if q is None else gq, None if k is None else gk, ctx.needs_input_grad
    if gq is None and gk is None:
        return (None,) * 8
    dq, dk, dwq, dwk = _qk_gradients_op(q, k, gq, gk, wq, wk, freqs, ctx.eps, need[4], need[5])
    return dq, None, dk, None, dwq, dwk, None, None


qk_norm_rope_fwd.register_autograd(_qk_op_backward, setup_context=_qk_setup_context)


def qk_norm_rope_with_tangent(q_withT, k_withT, q_weight, k_weight, eps, freqs):
    """RMSNorm of queries and keys for each head and their rotation, in one pass over both.

    ``((q, tq), (k, tk), wq [D], wk [D], eps, freqs) -> ((q', tq'), (k', tk'))`` for q [B, S, Hq, D]
    and k [B, S, Hk, D] (any head counts; bf16, fp16 or fp32; D in 16, 32, 64, 128, 256; any strides
    with contiguous 16-byte-aligned rows are read in place). Each head's row x becomes
    R(x / sqrt(mean(x^2) + eps) * w), R turning the pairs (x[2i], x[2i+1]) by freqs[s, i] as
    ``apply_rope_with_tangent`` does; float32 throughout, rounded once at the end (rows whose squares
    leave float32, elements above about 1e18 or, where eps is 0, below 1e-19, are not scaled first).
    This is the norm per head; ``rmsnorm_rope_with_tangent`` is the one over the whole model width.

    ``tq``/``tk``: tangents, given for both or for neither; their outputs are detached. ``k_withT``
    (or ``q_withT``) may be ``(None, None)``: the other alone. A weight of None skips that norm,
    ``freqs`` None the rotation; freqs are [S, D/2], or [B, S, D/2] for angles per sequence.
    Weights have the operands' type or float32. Differentiable (once) in q, k and the weights;
    angles that require a gradient and torch's own forward-mode tangents are refused.
    """
    (q, tq), (k, tk) = q_withT, k_withT
    eps = float(eps)
    eager = _eager_call(q, tq, k, tk, q_weight, k_weight, freqs)
    if not eager:
        refuse_forward_mode(_QK, q, tq, k, tk, q_weight, k_weight, freqs)
    sizes = _qk_check(q, tq, k, tk, q_weight, k_weight, freqs, eps)
    if not eager:
        tq, tk = (None if t is None else t.detach() for t in (tq, tk))
        outs = torch.ops.dmad.qk_norm_rope_fwd(q, tq, k, tk, q_weight, k_weight, freqs, eps)
        q, tq, k, tk = (None if t is None else y for t, y in zip((q, tq, k, tk), outs))
        return (q, None if tq is None else tq.detach()), (k, None if tk is None else tk.detach())
    call = _QkCall(sizes, q_weight, k_weight, freqs, eps)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, q_weight, k_weight)):
        q, tq, k, tk = _QkNormRope.apply(call, q, tq, k, tk, q_weight, k_weight)
    else:
        q, tq, k, tk = _qk_forward(call, q, tq, k, tk)[:4]
    return (q, tq), (k, tk)
