"""Operators around a block's attention for gfx950: gate, residual and norm in one pass, and rotations by position.

``gated_residual_norm_with_tangent`` is what stands between two parts of a transformer block: the branch's output is
gated (and, where the block has one, normed) and added to the residual stream, and the sum is normed, scaled and shifted
for the next part. The reference writes it out in its blocks
(train/wan/rcm/networks/wan2pt1_jvp.py:551-609, under ``torch.func.jvp``). ``qk_rotary_with_tangent`` turns queries and
keys by positions rather than by a table of angles: neighbours or halves of a head, the whole head or its first part, with
frequencies from ``rotary_frequencies``. Both take ``(x, x_dot)`` pairs and have a backward.
Device work only: tensors off the GPU raise.
"""
from __future__ import annotations

import ctypes
import math
from typing import List, Optional, Tuple

import torch

from . import _native as nat
from .jvp_attention import _eager_call
from .prologue import _check_same_device, _or_empty, refuse_forward_mode

_GN = "gated_residual_norm_with_tangent"
_NORMS = {"layer": 0, "rms": 1}
MAX_CHANNELS = 8192


def _strides3(t):
    """Strides of a [B, S, C] operand as the kernels take them (an axis of one element is never stepped along), None where
    its rows are not contiguous or not a multiple of 16 bytes apart."""
    (b, s, _), (sb, ss, sc) = t.shape, t.stride()
    sb, ss, step = 0 if b == 1 else sb, 0 if s == 1 else ss, 16 // t.element_size()
    return None if sc != 1 or sb % step or ss % step else (sb, ss, 1)


def _readable3(t):
    """(tensor, strides): ``t`` itself where the kernels read it in place, else a contiguous copy."""
    st = _strides3(t)
    if st is None or t.data_ptr() % 16:
        t = t.clone(memory_format=torch.contiguous_format)
        st = _strides3(t)
    return t, st


def _small_as_read(t, dtype):
    """A vector as the kernels take it: in the one type of all of them, rows readable in place."""
    if t is None or (t.dtype == dtype and t.stride(-1) == 1 and not t.data_ptr() % 16 and (t.dim() == 1 or _strides3(t))):
        return t
    return torch.empty(t.shape, device=t.device, dtype=dtype).copy_(t.detach())


_SMALL = ("gate", "scale", "shift")
_PER_CHANNEL = ("weight", "bias", "post_weight")


class _NormPlan:
    """What the sizes, types and strides of a call's operands settle, made once for them."""

    __slots__ = ("device", "B", "S", "C", "F", "code", "wcode", "dtype", "norm", "small", "in_place", "group_strides",
                 "dense", "forward_sizes", "backward_sizes", "workspace")

    def __init__(self, checked, norm, operands):
        x, self.F, self.dtype = checked
        self.B, self.S, self.C = x.shape
        self.device, self.code, self.wcode = x.device, nat.dtype_code(x.dtype), nat.dtype_code(self.dtype)
        self.norm, self.backward_sizes, self.workspace = _NORMS[norm], {}, {}
        # strides of a contiguous operand
        self.dense = (0 if self.B == 1 else self.S * self.C, 0 if self.S == 1 else self.C, 1)
        # gate, scale, shift, weight, bias and post_weight
        self.small = [None if t is None else (t.shape, t.dtype, t.stride()) for t in (*operands[4:10:2], *operands[10:])]
        # whether the kernels read every operand where it lies, if it starts aligned
        strides = [None if t is None else _strides3(t) for t in operands[:10]]
        self.in_place = all(t is None or st is not None for t, st in zip(operands, strides)) and all(
            t is None or t.dtype == self.dtype and (i < 10 or t.stride(0) == 1) for i, t in enumerate(operands) if i >= 4)
        self.forward_sizes = self.group_strides = None
        if self.in_place:
            x, tx, y, ty, gate, tgate, scale, tscale, shift, tshift = strides
            self.group_strides = gate, scale, shift
            self.forward_sizes = self.sizes(x, y, tx, ty, gate, scale, shift, tgate, tscale, tshift)

    def readable(self, t):
        """``_readable3`` of an operand [B, S, C] or None."""
        if t is None:
            return None, None
        return (t, self.dense) if t.is_contiguous() and not t.data_ptr() & 15 else _readable3(t)

    def sizes(self, *strides):
        """``dmad_gated_norm_sizes`` of these strides, for ctypes."""
        none = (0, 0, 1)
        return ctypes.byref(nat.GatedNormSizes(self.code, self.wcode, self.norm, self.B, self.S, self.C, self.F,
                                               *((ctypes.c_int64 * 3)(*(none if s is None else s)) for s in strides)))

    def sizes_back(self, *strides):
        found = self.backward_sizes.get(strides)
        if found is None:
            if len(self.backward_sizes) > 64:
                self.backward_sizes.clear()
            found = self.backward_sizes[strides] = self.sizes(*strides, None, None, None)
        return found


class _NormCall:
    """What a forward or a backward launch goes by: the plan, and the small operands as the kernels take them."""

    __slots__ = ("plan", "in_place", "eps", "residual_scale", *_SMALL, *_PER_CHANNEL)

    def __init__(self, plan, in_place, gate, scale, shift, weight, bias, post_weight, eps, residual_scale):
        self.plan, self.in_place, self.eps, self.residual_scale = plan, in_place, eps, residual_scale
        if not in_place:
            gate, scale, shift, weight, bias, post_weight = (_small_as_read(t, plan.dtype) for t in
                                                             (gate, scale, shift, weight, bias, post_weight))
        self.gate, self.scale, self.shift = gate, scale, shift
        self.weight, self.bias, self.post_weight = weight, bias, post_weight


# plans by what they are made from
_norm_plans: dict = {}


def _norm_check(x, tx, y, ty, gate, tgate, scale, tscale, shift, tshift, weight, bias, post_weight, eps, norm, residual_scale):
    """Refuses what the operator does not take; (x, groups of tokens, the small operands' type)."""
    op = _GN
    if x is None:
        raise ValueError(f"{op}: x must be given")
    _check_same_device(op, x, tx, y, ty, gate, tgate, scale, tscale, shift, tshift, weight, bias, post_weight)
    if x.dim() != 3:
        raise ValueError(f"{op}: x must be [B, S, C], got {tuple(x.shape)}")
    nat.dtype_code(x.dtype)
    B, S, C = x.shape
    if C % 8 or not 8 <= C <= MAX_CHANNELS:
        raise NotImplementedError(f"{op}: channels must be a multiple of 8 up to {MAX_CHANNELS}, got {C}")
    if norm not in _NORMS:
        raise ValueError(f"{op}: norm must be one of {tuple(_NORMS)}, got {norm!r}")
    if not (eps >= 0 and math.isfinite(eps)):
        raise ValueError(f"{op}: eps must be non-negative and finite, got {eps}")
    if not math.isfinite(residual_scale):
        raise ValueError(f"{op}: residual_scale must be finite, got {residual_scale}")
    if y is not None and (y.shape != x.shape or y.dtype != x.dtype):
        raise ValueError(f"{op}: y must have x's shape and type, got {tuple(y.shape)} {y.dtype}")
    if y is None and (gate is not None or post_weight is not None):
        raise ValueError(f"{op}: gate and post_weight belong to y, which is absent")
    if (ty is not None) != (tx is not None and y is not None):
        raise ValueError(f"{op}: tangents of both x and y, or of neither")
    for name, t, tt in (("x", x, tx), ("y", y, ty), ("gate", gate, tgate), ("scale", scale, tscale), ("shift", shift, tshift)):
        if tt is None:
            continue
        if t is None or tx is None:
            raise ValueError(f"{op}: a tangent of {name} without " + ("it" if t is None else "one of x"))
        if tt.shape != t.shape or (tt.dtype != t.dtype and name in ("x", "y")):
            raise ValueError(f"{op}: a tangent has its operand's shape and type")
    F, dtype = 0, x.dtype
    for name, t in (("gate", gate), ("scale", scale), ("shift", shift), ("gate", tgate), ("scale", tscale), ("shift", tshift)):
        if t is None:
            continue
        if t.dim() != 3 or t.shape[0] != B or t.shape[2] != C or t.shape[1] < 1 or S % t.shape[1] or (F > 0 and F != t.shape[1]):
            raise ValueError(f"{op}: gate, scale and shift must be [{B}, F, {C}] with one F that divides {S}, got {name} "
                             f"{tuple(t.shape)}")
        F = t.shape[1]
        dtype = _small_type(op, name, t, dtype)
    for name, t in (("weight", weight), ("bias", bias), ("post_weight", post_weight)):
        if t is None:
            continue
        if t.shape != (C,):
            raise ValueError(f"{op}: {name} must be [{C}], got {tuple(t.shape)}")
        dtype = _small_type(op, name, t, dtype)
    return x, F or 1, dtype


def _small_type(op, name, t, dtype):
    if t.dtype not in (torch.float32, torch.bfloat16, torch.float16):
        raise ValueError(f"{op}: {name} must be in the operands' type or float32, got {t.dtype}")
    return dtype if t.dtype == dtype else torch.float32


def _norm_plan(tensors, eps, norm, residual_scale):
    """The plan of an ordinary call's operands; what the operator does not take is refused."""
    key = (norm, *(None if t is None else (t.shape, t.stride(), t.dtype, t.device) for t in tensors))
    plan = _norm_plans.get(key)
    # (the two numbers are not part of the key)
    if plan is None or not (0 <= eps < math.inf) or not math.isfinite(residual_scale):
        checked = _norm_check(*tensors, eps, norm, residual_scale)
        if len(_norm_plans) > 1024:
            _norm_plans.clear()
        plan = _norm_plans[key] = _NormPlan(checked, norm, tensors)
    return plan


def _norm_forward(call, x, tx, y, ty, tgate, tscale, tshift):
    """The launch: (x', tx', n, tn) and x and y as they were read."""
    plan, ptr = call.plan, nat.ptr
    if call.in_place:
        sizes = plan.forward_sizes
    else:
        (x, sx), (tx, stx), (y, sy), (ty, sty) = map(plan.readable, (x, tx, y, ty))
        tgate, tscale, tshift = (None if t is None else _small_as_read(t, plan.dtype) for t in (tgate, tscale, tshift))
        sizes = plan.sizes(sx, sy, stx, sty, *(None if t is None else _strides3(t) for t in
                                               (call.gate, call.scale, call.shift, tgate, tscale, tshift)))
    n = torch.empty_like(x, memory_format=torch.contiguous_format)
    tn = None if tx is None else torch.empty_like(n)
    xo = None if y is None else torch.empty_like(n)
    txo = None if ty is None else torch.empty_like(n)
    with nat.on_device(plan.device):
        nat.check(nat.lib().dmad_gated_norm(
            sizes, ptr(x), ptr(tx), ptr(y), ptr(ty), ptr(call.gate), ptr(tgate), ptr(call.scale), ptr(tscale),
            ptr(call.shift), ptr(tshift), ptr(call.weight), ptr(call.bias), ptr(call.post_weight), call.eps,
            call.residual_scale, ptr(xo), ptr(txo), ptr(n), ptr(tn), nat.stream_ptr(plan.device)))
    return xo, txo, n, tn, x, y


def _check_norm_saved(t, g):
    """The kernels read an operand as the forward did: one that came back from a saved-tensor hook in another shape, type
    or place is refused."""
    if t is None or t.shape != g.shape or t.dtype != g.dtype or t.device != g.device:
        got = "nothing" if t is None else f"{tuple(t.shape)} {t.dtype} on {t.device}"
        raise RuntimeError(f"{_GN}: the backward needs the operand of a gradient {tuple(g.shape)} {g.dtype} on "
                           f"{g.device} as the forward read it, got {got}")


def _saved_call(plan, small, eps, residual_scale):
    """The call of a backward, from the saved small operands, which are those that the plan was made from: one that came
    back in another shape, type or place is refused, and one that lies otherwise is copied (what was absent stays so)."""
    in_place = plan.in_place
    for t, want in zip(small, plan.small):
        if want is None:
            continue
        if t is None or t.dtype != want[1] or t.shape != want[0] or t.device != plan.device:
            got = "nothing" if t is None else f"{tuple(t.shape)} {t.dtype} on {t.device}"
            raise RuntimeError(f"{_GN}: the backward needs a small operand as the forward read it, got {got}")
        in_place = in_place and t.stride() == want[2] and not t.data_ptr() & 15
    return _NormCall(plan, in_place, *small, eps, residual_scale)


def _norm_gradients(call, x, y, gx, gn, originals, need):
    """The launch: gradients of (x, y, gate, scale, shift, weight, bias, post_weight), None where none is asked for.
    ``originals``: the small operands as the caller has them; ``need``: which of the eight are wanted."""
    g = gn if gx is None else gx
    _check_norm_saved(x, g)
    if y is not None or call.gate is not None or call.post_weight is not None:
        _check_norm_saved(y, g)
    plan, ptr = call.plan, nat.ptr
    (x, sx), (y, sy), (gx, sgx), (gn, sgn) = map(plan.readable, (x, y, gx, gn))
    dx = torch.empty_like(x, memory_format=torch.contiguous_format)
    dy = torch.empty_like(dx) if need[1] and y is not None else None
    shape, dtype = (plan.B, plan.F, plan.C), plan.dtype
    as_read = (call.gate, call.scale, call.shift, call.weight, call.bias, call.post_weight)
    small = [None if t is None or not n else dx.new_empty(shape if i < 3 else shape[2:], dtype=dtype)
             for i, (t, n) in enumerate(zip(as_read, need[2:]))]
    if x.numel() == 0:
        for t in small:
            if t is not None:
                t.zero_()
    else:
        groups = plan.group_strides if call.in_place else (None if t is None else _strides3(t) for t in as_read[:3])
        sizes = plan.sizes_back(sx, sy, sgx, sgn, *groups)
        ws_ptr, ws_size, ws = None, 0, None
        per_channel = not (small[3] is None and small[4] is None and small[5] is None)
        if per_channel or not (small[0] is None and small[1] is None and small[2] is None):
            size = plan.workspace.get(per_channel)
            if size is None:
                n = ctypes.c_size_t(0)
                nat.check(nat.lib().dmad_gated_norm_bwd_workspace_bytes_for(sizes, per_channel, ctypes.byref(n)))
                size = plan.workspace[per_channel] = n.value
            ws_ptr, ws_size, ws = nat.workspace(size, plan.device)
        with nat.on_device(plan.device):
            nat.check(nat.lib().dmad_gated_norm_bwd(
                sizes, ptr(x), ptr(y), ptr(gx), ptr(gn), ptr(call.gate), ptr(call.scale), ptr(call.weight), ptr(call.bias),
                ptr(call.post_weight), call.eps, call.residual_scale, ptr(dx), ptr(dy), *map(ptr, small), ws_ptr, ws_size,
                nat.stream_ptr(plan.device)))
    small = [t if t is None or t.dtype == o.dtype else t.to(o.dtype) for t, o in zip(small, originals)]
    return (dx, dy, *small)


class _GatedNorm(torch.autograd.Function):
    """(call, x, tx, y, ty, gate, tgate, scale, tscale, shift, tshift, weight, bias, post_weight) -> (x', tx', n, tn);
    gradients of the primal outputs."""

    @staticmethod
    def forward(ctx, call, x, tx, y, ty, gate, tgate, scale, tscale, shift, tshift, weight, bias, post_weight):
        xo, txo, n, tn, x, y = _norm_forward(call, x, tx, y, ty, tgate, tscale, tshift)
        # no operand is kept but by its saved tensor, which hooks may move and the backward frees
        ctx.save_for_backward(x, y, gate, scale, shift, weight, bias, post_weight)
        ctx.plan, ctx.eps, ctx.residual_scale = call.plan, call.eps, call.residual_scale
        ctx.set_materialize_grads(False)
        tangents = [t for t in (txo, tn) if t is not None]
        if tangents:
            ctx.mark_non_differentiable(*tangents)
        return xo, txo, n, tn

    @staticmethod
    def backward(ctx, gx, _gtx, gn, _gtn):
        # a backward that is itself recorded (create_graph) must refuse to be differentiated
        if torch.is_grad_enabled():
            return _norm_backward_once(ctx, gx, gn)
        return _norm_backward(ctx, gx, gn)


def _spread(grads):
    """The eight gradients at the places of their operands in the op's order, tangents between."""
    dx, dy, dgate, dscale, dshift, dweight, dbias, dpost = grads
    return dx, None, dy, None, dgate, None, dscale, None, dshift, None, dweight, dbias, dpost


def _needed(ctx, first):
    """Which of the eight gradients are asked for; ``first`` is x's place among the operands."""
    need = ctx.needs_input_grad[first:]
    return [need[0], need[2], need[4], need[6], need[8], need[10], need[11], need[12]]


def _norm_backward(ctx, gx, gn):
    x, y, *small = ctx.saved_tensors
    if gx is None and gn is None:
        return (None,) * 14
    plan, eps, residual_scale, need = ctx.plan, ctx.eps, ctx.residual_scale, _needed(ctx, 1)
    if _eager_call(gx, gn, x, y, *small):
        call = _saved_call(plan, small, eps, residual_scale)
        grads = _norm_gradients(call, x, y, gx, gn, small, need)
    else:
        grads = _norm_gradients_op(x, y, gx, gn, *small, eps, plan.norm == 1, residual_scale, need)
    return (None, *_spread(grads))


_norm_backward_once = torch.autograd.function.once_differentiable(_norm_backward)


# The same as registered ops, for whatever watches or replaces operators (compilers, dispatch modes, the profiler)
# and for operands whose memory does not hold their values. What is absent comes back with 0 elements.
@torch.library.custom_op("dmad::gated_norm_fwd", mutates_args=())
def gated_norm_fwd(x: torch.Tensor, tx: Optional[torch.Tensor], y: Optional[torch.Tensor], ty: Optional[torch.Tensor],
                   gate: Optional[torch.Tensor], tgate: Optional[torch.Tensor], scale: Optional[torch.Tensor],
                   tscale: Optional[torch.Tensor], shift: Optional[torch.Tensor], tshift: Optional[torch.Tensor],
                   weight: Optional[torch.Tensor], bias: Optional[torch.Tensor], post_weight: Optional[torch.Tensor],
                   eps: float, rms: bool,
                   residual_scale: float) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """(x', tx', n, tn) of ``gated_residual_norm_with_tangent``."""
    norm = "rms" if rms else "layer"
    tensors = (x, tx, y, ty, gate, tgate, scale, tscale, shift, tshift, weight, bias, post_weight)
    plan = _NormPlan(_norm_check(*tensors, eps, norm, residual_scale), norm, tensors)
    call = _NormCall(plan, False, gate, scale, shift, weight, bias, post_weight, eps, residual_scale)
    return _or_empty(x, _norm_forward(call, x, tx, y, ty, tgate, tscale, tshift)[:4])


@gated_norm_fwd.register_fake
def _(x, tx, y, ty, gate, tgate, scale, tscale, shift, tshift, weight, bias, post_weight, eps, rms, residual_scale):
    return _or_empty(x, (None if t is None else x.new_empty(x.shape) for t in (y, ty, x, tx)))


@torch.library.custom_op("dmad::gated_norm_bwd", mutates_args=())
def gated_norm_bwd(x: torch.Tensor, y: Optional[torch.Tensor], gx: Optional[torch.Tensor], gn: Optional[torch.Tensor],
                   gate: Optional[torch.Tensor], scale: Optional[torch.Tensor], shift: Optional[torch.Tensor],
                   weight: Optional[torch.Tensor], bias: Optional[torch.Tensor], post_weight: Optional[torch.Tensor],
                   eps: float, rms: bool, residual_scale: float,
                   need: List[bool]) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor,
                                              torch.Tensor, torch.Tensor, torch.Tensor]:
    """Gradients of (x, y, gate, scale, shift, weight, bias, post_weight) over those of the primal outputs, of which one
    may be absent."""
    norm = "rms" if rms else "layer"
    tensors = (x, None, y, None, gate, None, scale, None, shift, None, weight, bias, post_weight)
    plan = _NormPlan(_norm_check(*tensors, eps, norm, residual_scale), norm, tensors)
    if gx is None and gn is None:
        raise ValueError(f"{_GN}: the gradient of neither output")
    for g in (gx, gn):
        if g is not None:
            _check_norm_saved(x, g)
    call = _NormCall(plan, False, gate, scale, shift, weight, bias, post_weight, eps, residual_scale)
    return _or_empty(x, _norm_gradients(call, x, y, gx, gn, (gate, scale, shift, weight, bias, post_weight), need))


@gated_norm_bwd.register_fake
def _(x, y, gx, gn, gate, scale, shift, weight, bias, post_weight, eps, rms, residual_scale, need):
    ts = (x, y, gate, scale, shift, weight, bias, post_weight)
    return _or_empty(x, (t.new_empty(t.shape) if t is not None and (n or i == 0) else None for i, (t, n) in enumerate(zip(ts, need))))


def _norm_gradients_op(x, y, gx, gn, gate, scale, shift, weight, bias, post_weight, eps, rms, residual_scale, need):
    """The eight gradients by the registered op, None where there is none."""
    outs = torch.ops.dmad.gated_norm_bwd(x, y, gx, gn, gate, scale, shift, weight, bias, post_weight, eps, rms,
                                         residual_scale, need)
    ts = (x, y, gate, scale, shift, weight, bias, post_weight)
    return tuple(o if t is not None and n else None for o, t, n in zip(outs, ts, need))


def _norm_setup_context(ctx, inputs, output):
    x, _, y, _, gate, _, scale, _, shift, _, weight, bias, post_weight, *ctx.rest = inputs
    ctx.save_for_backward(x, y, gate, scale, shift, weight, bias, post_weight)
    ctx.set_materialize_grads(False)


def _norm_op_backward(ctx, gx, _gtx, gn, _gtn):
    x, y, *small = ctx.saved_tensors
    gx = None if y is None else gx  # the gradient of an absent output's 0 elements is none
    if gx is None and gn is None:
        return (None,) * 16
    grads = _norm_gradients_op(x, y, gx, gn, *small, *ctx.rest, _needed(ctx, 0))
    return (*_spread(grads), None, None, None)


gated_norm_fwd.register_autograd(_norm_op_backward, setup_context=_norm_setup_context)


def gated_residual_norm_with_tangent(x_withT, y_withT=(None, None), gate_withT=(None, None), scale_withT=(None, None),
                                     shift_withT=(None, None), weight=None, bias=None, post_weight=None, eps=1e-6,
                                     norm="layer", residual_scale=1.0):
    """Gate, residual and the next norm in one pass: ``((x', tx'), (n, tn))``.

    ``y' = y``, or ``y / sqrt(mean(y^2) + eps) * post_weight`` where the block has a norm after it;
    ``x' = x + residual_scale * gate * y'``;
    ``n = (N(x') * weight + bias) * (1 + scale) + shift`` with N the layer norm or the RMS norm over the channels.

    x, y: [B, S, C], C a multiple of 8 up to 8192, bf16, fp16 or fp32; any strides with contiguous 16-byte-aligned rows
    are read in place. ``y_withT`` (None, None): there is no branch, and x and its tangent come back as they are. gate,
    scale, shift: [B, F, C], one row for S / F consecutive tokens (F = 1: one per sequence, the latent frames of a clip,
    S: one per token; expand what is shared); weight, bias, post_weight: [C]. Any of them may be None. They have the
    operands' type or float32; types that differ among them are read as float32 copies. Computed in float32 and rounded
    once: n is the norm of x' as computed, not as rounded (rows whose squares leave float32 are not scaled first).

    Tangents: of x and y both or of neither, then also of gate, scale and shift where they are not zero; tangent outputs
    are detached. Differentiable (once) in x, y and the small operands, whose gradients are summed in a fixed order;
    torch's own forward-mode tangents are refused. The backward's scratch is 12 C bytes per workgroup, of which a
    group of tokens has one or more; none where it has one, as with a row per token, and no gradient of weight, bias or
    post_weight is wanted.
    """
    (x, tx), (y, ty), (gate, tgate), (scale, tscale), (shift, tshift) = x_withT, y_withT, gate_withT, scale_withT, shift_withT
    eps, residual_scale = float(eps), float(residual_scale)
    tensors = (x, tx, y, ty, gate, tgate, scale, tscale, shift, tshift, weight, bias, post_weight)
    if not _eager_call(*tensors):
        refuse_forward_mode(_GN, *tensors)
        _norm_check(*tensors, eps, norm, residual_scale)
        detached = [t if t is None or i % 2 == 0 or i > 9 else t.detach() for i, t in enumerate(tensors)]
        xo, txo, n, tn = torch.ops.dmad.gated_norm_fwd(*detached, eps, norm == "rms", residual_scale)
        txo, tn = (None if t is None else o.detach() for t, o in ((ty, txo), (tx, tn)))
    else:
        plan = _norm_plan(tensors, eps, norm, residual_scale)
        in_place = plan.in_place and not any(t is not None and t.data_ptr() & 15 for t in tensors)
        call = _NormCall(plan, in_place, gate, scale, shift, weight, bias, post_weight, eps, residual_scale)
        if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in
                                           (x, y, gate, scale, shift, weight, bias, post_weight)):
            xo, txo, n, tn = _GatedNorm.apply(call, *tensors)
        else:
            xo, txo, n, tn, _, _ = _norm_forward(call, x, tx, y, ty, tgate, tscale, tshift)
    return ((x, tx) if y is None else (xo, txo)), (n, tn)


# ---------------------------------------------------------------- rotations by position

_QR = "qk_rotary_with_tangent"
_LAYOUTS = {"interleaved": 0, "half": 1}


def rotary_frequencies(dim, theta=10000.0, scaling=None, factor=1.0, trained_length=None, fast=32.0, slow=1.0, device="cuda"):
    """``(frequencies [dim / 2] float64, factor of sines and cosines)`` for ``qk_rotary_with_tangent``.

    Frequency i is theta^(-2i / dim) radians per position. For contexts ``factor`` times the trained one:
      * scaling "linear": positions are interpolated, every frequency divided by ``factor``;
      * "ntk": theta is multiplied by factor^(dim / (dim - 2)), which divides the lowest frequency by ``factor`` and leaves
        the highest as it is;
      * "yarn": frequencies that make at least ``fast`` turns over ``trained_length`` positions stay, those that make at
        most ``slow`` are divided by ``factor``, those between are blended linearly in their turns; sines and cosines are
        multiplied by 0.1 ln(factor) + 1. (Some programs blend linearly in i between the two instead: weights trained so
        need that table, which ``qk_rotary_with_tangent`` takes like any other.)
    """
    op = "rotary_frequencies"
    if dim < 2 or dim % 2:
        raise ValueError(f"{op}: dim must be even and at least 2, got {dim}")
    if not (theta > 0 and math.isfinite(theta)) or not (factor > 0 and math.isfinite(factor)):
        raise ValueError(f"{op}: theta and factor must be positive and finite, got {theta} and {factor}")
    if scaling == "ntk":
        if dim < 4:
            raise ValueError(f"{op}: ntk needs at least two frequencies")
        theta = theta * factor ** (dim / (dim - 2))
    freqs = float(theta) ** (torch.arange(dim // 2, dtype=torch.float64) * (-2.0 / dim))
    by = 1.0
    if scaling == "linear":
        freqs = freqs / factor
    elif scaling == "yarn":
        if trained_length is None or trained_length < 1 or not fast > slow:
            raise ValueError(f"{op}: yarn needs trained_length >= 1 and fast > slow, got {trained_length}, {fast}, {slow}")
        keep = ((trained_length * freqs / (2 * math.pi) - slow) / (fast - slow)).clamp(0, 1)
        freqs, by = freqs * (keep + (1 - keep) / factor), 0.1 * math.log(factor) + 1
    elif scaling not in (None, "ntk"):
        raise ValueError(f"{op}: scaling must be None, 'linear', 'ntk' or 'yarn', got {scaling!r}")
    return freqs.to(device), by


class _RotaryCall:
    """What a forward or a backward launch goes by: sizes, and the positions and frequencies as the kernels take them."""

    __slots__ = ("sizes", "positions", "pos_strides", "frequencies", "layout", "factor")

    def __init__(self, sizes, positions, pos_strides, frequencies, layout, factor):
        self.sizes, self.positions, self.pos_strides, self.layout, self.factor = sizes, positions, pos_strides, layout, factor
        self.frequencies = frequencies if frequencies.is_contiguous() else frequencies.contiguous()


# the sizes of a _RotaryCall by shapes, types and strides of its operands: (device, type code, B, S, D, R, whether positions have
# 64 bits, their strides for ctypes, (shape, type and strides of positions, shape of frequencies))
_rotary_sizes: dict = {}


def _rotary_plan(q, tq, k, tk, positions, frequencies, layout, factor):
    """The sizes of an ordinary call's operands; what the operator does not take is refused."""
    tensors = (q, tq, k, tk, positions, frequencies)
    key = (layout, *(None if t is None else (t.shape, t.dtype, t.device) for t in tensors),
           None if positions is None else positions.stride())
    sizes = _rotary_sizes.get(key)
    # (the factor and whether a gradient is wanted are not part of the key)
    if sizes is None or not math.isfinite(factor) or frequencies.requires_grad:
        x, B, S, D, R = _rotary_check(*tensors, layout, factor)
        if len(_rotary_sizes) > 1024:
            _rotary_sizes.clear()
        sizes = _rotary_sizes[key] = (x.device, nat.dtype_code(x.dtype), B, S, D, R, int(positions.dtype == torch.int64),
                                      _position_strides(positions),
                                      (positions.shape, positions.dtype, positions.stride(), frequencies.shape))
    return sizes


def _position_strides(positions):
    st = positions.stride()
    return nat.int64_array((st[0] if len(st) == 2 and positions.shape[0] > 1 else 0, st[-1]))


def _rotary_check(q, tq, k, tk, positions, frequencies, layout, factor):
    """Refuses what the operator does not take; (an operand, B, S, D, R)."""
    op = _QR
    _check_same_device(op, q, tq, k, tk, positions, frequencies)
    x = q if q is not None else k
    if x is None:
        raise ValueError(f"{op}: neither q nor k")
    for t in (q, k):
        if t is not None and t.dim() != 4:
            raise ValueError(f"{op}: q and k must be [B, S, H, D], got {tuple(t.shape)}")
    B, S, _, D = x.shape
    if q is not None and k is not None:
        if k.shape[:2] != q.shape[:2] or k.shape[3] != D:
            raise ValueError(f"{op}: q {tuple(q.shape)} and k {tuple(k.shape)} differ in more than their heads")
        if q.dtype != k.dtype:
            raise ValueError(f"{op}: q is {q.dtype} and k {k.dtype}")
    nat.dtype_code(x.dtype)
    if tq is not None or tk is not None:
        for y, t in ((q, tq), (k, tk)):
            if (y is None) != (t is None):
                raise ValueError(f"{op}: tangents of both q and k, or of neither")
            if t is not None and (t.shape != y.shape or t.dtype != y.dtype):
                raise ValueError(f"{op}: a tangent has its operand's shape and type")
    if positions is None or frequencies is None:
        raise ValueError(f"{op}: positions and frequencies must be given")
    if positions.dtype not in (torch.int32, torch.int64) or tuple(positions.shape) not in ((S,), (B, S), (1, S)):
        raise ValueError(f"{op}: positions must be [{S}] or [{B}, {S}] int32 or int64, got {tuple(positions.shape)} "
                         f"{positions.dtype}")
    if frequencies.dim() != 1 or frequencies.dtype != torch.float64 or not 2 <= 2 * frequencies.shape[0] <= D:
        raise ValueError(f"{op}: frequencies must be [R / 2] float64 with R at most the head dim {D}, got "
                         f"{tuple(frequencies.shape)} {frequencies.dtype}")
    if frequencies.requires_grad and torch.is_grad_enabled():
        raise RuntimeError(f"{op} has no gradient of the frequencies: detach them")
    if layout not in _LAYOUTS:
        raise ValueError(f"{op}: layout must be one of {tuple(_LAYOUTS)}, got {layout!r}")
    if not math.isfinite(factor):
        raise ValueError(f"{op}: factor must be finite, got {factor}")
    return x, B, S, D, 2 * frequencies.shape[0]


_head_strides: dict = {}
_ABSENT = (None, None)


def _heads4(t):
    """(tensor, ctypes strides) of a [B, S, H, D] operand, copied only where its rows are not contiguous: the kernel takes
    any alignment of whole elements. An axis of one element is never stepped along."""
    if t is None:
        return _ABSENT
    key = (t.shape, t.stride())
    arr = _head_strides.get(key, 0)
    if arr == 0:
        if len(_head_strides) > 4096:
            _head_strides.clear()
        st = [0 if n == 1 else s for n, s in zip(t.shape[:3], t.stride()[:3])]
        arr = _head_strides[key] = None if t.shape[3] > 1 and t.stride(3) != 1 else nat.int64_array((*st, 1))
    if arr is None:
        return _heads4(t.clone(memory_format=torch.contiguous_format))
    return t, arr


def _rotary_launch(call, q, tq, k, tk, transposed):
    """The launch: (q', tq', k', tk')."""
    dev, code, B, S, D, R, pos64, _, _ = call.sizes
    ptr, dense = nat.ptr, torch.contiguous_format
    oq = None if q is None else torch.empty_like(q, memory_format=dense)
    ok = None if k is None else torch.empty_like(k, memory_format=dense)
    otq = None if tq is None else torch.empty_like(tq, memory_format=dense)
    otk = None if tk is None else torch.empty_like(tk, memory_format=dense)
    # an operand without heads has nothing to turn
    Hq, Hk = 0 if q is None else q.shape[2], 0 if k is None else k.shape[2]
    if B * S * (Hq + Hk) == 0:
        return [oq, otq, ok, otk]
    (q, sq), (tq, stq) = (_heads4(q), _heads4(tq)) if Hq else (_ABSENT, _ABSENT)
    (k, sk), (tk, stk) = (_heads4(k), _heads4(tk)) if Hk else (_ABSENT, _ABSENT)
    with nat.on_device(dev):
        nat.check(nat.lib().dmad_qk_rotary(
            code, B, S, Hq, Hk, D, R, ptr(q), ptr(tq), ptr(k), ptr(tk), sq, stq, sk, stk, ptr(call.positions), pos64,
            call.pos_strides, ptr(call.frequencies), call.layout, transposed, call.factor,
            ptr(oq), ptr(otq), ptr(ok), ptr(otk), nat.stream_ptr(dev)))
    return [oq, otq, ok, otk]


class _Rotary(torch.autograd.Function):
    """(call, q, tq, k, tk, positions, frequencies) -> (q', tq', k', tk'); gradients of the primal outputs."""

    @staticmethod
    def forward(ctx, call, q, tq, k, tk, positions, frequencies):
        outs = _rotary_launch(call, q, tq, k, tk, 0)
        # positions and frequencies are kept by their saved tensors alone, which hooks may move and the backward frees
        ctx.save_for_backward(positions, frequencies)
        ctx.plan = call.sizes, call.layout, call.factor
        ctx.set_materialize_grads(False)
        tangents = [t for t in (outs[1], outs[3]) if t is not None]
        if tangents:
            ctx.mark_non_differentiable(*tangents)
        return tuple(outs)

    @staticmethod
    def backward(ctx, gq, _gtq, gk, _gtk):
        if torch.is_grad_enabled():
            return _rotary_backward_once(ctx, gq, gk)
        return _rotary_backward(ctx, gq, gk)


def _rotary_backward(ctx, gq, gk):
    positions, frequencies = ctx.saved_tensors
    if gq is None and gk is None:
        return (None,) * 7
    sizes, layout, factor = ctx.plan
    dev, pos_strides, (shape, dtype, strides, table) = sizes[0], *sizes[-2:]
    if positions is None or frequencies is None or positions.shape != shape or positions.dtype != dtype or \
            frequencies.shape != table or frequencies.dtype != torch.float64 or positions.device != dev or frequencies.device != dev:
        got = ", ".join("nothing" if t is None else f"{tuple(t.shape)} {t.dtype} on {t.device}" for t in (positions, frequencies))
        raise RuntimeError(f"{_QR}: the backward needs positions and frequencies as the forward read them, got {got}")
    if _eager_call(gq, gk, positions, frequencies):
        if positions.stride() != strides:
            pos_strides = _position_strides(positions)
        call = _RotaryCall(sizes, positions, pos_strides, frequencies, layout, factor)
        dq, _, dk, _ = _rotary_launch(call, gq, None, gk, None, 1)
    else:
        dq, dk = _rotary_gradients_op(gq, gk, positions, frequencies, layout == 1, factor)
    return None, dq, None, dk, None, None, None


_rotary_backward_once = torch.autograd.function.once_differentiable(_rotary_backward)


@torch.library.custom_op("dmad::qk_rotary_fwd", mutates_args=())
def qk_rotary_fwd(q: Optional[torch.Tensor], tq: Optional[torch.Tensor], k: Optional[torch.Tensor],
                  tk: Optional[torch.Tensor], positions: torch.Tensor, frequencies: torch.Tensor, half: bool,
                  factor: float) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """(q', tq', k', tk') of ``qk_rotary_with_tangent``."""
    layout = "half" if half else "interleaved"
    sizes = _rotary_plan(q, tq, k, tk, positions, frequencies, layout, factor)
    call = _RotaryCall(sizes, positions, sizes[7], frequencies, int(half), factor)
    return _or_empty(k if q is None else q, _rotary_launch(call, q, tq, k, tk, 0))


@qk_rotary_fwd.register_fake
def _(q, tq, k, tk, positions, frequencies, half, factor):
    return _or_empty(k if q is None else q, (None if t is None else t.new_empty(t.shape) for t in (q, tq, k, tk)))


@torch.library.custom_op("dmad::qk_rotary_bwd", mutates_args=())
def qk_rotary_bwd(gq: Optional[torch.Tensor], gk: Optional[torch.Tensor], positions: torch.Tensor, frequencies: torch.Tensor,
                  half: bool, factor: float) -> Tuple[torch.Tensor, torch.Tensor]:
    """(dq, dk): the outputs' gradients, of which one may be absent, turned back."""
    layout = "half" if half else "interleaved"
    sizes = _rotary_plan(gq, None, gk, None, positions, frequencies, layout, factor)
    call = _RotaryCall(sizes, positions, sizes[7], frequencies, int(half), factor)
    dq, _, dk, _ = _rotary_launch(call, gq, None, gk, None, 1)
    return _or_empty(gk if gq is None else gq, (dq, dk))


@qk_rotary_bwd.register_fake
def _(gq, gk, positions, frequencies, half, factor):
    return _or_empty(gk if gq is None else gq, (None if t is None else t.new_empty(t.shape) for t in (gq, gk)))


def _rotary_gradients_op(gq, gk, positions, frequencies, half, factor):
    dq, dk = torch.ops.dmad.qk_rotary_bwd(gq, gk, positions, frequencies, half, factor)
    return None if gq is None else dq, None if gk is None else dk


def _rotary_setup_context(ctx, inputs, output):
    q, _, k, _, positions, frequencies, *ctx.rest = inputs
    ctx.has_q, ctx.has_k = q is not None, k is not None
    ctx.save_for_backward(positions, frequencies)
    ctx.set_materialize_grads(False)


def _rotary_op_backward(ctx, gq, _gtq, gk, _gtk):
    positions, frequencies = ctx.saved_tensors
    # the gradient of an absent operand's 0-element output is none
    gq, gk = gq if ctx.has_q else None, gk if ctx.has_k else None
    if gq is None and gk is None:
        return (None,) * 8
    dq, dk = _rotary_gradients_op(gq, gk, positions, frequencies, *ctx.rest)
    return dq, None, dk, None, None, None, None, None


qk_rotary_fwd.register_autograd(_rotary_op_backward, setup_context=_rotary_setup_context)


def qk_rotary_with_tangent(q_withT, k_withT, positions, frequencies, layout="interleaved", factor=1.0):
    """Queries and keys turned by their positions: ``((q', tq'), (k', tk'))``.

    q [B, S, Hq, D], k [B, S, Hk, D]: any head counts and head dim, bf16, fp16 or fp32, any strides with contiguous rows.
    ``positions`` [S] or [B, S], int32 or int64 (a cache's ``seen`` gives those of new tokens); ``frequencies`` [R / 2]
    float64, radians per position (``rotary_frequencies``). The first R elements of every head are R / 2 pairs, neighbours
    (2i, 2i + 1) with layout "interleaved" or (i, i + R / 2) with "half"; pair i is turned by position * frequencies[i] and
    multiplied by ``factor``. The other elements stay. Angles are taken in float64 and reduced to a part of a turn
    before they are rounded, so far positions are as exact as near ones; the rotation is in float32, rounded once.
    ``apply_rope_with_tangent`` is the one by a table of angles, ``qk_norm_rope_with_tangent`` the one with the norm per head.

    ``tq``/``tk``: tangents, given for both or for neither; their outputs are detached. ``k_withT`` (or ``q_withT``) may be
    ``(None, None)``. Differentiable (once) in q and k; torch's own forward-mode tangents are refused.
    """
    (q, tq), (k, tk) = q_withT, k_withT
    factor = float(factor)
    tensors = (q, tq, k, tk, positions, frequencies)
    if not _eager_call(*tensors):
        refuse_forward_mode(_QR, *tensors)
        _rotary_check(*tensors, layout, factor)
        tq, tk = (None if t is None else t.detach() for t in (tq, tk))
        outs = torch.ops.dmad.qk_rotary_fwd(q, tq, k, tk, positions, frequencies, layout == "half", factor)
        q, tq, k, tk = (None if t is None else y for t, y in zip((q, tq, k, tk), outs))
        return (q, None if tq is None else tq.detach()), (k, None if tk is None else tk.detach())
    sizes = _rotary_plan(*tensors, layout, factor)
    call = _RotaryCall(sizes, positions, sizes[7], frequencies, _LAYOUTS[layout], factor)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k)):
        q, tq, k, tk = _Rotary.apply(call, q, tq, k, tk, positions, frequencies)
    else:
        q, tq, k, tk = _rotary_launch(call, q, tq, k, tk, 0)
    return (q, tq), (k, tk)
