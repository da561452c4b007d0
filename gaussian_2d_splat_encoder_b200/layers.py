"""Layer operators with gradients on the library's kernels, for training what surrounds the frozen encoder.

The encoder's forward fuses its own convolutions, GroupNorms and heads and is inference-only.  A stage, head
or projection that is trained needs the same pieces one by one, differentiable, at sizes of its own:

* ``group_norm_act``  GroupNorm with an activation before or after it, on channels-last maps (the encoder's
  stages are Conv -> GELU -> GroupNorm, efficient_encoder.py:53-58)
* ``linear_act``      ``act(x @ weight.T + bias) + residual``: 1x1 heads, projections of ``backbone_features``,
  ``splat_features`` or ``gather_splat_latents`` and the layers of a residual block

Both take fp32, bf16 or fp16 CUDA tensors, keep every sum and statistic in fp32, round once to the tensor's
type and give the same bits for the same inputs; activations and their slopes are within 7e-7 (1 + |z|) of the
exact ones.  They run on the current stream of the tensors' device and can be captured into a CUDA graph (a
training step with ``torch.autograd.grad``, once eager graphs of the same leaves are gone, as torch asks).  The
gradients are once differentiable, in reverse mode alone: dual tensors and the transforms of torch.func are
refused.

The waits inside linear_act's kernels are bounded.  One that gives up leaves that call's outputs invalid; calls are
asynchronous, so the next call of linear_act (or its backward) raises RuntimeError, or ``check_linear_waits()``, which
waits for the device first: after the replays of a captured graph, or before results are used for good.
"""

from __future__ import annotations

import ctypes as C
import functools

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_ACTS = {"none": 0, "gelu": 1, "silu": 2}
_MAX_IMAGES = 1 << 30  # of a norm call
_NO_WORKSPACE = 256  # a linear call whose size query answers this needs none


class _NormDesc(C.Structure):
    """Mirror of gs_norm_desc."""

    _fields_ = [("B", C.c_int32), ("C", C.c_int32), ("groups", C.c_int32), ("dtype", C.c_int32),
                ("param_dtype", C.c_int32), ("act", C.c_int32), ("act_first", C.c_int32), ("eps", C.c_float),
                ("rows", C.c_int64), ("x_row", C.c_int64), ("x_img", C.c_int64), ("dy_row", C.c_int64),
                ("dy_img", C.c_int64)]


class _LinearDesc(C.Structure):
    """Mirror of gs_linear_desc."""

    _fields_ = [("M", C.c_int64), ("N", C.c_int32), ("K", C.c_int32), ("dtype", C.c_int32), ("act", C.c_int32),
                ("ldx", C.c_int64), ("ldw", C.c_int64), ("ldr", C.c_int64), ("ldy", C.c_int64),
                ("unaligned", C.c_int32)]


def _act_code(act):
    if act not in _ACTS:
        raise ValueError(f"act must be one of {', '.join(_ACTS)}, got {act!r}")
    return _ACTS[act]


def _dtype_code(name, t):
    if t.dtype not in _DTYPES:
        raise ValueError(f"{name} must be float32, bfloat16 or float16, got {t.dtype}")
    return _DTYPES[t.dtype]


def _refuse_tangents(*tensors):
    """The kernels see values alone: the tangent of a dual tensor would be dropped without a word."""
    if forward_ad._current_level < 0:
        return
    if any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise RuntimeError("the layer operators have no forward-mode derivatives (got a dual tensor)")


def _elsewhere(dev):
    """Whether another device than the tensors' is current (the call is then repeated under a switch)."""
    return torch.cuda.current_device() != dev.index


# the handle of a device's current stream, without the Stream object around it
_raw_stream = torch._C._cuda_getCurrentRawStream


def _in_order(p):
    """A parameter [C] with its values adjacent and no pending sign."""
    return (p.resolve_neg() if p.is_neg() else p).contiguous()


def _rows_of(t, first):
    """Stride of the flattened axes first..-2 of `t` (whose last axis is adjacent), or None where they do
    not form one axis."""
    stride = size = None
    for i in range(t.dim() - 2, first - 1, -1):
        n = t.shape[i]
        if n == 1:
            continue
        if stride is None:
            stride, size = t.stride(i), n
        elif t.stride(i) != stride * size:
            return None
        else:
            size *= n
    return t.shape[-1] if stride is None else stride


def _save(ctx, *tensors):
    ctx.save_for_backward(*tensors)
    ctx.saved = [None if t is None else (t.shape, t.dtype, t.device) for t in tensors]


def _unpack(ctx):
    """The saved tensors.  Hooks on them (save_on_cpu, a checkpoint) may hand back copies in other strides, so a
    backward takes layouts from what it gets here, never from the forward."""
    tensors = ctx.saved_tensors
    for t, kept in zip(tensors, ctx.saved):
        if t is not None and (t.shape != kept[0] or t.dtype is not kept[1] or t.device != kept[2]):
            raise RuntimeError(f"a saved tensor came back as {tuple(t.shape)} {t.dtype} on {t.device}, kept was "
                               f"{tuple(kept[0])} {kept[1]} on {kept[2]}")
    return tensors


# ------------------------------------------------------------------------------------ GroupNorm
@functools.lru_cache(maxsize=1024)
def _norm_plan(B, rows, channels, groups, dtype, param_dtype, act, act_first, eps, x_row, x_img, dy_row, dy_img):
    """Descriptor of a call's sizes and the workspace of its forward and backward."""
    if B > _MAX_IMAGES:  # (beyond its field in the descriptor, which would keep the low bits)
        return None, 0, 0, None
    d = _NormDesc(B, channels, groups, dtype, param_dtype, act, act_first, eps, rows, x_row, x_img, dy_row, dy_img)
    L = _lib.load()
    size = L.gs_group_norm_act_workspace_size
    return C.byref(d), int(size(C.byref(d), 0)), int(size(C.byref(d), 1)), d


def _image_layout(t):
    """`t` [B, ..., C] with its row and image strides; a copy where the layout has no such strides (or the values
    a pending sign)."""
    if t.is_neg():
        t = t.resolve_neg()
    if t.is_contiguous():
        C_ = t.shape[-1]
        return t, C_, t.numel() // max(1, t.shape[0])
    row = _rows_of(t, 1) if t.stride(-1) == 1 or t.shape[-1] == 1 else None
    if row is None:
        return _image_layout(t.contiguous())
    return t, row, t.stride(0) if t.shape[0] > 1 else 0


def _norm_forward(x, weight, bias, groups, eps, act, act_first, train):
    dev = x.device
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            return _norm_forward(x, weight, bias, groups, eps, act, act_first, train)
    x, x_row, x_img = _image_layout(x)
    shape = x.shape
    B, channels = shape[0], shape[-1]
    p = weight if weight is not None else bias
    key = (B, x.numel() // (B * channels), channels, groups, _DTYPES[x.dtype], 0 if p is None else _DTYPES[p.dtype],
           act, act_first, eps)
    desc, nbytes, _, _ = _norm_plan(*key, x_row, x_img, 0, 0)
    if nbytes == 0:
        raise ValueError(f"unsupported sizes: {tuple(shape)} in {groups} groups")
    y = x.new_empty(shape)
    # one buffer: the statistics the backward reads (8 bytes per image and group), then the workspace
    head = (B * groups * 8 + 255) // 256 * 256 if train else 0
    buf = x.new_empty(head + nbytes, dtype=torch.uint8)
    at = buf.data_ptr()
    _lib.check(_lib.load().gs_group_norm_act_fwd(desc, x.data_ptr(), None if weight is None else weight.data_ptr(),
                                                 None if bias is None else bias.data_ptr(), y.data_ptr(),
                                                 at if train else None, at + head, nbytes, _raw_stream(dev.index)),
               "gs_group_norm_act_fwd")
    return y, x, buf, key


def _norm_backward(ctx, dy):
    _refuse_tangents(dy)
    x, weight, bias, buf = _unpack(ctx)
    dev = x.device
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            return _norm_backward(ctx, dy)
    need = ctx.needs_input_grad
    x, x_row, x_img = _image_layout(x)
    weight, bias, buf = (t if t is None else t.contiguous() for t in (weight, bias, buf))
    if buf.data_ptr() & 7:  # (bytes may come back at any address; the statistics are read as pairs of floats)
        buf = buf.clone()
    dy, dy_row, dy_img = _image_layout(dy)
    desc, _, nbytes, _ = _norm_plan(*ctx.key, x_row, x_img, dy_row, dy_img)
    dx = x.new_empty(x.shape) if need[0] else None
    dw = weight.new_empty(weight.shape) if need[1] else None
    db = bias.new_empty(bias.shape) if need[2] else None
    ws = x.new_empty(nbytes, dtype=torch.uint8)
    _lib.check(_lib.load().gs_group_norm_act_bwd(desc, x.data_ptr(), None if weight is None else weight.data_ptr(),
                                                 None if bias is None else bias.data_ptr(), buf.data_ptr(),
                                                 dy.data_ptr(), None if dx is None else dx.data_ptr(),
                                                 None if dw is None else dw.data_ptr(),
                                                 None if db is None else db.data_ptr(), ws.data_ptr(), nbytes,
                                                 _raw_stream(dev.index)), "gs_group_norm_act_bwd")
    return dx, dw, db, None, None, None, None


class _GroupNormAct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, groups, eps, act, act_first):
        y, x, buf, ctx.key = _norm_forward(x, weight, bias, groups, eps, act, act_first, True)
        _save(ctx, x, weight, bias, buf)
        return y

    backward = staticmethod(once_differentiable(_norm_backward))


def _check_param(name, p, x, channels):
    if p.dim() != 1 or p.shape[0] != channels:
        raise ValueError(f"{name} must be [{channels}], got {tuple(p.shape)}")
    if p.dtype != torch.float32 and p.dtype != x.dtype:
        raise ValueError(f"{name} must be float32 or {x.dtype}, got {p.dtype}")


def group_norm_act(x: torch.Tensor, num_groups: int, weight: torch.Tensor | None = None,
                   bias: torch.Tensor | None = None, eps: float = 1e-5, *, act: str = "none",
                   act_first: bool = False) -> torch.Tensor:
    """GroupNorm of a channels-last map ``x`` [B, ..., C] with an activation, differentiable in x, weight and
    bias.

    Statistics are per image and group of C / num_groups adjacent channels over all axes between the first and
    the last (biased variance, as nn.GroupNorm).  ``act`` ("none", "gelu" in the erf form, "silu") is applied
    to the result, or with ``act_first`` to the input before it is normalised: the encoder's stages.
    num_groups = C is an instance norm.  weight and bias [C] are float32 or of x's type, both alike, and
    default to 1 and 0.  An NCHW tensor in channels_last memory format enters as ``x.permute(0, 2, 3, 1)``
    without a copy; so do channel slices of a wider map and expanded tensors, while other strides are
    copied.  Returns a contiguous tensor of x's shape and type.  C is at most 2048, images and the
    rows of one at most 2^30."""
    dev = _lib.require_cuda(x, weight, bias)
    _refuse_tangents(x, weight, bias)
    code = _act_code(act)
    _dtype_code("x", x)
    if x.dim() < 2:
        raise ValueError(f"x must be [B, ..., C], got {tuple(x.shape)}")
    num_groups, channels = int(num_groups), x.shape[-1]
    if num_groups < 1 or channels < 1 or channels % num_groups:
        raise ValueError(f"{channels} channels do not divide into {num_groups} groups")
    if channels > 2048:
        raise ValueError(f"at most 2048 channels, got {channels}")
    if not eps >= 0:
        raise ValueError(f"eps must not be negative, got {eps}")
    grad = x.requires_grad
    if weight is not None:
        _check_param("weight", weight, x, channels)
        grad, weight = grad or weight.requires_grad, _in_order(weight)
    if bias is not None:
        _check_param("bias", bias, x, channels)
        grad, bias = grad or bias.requires_grad, _in_order(bias)
        if weight is not None and weight.dtype != bias.dtype:
            raise ValueError(f"weight and bias must be of one type, got {weight.dtype} and {bias.dtype}")
    args = (x, weight, bias, num_groups, float(eps), code, int(bool(act_first)))
    if x.numel() == 0:
        # nothing to normalise; the graph stays connected, with zero gradients
        y = torch.empty(x.shape, dtype=x.dtype, device=dev)
        return y + sum((p.sum() * 0).to(x.dtype) for p in (x, weight, bias) if p is not None)
    if grad and torch.is_grad_enabled():
        return _GroupNormAct.apply(*args)
    return _norm_forward(*args, False)[0]


# --------------------------------------------------------------------------------------- linear
@functools.lru_cache(maxsize=1024)
def _linear_plan(M, N, K, dtype, act, ldx, ldw, ldr, ldy, unaligned):
    d = _LinearDesc(M, N, K, dtype, act, ldx, ldw, ldr, ldy, unaligned)
    L = _lib.load()
    size = L.gs_linear_act_workspace_size
    return C.byref(d), int(size(C.byref(d), 0)), int(size(C.byref(d), 1)), d


def _row_layout(t):
    """`t` [..., n] with the stride of its flattened rows, at least n; a copy where there is none (or the values have
    a pending sign)."""
    if t.is_neg():
        t = t.resolve_neg()
    n = t.shape[-1]
    if t.is_contiguous():
        return t, n
    row = _rows_of(t, 0) if t.stride(-1) == 1 or n == 1 else None
    return (t.contiguous(), n) if row is None or row < n else (t, row)


def _unaligned(px, pw, pg):
    return (1 if px & 15 else 0) | (2 if pw & 15 else 0) | (4 if pg & 15 else 0)


def _linear_forward(x, weight, bias, residual, act, train):
    dev = x.device
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            return _linear_forward(x, weight, bias, residual, act, train)
    x, ldx = _row_layout(x)
    weight, ldw = _row_layout(weight)
    ldr = 0
    if residual is not None:
        residual, ldr = _row_layout(residual)
    N, K = weight.shape
    px, pw = x.data_ptr(), weight.data_ptr()
    key = (x.numel() // K, N, K, _DTYPES[x.dtype], act)
    desc, nbytes, _, _ = _linear_plan(*key, ldx, ldw, ldr, 0, _unaligned(px, pw, 0))
    if nbytes == 0:
        raise ValueError(f"unsupported sizes: {tuple(x.shape)} and {tuple(weight.shape)}")
    shape = x.shape[:-1] + (N,)
    y = x.new_empty(shape)
    slope = None
    if train and act:
        slope = x.new_empty(shape, dtype=torch.float32)  # the activation's, for the backward
    ws = x.new_empty(nbytes, dtype=torch.uint8) if nbytes > _NO_WORKSPACE else None
    _lib.check(_lib.load().gs_linear_act_fwd(desc, px, pw, None if bias is None else bias.data_ptr(),
                                             None if residual is None else residual.data_ptr(), y.data_ptr(),
                                             None if slope is None else slope.data_ptr(),
                                             None if ws is None else ws.data_ptr(), nbytes, _raw_stream(dev.index)),
               "gs_linear_act_fwd")
    return y, x, weight, slope, key


def _linear_backward(ctx, dy):
    _refuse_tangents(dy)
    need = ctx.needs_input_grad
    if not (need[0] or need[1] or need[2]):
        return None, None, None, dy if need[3] else None, None
    x, weight, slope = _unpack(ctx)
    dev = x.device
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            return _linear_backward(ctx, dy)
    x, ldx = _row_layout(x)
    weight, ldw = _row_layout(weight)
    slope = None if slope is None else slope.contiguous()
    g, ldy = _row_layout(dy)
    px, pw, pg = x.data_ptr(), weight.data_ptr(), g.data_ptr()
    desc, _, nbytes, _ = _linear_plan(*ctx.key, ldx, ldw, 0, ldy, _unaligned(px, pw, pg))
    dx = x.new_empty(x.shape) if need[0] else None
    dw = weight.new_empty(weight.shape) if need[1] else None
    db = weight.new_empty(weight.shape[0]) if need[2] else None
    ws = x.new_empty(nbytes, dtype=torch.uint8)
    _lib.check(_lib.load().gs_linear_act_bwd(desc, px, pw,
                                             None if slope is None else slope.data_ptr(), pg,
                                             None if dx is None else dx.data_ptr(),
                                             None if dw is None else dw.data_ptr(),
                                             None if db is None else db.data_ptr(), ws.data_ptr(), nbytes,
                                             _raw_stream(dev.index)), "gs_linear_act_bwd")
    return dx, dw, db, dy if need[3] else None, None


class _LinearAct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act):
        y, x, weight, slope, ctx.key = _linear_forward(x, weight, bias, residual, act, True)
        _save(ctx, x, weight, slope)
        return y

    backward = staticmethod(once_differentiable(_linear_backward))


def linear_act(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, *, act: str = "none",
               residual: torch.Tensor | None = None) -> torch.Tensor:
    """``act(x @ weight.T + bias) + residual``, differentiable in all four tensors.

    x [..., K], weight [N, K] (nn.Linear's, or a 1x1 convolution's ``weight.flatten(1)``), bias [N],
    residual [..., N] of the output's shape; all of one type, float32, bfloat16 or float16.  ``act`` is
    "none", "gelu" (erf form) or "silu".  Sums are fp32 (fp32 inputs of 1e-34 and more keep fp32 accuracy); the result is
    rounded once, after the residual, and each gradient once.  Infinities come out as the formula has them but for
    two cases that give NaN: fp32 infinities of both factors that meet, and 16-bit ones of x or weight in a gradient.  Rows may be strided (channel slices of a wider map); other strides are
    copied.  Returns a contiguous tensor [..., N]."""
    _lib.require_cuda(x, weight, bias, residual)
    _refuse_tangents(x, weight, bias, residual)
    code = _act_code(act)
    _dtype_code("x", x)
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"x must be [..., K] and weight [N, K], got {tuple(x.shape)} and {tuple(weight.shape)}")
    N, K = weight.shape
    if not (1 <= N <= 1 << 20 and 1 <= K <= 1 << 20):
        raise ValueError(f"weight sides must be 1..2^20, got {tuple(weight.shape)}")
    if bias is not None and bias.shape != (N,):
        raise ValueError(f"bias must be [{N}], got {tuple(bias.shape)}")
    if residual is not None and residual.shape != x.shape[:-1] + (N,):
        raise ValueError(f"residual must be {tuple(x.shape[:-1] + (N,))}, got {tuple(residual.shape)}")
    grad = x.requires_grad or weight.requires_grad
    for name, t in (("weight", weight), ("bias", bias), ("residual", residual)):
        if t is not None:
            if t.dtype != x.dtype:
                raise ValueError(f"{name} must be {x.dtype} like x, got {t.dtype}")
            grad = grad or t.requires_grad
    bias = None if bias is None else _in_order(bias)
    if grad and torch.is_grad_enabled():
        return _LinearAct.apply(x, weight, bias, residual, code)
    return _linear_forward(x, weight, bias, residual, code, False)[0]


def check_linear_waits() -> None:
    """Waits for the current device and raises RuntimeError if a device wait of an earlier ``linear_act`` (or its
    backward, or a replay of either) gave up since the last such error: outputs since then may be invalid."""
    L, code = _lib.load(), C.c_int(0)
    _lib.check(L.gs_linear_error_flag(C.byref(code)), "gs_linear_error_flag")
    if code.value:
        raise RuntimeError(f"linear_act: a device wait gave up (code {code.value}); outputs of earlier calls are not valid")
