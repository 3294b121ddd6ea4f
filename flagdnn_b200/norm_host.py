"""Host side of group norm with an activation, channels last, and its gradient.

``group_norm`` keeps the argument order of ``torch.nn.functional.group_norm`` and adds the activation behind it, so that a
convolution's output is read once and written once.  Images stay in the layout they come in (channels-last ones take the
fast kernels), rows of tokens are ``[N, C]``.  It is differentiable; ``group_norm_backward`` is the gradient by itself.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Tuple

import torch
from torch.autograd.forward_ad import unpack_dual

from . import _native as nat
from . import conv_host as _conv

_DTYPE_IDS = {torch.float16: nat.F16, torch.bfloat16: nat.BF16, torch.float32: nat.F32}
ACTIVATIONS = {"none": nat.ACT_NONE, "relu": nat.ACT_RELU, "gelu": nat.ACT_GELU, "gelu_tanh": nat.ACT_GELU_TANH,
               "silu": nat.ACT_SILU}


def activation_id(activation: str) -> int:
    if activation not in ACTIVATIONS:
        raise RuntimeError(f"activation must be one of {', '.join(ACTIVATIONS)}, got {activation!r}")
    return ACTIVATIONS[activation]


def answered(result):
    """What the native host path answered: a status is raised."""
    if result.__class__ is int:
        nat.check(result)
    return result


def refuse_tangents(what: str, *tensors: Optional[torch.Tensor]) -> None:
    """Forward-mode differentiation: a result without a tangent would count as a constant."""
    if not torch.is_inference_mode_enabled() and any(t is not None and unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError(f"flag_dnn {what} computes no forward-mode derivatives")


def refuse_grad(what: str, *tensors: Optional[torch.Tensor]) -> None:
    refuse_tangents(what, *tensors)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise NotImplementedError(f"flag_dnn {what} computes no gradients: call it under torch.no_grad()")


def workspace(nbytes: int, device: torch.device) -> Optional[torch.Tensor]:
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


def address(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _check(x: torch.Tensor, num_groups: int, weight, bias) -> None:
    if not 2 <= x.dim() <= 4:
        raise RuntimeError(f"group_norm expects 2 to 4 dimensions ([N, C], [N, C, L] or [N, C, H, W]), got {x.dim()}")
    if x.dtype not in _DTYPE_IDS:
        raise NotImplementedError(f"flag_dnn group_norm does not support dtype={x.dtype}")
    if not x.is_cuda:
        raise NotImplementedError("flag_dnn group_norm CUDA implementation requires CUDA input")
    c = x.shape[1]
    if num_groups <= 0 or c == 0 or c % num_groups != 0:
        raise RuntimeError(f"Expected number of channels in input to be divisible by num_groups, but got {c} channels "
                           f"and num_groups={num_groups}")
    if max(x.shape) > 0x7fffffff:
        raise RuntimeError("group_norm: an extent is too large")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is None:
            continue
        if t.dim() != 1 or t.numel() != c:
            raise RuntimeError(f"{name} shape mismatch, expected ({c},)")
        if t.device != x.device:
            raise RuntimeError(f"{name} must be on the input's device")
        if t.dtype not in (x.dtype, torch.float32):
            raise RuntimeError(f"{name} must be of the input's type or float32, got {t.dtype}")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise RuntimeError("weight and bias must have the same dtype")


def _strides4(t: torch.Tensor) -> Tuple[int, int, int, int]:
    s = t.stride()
    if t.dim() == 4:
        return s
    if t.dim() == 3:
        return (s[0], s[1], s[2] * t.shape[2], s[2])
    return (s[0], s[1], s[1] * t.shape[1], s[1] * t.shape[1])


def _desc(x: torch.Tensor, num_groups: int, weight, bias, eps: float, act: int) -> "nat.NormDesc":
    d = nat.NormDesc()
    d.dtype = _DTYPE_IDS[x.dtype]
    p = weight if weight is not None else bias
    d.param_dtype = d.dtype if p is None else _DTYPE_IDS[p.dtype]
    d.n, d.c = x.shape[:2]
    d.h, d.w = x.shape[2:] if x.dim() == 4 else (1, x.shape[2] if x.dim() == 3 else 1)
    d.groups, d.activation, d.eps = num_groups, act, eps
    for i, s in enumerate(_strides4(x)):
        d.x_strides[i] = s
    return d


def empty_like(x: torch.Tensor) -> torch.Tensor:
    """A dense tensor of x's shape: channels last where x has its channels together, contiguous otherwise."""
    if x.dim() > 2 and x.stride(1) == 1 and x.shape[1] > 1:
        order = (0, *range(2, x.dim()), 1)
        back = [order.index(i) for i in range(x.dim())]
        return torch.empty([x.shape[i] for i in order], dtype=x.dtype, device=x.device).permute(back)
    return torch.empty(x.shape, dtype=x.dtype, device=x.device)


def _forward(x, num_groups, weight, bias, eps, act, want_stats):
    weight = None if weight is None else weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    y = empty_like(x)
    mean = rstd = None
    if want_stats:
        make = torch.empty if x.numel() else torch.zeros
        mean, rstd = (make((x.shape[0], num_groups), dtype=torch.float32, device=x.device) for _ in range(2))
    d = _desc(x, num_groups, weight, bias, eps, act)
    for i, s in enumerate(_strides4(y)):
        d.y_strides[i] = s
    lib = nat.load()
    nbytes = ctypes.c_int64()
    with torch.cuda.device(x.device):
        nat.check(lib.fdnn_group_norm_workspace_bytes(ctypes.byref(d), 0, ctypes.byref(nbytes)))
        ws = workspace(nbytes.value, x.device)
        nat.check(lib.fdnn_group_norm_fwd(ctypes.byref(d), x.data_ptr(), address(weight), address(bias), y.data_ptr(), address(mean),
                                          address(rstd), address(ws), nbytes.value, torch.cuda.current_stream().cuda_stream))
    return y, mean, rstd


def _backward(dy, x, mean, rstd, num_groups, weight, bias, act, wants=(True, True, True)):
    weight = None if weight is None else weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    dx = empty_like(x) if wants[0] else None
    dw = torch.empty_like(weight) if weight is not None and wants[1] else None
    db = torch.empty_like(bias) if bias is not None and wants[2] else None
    d = _desc(x, num_groups, weight, bias, 0.0, act)
    for i, s in enumerate(_strides4(dy)):
        d.dy_strides[i] = s
    for i, s in enumerate(_strides4(dx if dx is not None else x)):
        d.dx_strides[i] = s
    lib = nat.load()
    nbytes = ctypes.c_int64()
    with torch.cuda.device(x.device):
        nat.check(lib.fdnn_group_norm_workspace_bytes(ctypes.byref(d), 1, ctypes.byref(nbytes)))
        ws = workspace(nbytes.value, x.device)
        nat.check(lib.fdnn_group_norm_bwd(ctypes.byref(d), dy.data_ptr(), x.data_ptr(), mean.data_ptr(), rstd.data_ptr(),
                                          address(weight), address(bias), address(dx), address(dw), address(db), address(ws),
                                          nbytes.value, torch.cuda.current_stream().cuda_stream))
    return dx, dw, db


class _GroupNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, num_groups, eps, act):
        y, mean, rstd = _forward(x, num_groups, weight, bias, eps, act, True)
        ctx.save_for_backward(x, mean, rstd, weight, bias)
        ctx.num_groups, ctx.act = num_groups, act
        ctx.mark_non_differentiable(mean, rstd)
        return y, mean, rstd

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, _mean, _rstd):
        x, mean, rstd, weight, bias = ctx.saved_tensors
        return (*_backward(dy, x, mean, rstd, ctx.num_groups, weight, bias, ctx.act, ctx.needs_input_grad[:3]), None, None, None)


def group_norm(input: torch.Tensor, num_groups: int, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5, activation: str = "none", return_stats: bool = False):
    """``activation(torch.nn.functional.group_norm(input, num_groups, weight, bias, eps))`` in one pass over ``input``
    [N, C], [N, C, L] or [N, C, H, W] (f16, bf16, f32); activations: none, relu, gelu, gelu_tanh, silu.

    Weight and bias are of the input's type or float32.  With ``return_stats`` the result is ``(y, mean, rstd)``, the float32
    [N, num_groups] statistics that ``group_norm_backward`` takes.  Differentiable once, backwards; tensors with a tangent of
    forward-mode differentiation are refused."""
    act = activation_id(activation)
    fast = _conv._fast or _conv.native_host()
    if fast:
        y = fast.group_norm(input, num_groups, weight, bias, float(eps), act, bool(return_stats))
        if y is not None:
            return answered(y)
    _check(input, num_groups, weight, bias)
    refuse_tangents("group_norm", input, weight, bias)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (input, weight, bias)):
        y, mean, rstd = _GroupNorm.apply(input, weight, bias, num_groups, float(eps), act)
    else:
        y, mean, rstd = _forward(input, num_groups, weight, bias, float(eps), act, return_stats)
    return (y, mean, rstd) if return_stats else y


def group_norm_backward(dy: torch.Tensor, input: torch.Tensor, mean: torch.Tensor, rstd: torch.Tensor, num_groups: int,
                        weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, activation: str = "none"):
    """The gradient of ``group_norm`` for ``dy``: ``(dx, dweight, dbias)``, None in the place of a parameter that is None.
    ``mean`` and ``rstd`` are what the forward call returned.  The sums are made in a fixed order.  Not differentiable itself:
    tensors that ask for a gradient are refused outside of ``torch.no_grad()``."""
    act = activation_id(activation)
    fast = _conv._fast or _conv.native_host()
    if fast:
        grads = fast.group_norm_backward(dy, input, mean, rstd, num_groups, weight, bias, act)
        if grads is not None:
            return answered(grads)
    _check(input, num_groups, weight, bias)
    if dy.shape != input.shape or dy.dtype != input.dtype or dy.device != input.device:
        raise RuntimeError("dy must have the input's shape, dtype and device")
    for name, t in (("mean", mean), ("rstd", rstd)):
        if tuple(t.shape) != (input.shape[0], num_groups) or t.dtype != torch.float32 or t.device != input.device:
            raise RuntimeError(f"{name} must be a float32 tensor of shape ({input.shape[0]}, {num_groups}) on the input's device")
    refuse_grad("group_norm_backward", dy, input, mean, rstd, weight, bias)
    return _backward(dy, input, mean.contiguous(), rstd.contiguous(), num_groups, weight, bias, act)
