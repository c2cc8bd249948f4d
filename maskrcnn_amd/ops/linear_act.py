"""Dense layer with bias, activation and residual in one product.

    y = act(x W^T + bias) + residual

GPU: csrc/hip/linear_act.hip, the forward and both gradients' products on
the matrix cores. CPU: the same formulas in plain torch (the numerics
oracle).
"""

from __future__ import annotations

import math

import torch

from ._ext import require_ext

ACTIVATIONS = ("none", "relu", "gelu", "silu")
_INDEX = {name: i for i, name in enumerate(ACTIVATIONS)}   # of csrc's enum


def _act_torch(z, act):
    """The activation and its derivative."""
    if act == "relu":
        return z.clamp(min=0), (z > 0).to(z.dtype)
    if act == "gelu":
        cdf = 0.5 * torch.erfc(z * -math.sqrt(0.5))
        return z * cdf, cdf + z * torch.exp(-0.5 * z * z) / \
            math.sqrt(2.0 * math.pi)
    if act == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1.0 + z * (1.0 - s))
    return z, torch.ones_like(z)


# Mantissa bits of a small derivative in 16 bits, and its smallest exponent.
_KEPT = {torch.bfloat16: (8, -52), torch.float16: (9, -28)}


def _keep(slope, dtype):
    """The derivative as it is kept beside 16-bit tensors: in steps of 2^-15,
    small ones in those of their own exponent (csrc/hip/linear_act.hip)."""
    bits, least = _KEPT[dtype]
    _, e = torch.frexp(slope)
    step = torch.ldexp(torch.ones_like(slope),
                       (e - 1).clamp(min=least, max=bits - 15) - bits)
    return torch.round(slope / step) * step


def _fwd_torch(x, weight, bias, act, residual):
    wide = torch.float64 if x.dtype == torch.float64 else torch.float32
    z = x.to(wide) @ weight.to(wide).t()
    if bias is not None:
        z = z + bias.to(wide)
    y, slope = _act_torch(z, act)
    if residual is not None:
        y = y + residual.to(wide)
    if act == "none":
        return y.to(x.dtype), None
    if x.dtype in _KEPT:
        slope = _keep(slope, x.dtype)
    return y.to(x.dtype), slope


def _bwd_torch(grad, slope, x, weight):
    wide = torch.float64 if x.dtype == torch.float64 else torch.float32
    n, k = weight.shape
    dz = grad.to(wide).reshape(-1, n)
    if slope is not None:
        dz = dz * slope.reshape(-1, n)
    dx = (dz @ weight.to(wide)).reshape(x.shape)
    dw = dz.t() @ x.to(wide).reshape(dz.shape[0], k)
    return dx.to(x.dtype), dw.to(x.dtype), dz.sum(0).to(x.dtype)


class _LinearActFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act):
        y, slope = _fwd_torch(x, weight, bias, act, residual)
        ctx.save_for_backward(x, weight, slope)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        x, weight, slope = ctx.saved_tensors
        grads = (*_bwd_torch(grad, slope, x, weight), grad)
        return (*(g if n else None
                  for g, n in zip(grads, ctx.needs_input_grad)), None)


def linear_act(x: torch.Tensor, weight: torch.Tensor,
               bias: torch.Tensor = None, activation: str = "none",
               residual: torch.Tensor = None) -> torch.Tensor:
    """act(x @ weight.T + bias) + residual.

    x: [..., K]; weight: [N, K] (nn.Linear's layout); bias: [N] or None;
    residual: [..., N] or None. All in one type, float32, bfloat16 or
    float16, of any strides; sums are in fp32. activation: "none", "relu",
    "gelu" (by erf) or "silu". Returns a contiguous [..., N] in x's type.
    In 16 bits act'(z) is kept for the backward to 2^-16, and where it is
    small to 2^-9 (bf16) or 2^-10 (fp16) of itself (ReLU's is exact); the
    gradient of z goes into the products as two numbers of x's type. The
    gradients have no gradients (create_graph), and forward-mode derivatives
    are refused. On the GPU rows may lie up to 8 MB apart.
    """
    act = _INDEX.get(activation)
    if act is None:
        raise ValueError(f"linear_act: activation {activation!r}, not one "
                         f"of {ACTIVATIONS}")
    if x.is_cuda:
        return require_ext().linear_act(x, weight, bias, act, residual)
    if not x.is_floating_point():
        raise RuntimeError(f"linear_act: float32, bfloat16 or float16, not "
                           f"{x.dtype}")
    if x.dim() < 1 or weight.dim() != 2 or not weight.shape[0] or \
            weight.shape[1] != x.shape[-1]:
        raise RuntimeError(
            "linear_act: x [..., K] and weight [N, K], N at least 1; "
            f"got {tuple(x.shape)} and {tuple(weight.shape)}")
    shape = (*x.shape[:-1], weight.shape[0])
    for name, t, want in (("weight", weight, weight.shape),
                          ("bias", bias, shape[-1:]),
                          ("residual", residual, shape)):
        if t is None:
            continue
        if t.dtype != x.dtype or t.device != x.device:
            raise RuntimeError(
                f"linear_act: {name} must have x's type and device")
        if tuple(t.shape) != tuple(want):
            raise RuntimeError(f"linear_act: {name} must be {list(want)}")
    return _LinearActFn.apply(x, weight, bias, residual, activation)
