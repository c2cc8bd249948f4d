"""Layer norm over the last dimension.

y = (x - mean) / sqrt(var + eps) * weight + bias, the statistics taken over
the last dimension in fp32. GPU: csrc/hip/layer_norm.hip, forward and
backward, the weight's and bias's gradients summed in a fixed order. CPU:
the same formulas in plain torch (the numerics oracle).
"""

from __future__ import annotations

import torch
import torch.nn as nn

from ._ext import require_ext


def _fwd_torch(x, weight, bias, eps):
    """(y, [mean, rstd]) of x [..., C], in fp32 (fp64 for fp64)."""
    xf = x.double() if x.dtype == torch.float64 else x.float()
    mean = xf.mean(-1, keepdim=True)
    xc = xf - mean
    rstd = 1.0 / torch.sqrt(xc.square().mean(-1, keepdim=True) + eps)
    y = xc * rstd
    if weight is not None:
        y = y * weight.to(y.dtype)
    if bias is not None:
        y = y + bias.to(y.dtype)
    return y.to(x.dtype).contiguous(), torch.stack([mean, rstd])


def _bwd_torch(grad, x, weight, wtype, stats):
    mean, rstd = stats
    dy = grad.to(rstd.dtype)
    xh = (x.to(rstd.dtype) - mean) * rstd
    d = dy if weight is None else dy * weight.to(dy.dtype)
    dx = rstd * (d - d.mean(-1, keepdim=True) -
                 xh * (d * xh).mean(-1, keepdim=True))
    width = x.shape[-1]
    return (dx.to(x.dtype), (dy * xh).reshape(-1, width).sum(0).to(wtype),
            dy.reshape(-1, width).sum(0).to(wtype))


class _LayerNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, stats = _fwd_torch(x, weight, bias, eps)
        ctx.save_for_backward(x, weight, stats)
        given = weight if weight is not None else bias
        ctx.wtype = given.dtype if given is not None else x.dtype
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        x, weight, stats = ctx.saved_tensors
        grads = _bwd_torch(grad, x, weight, ctx.wtype, stats)
        return (*(g if n else None
                  for g, n in zip(grads, ctx.needs_input_grad)), None)


def layer_norm(x: torch.Tensor, weight: torch.Tensor = None,
               bias: torch.Tensor = None, eps: float = 1e-5) -> torch.Tensor:
    """Layer norm of x [..., C] over its last dimension.

    weight, bias: [C] or None (1 and 0), in x's type or float32, both in
    one type. Returns a contiguous tensor of x's shape and type. x may be
    float32, bfloat16 or float16, of any strides. The gradients have no
    gradients (create_graph), and forward-mode derivatives are refused.
    """
    if x.is_cuda:
        return require_ext().layer_norm(x, weight, bias, eps)
    if not x.is_floating_point():
        raise RuntimeError(f"layer_norm: float32, bfloat16 or float16, not "
                           f"{x.dtype}")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise RuntimeError("layer_norm: the last dimension is empty")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None and tuple(t.shape) != (x.shape[-1],):
            raise RuntimeError(f"layer_norm: {name} must be [{x.shape[-1]}]")
    return _LayerNormFn.apply(x, weight, bias, float(eps))


class LayerNorm(nn.Module):
    """Module form of layer_norm, parameters in fp32 as the other norms'."""

    def __init__(self, num_features, eps=1e-5):
        super().__init__()
        self.num_features = num_features
        self.eps = eps
        self.weight = nn.Parameter(torch.ones(num_features))
        self.bias = nn.Parameter(torch.zeros(num_features))

    def forward(self, x):
        return layer_norm(x, self.weight, self.bias, self.eps)

    def extra_repr(self):
        return f"{self.num_features}, eps={self.eps}"
