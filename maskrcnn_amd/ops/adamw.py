"""AdamW step over many tensors, with states in 32 or 8 bits.

    c = min(1, max_grad_norm / (grad_norm + 1e-6))
    m = beta1 m + (1 - beta1) c g       v = beta2 v + (1 - beta2) (c g)^2
    p = p (1 - lr wd) - lr / (1 - beta1^t) * m / (sqrt(v / (1 - beta2^t)) + eps)

GPU: csrc/hip/adamw.hip, a launch for some 60 to 90 tensors; the gradients
are read, never rewritten, so the clipped norm costs no pass of its own over
them. CPU: the same operations in plain torch (the numerics oracle; the two
give the same bits).

With betas from 0.5 on a state is formed as m + (1 - beta1) (c g - m) with one
rounding of the result.

8-bit states: 256 values in memory order share a power of two, and a value
is its ratio to it with 3 bits of mantissa (pack_state8, unpack_state8).
Without a seed a step's new codes are the nearest to the unrounded states.
With one they are the code below or above, at random, so that their mean is
the unrounded state: over many steps the nearest codes would lose whatever
moves a state by less than half a code, a beta of 0.999 all of its decay.
"""

from __future__ import annotations

import math

import torch

from ._ext import require_ext

BLOCK8 = 256        # values of an 8-bit state that share one scale
_MIN_EXP = 40       # keeps every power and step a normal fp32 number


def _dense(t):
    """A dense tensor's values in memory order, as a view."""
    return t.as_strided((t.numel(),), (1,))


def _is_dense(t):
    return torch.ops.aten.is_non_overlapping_and_dense(t)


# Bits of random numbers (csrc/hip/adamw.hip has the same).
_WORD = 0xFFFFFFFF
_ODD = (0xAC9B39D5, 0x8FE44835)


def _mix(x):
    """A hash of 32 bits, of an int or of int64 values."""
    x = ((x ^ (x >> 16)) * _ODD[0]) & _WORD
    x = ((x ^ (x >> 15)) * _ODD[1]) & _WORD
    return x ^ (x >> 16)


def _keys(seed, step, count):
    """A key for each tensor of a call, by its number."""
    key = 0
    for word in (seed & _WORD, seed >> 32 & _WORD, step & _WORD, step >> 32):
        key = _mix((key + word + _ODD[0]) & _WORD)
    return [_mix((key + i + _ODD[0]) & _WORD) for i in range(count)]


def _hashes(key, n):
    at = torch.arange(n)
    return _mix((at & _WORD) ^ (key ^ (((at >> 32) * _ODD[1]) & _WORD)))


def _cut(x, bits):
    """x up or down to 3 bits of mantissa, by 20 random bits."""
    raw = x.view(torch.int32)
    mag = raw & 0x7FFFFFFF
    up = mag.long() + bits
    y = torch.where(up < 0x7F800000, up, mag.long()) & 0x7FF00000
    return (y.to(torch.int32) | (raw & -0x80000000)).view(torch.float32)


def _pack_torch(x, signed, hashes=None):
    low, top = (14, 127) if signed else (30, 255)
    n = x.numel()
    flat = torch.zeros(-(-n // BLOCK8) * BLOCK8, dtype=torch.float32)
    flat[:n] = _dense(x)
    above = flat > 0
    if hashes is not None:
        h = torch.zeros(flat.numel(), dtype=torch.int64)
        h[:n] = hashes
        flat = _cut(flat, h & 0xFFFFF if signed else h >> 12)
    bits = flat.view(torch.int32) & 0x7FFFFFFF
    blocks = bits.view(-1, BLOCK8)
    e = (blocks.amax(1) >> 23).clamp(min=_MIN_EXP) if n else \
        torch.zeros(0, dtype=torch.int32)
    inv = ((254 - e).clamp(min=0) << 23)
    inv = torch.where(e == 254, torch.full_like(inv, 1 << 22),
                      inv).view(torch.float32)        # 2^(127 - E)
    r = (flat.abs().view(-1, BLOCK8) * inv[:, None]).view(-1)
    rb = r.view(torch.int32)
    code = ((rb + 0x7FFFF + ((rb >> 20) & 1)) >> 20) - ((126 - low) << 3)
    small = r < 2.0 ** -low
    q = torch.where(small, r, torch.zeros_like(r)) * 2.0 ** (low + 3)
    if hashes is None:
        q = torch.round(q)
    else:
        u = (_mix((h + (1 if signed else 2)) & _WORD) >> 8) * 2.0 ** -24
        q = torch.floor(q) + (u < q - torch.floor(q))
    code = torch.where(small, q.to(torch.int32), code.clamp(max=top))
    if signed:
        code = code | ((flat.view(torch.int32) < 0).to(torch.int32) << 7)
    else:
        code = torch.where(above & (code == 0), torch.ones_like(code), code)
    code = torch.where((e == 255).repeat_interleave(BLOCK8),
                       torch.zeros_like(code), code)
    codes = torch.empty_strided(x.shape, x.stride(), dtype=torch.uint8)
    _dense(codes).copy_(code[:n])
    return codes, e.to(torch.uint8)


def _unpack_torch(codes, scales, signed, dtype):
    low = 14 if signed else 30
    c = _dense(codes).to(torch.int32)
    mag = c & 127 if signed else c
    r = torch.where(mag >= 8,
                    ((mag + ((126 - low) << 3)) << 20).view(torch.float32),
                    mag * 2.0 ** -(low + 3))
    if signed:
        r = torch.where(c > 127, -r, r)
    e = scales.to(torch.int32)
    one = (e << 23).view(torch.float32)
    one = torch.where(e == 255, torch.full_like(one, math.nan), one)
    out = torch.empty_strided(codes.shape, codes.stride(), dtype=dtype)
    _dense(out).copy_(r * one.repeat_interleave(BLOCK8)[:c.numel()])
    return out


def pack_state8(x: torch.Tensor, signed: bool):
    """fp32 values -> (codes, scales), both uint8.

    signed: the first moment's code (sign, 4 bits of exponent, 3 of
    mantissa), else the second's (5 bits of exponent), whose values above
    zero never get the code of zero. codes has x's shape and strides,
    scales one value for 256 of x in memory order. A block with an infinity
    or NaN stands for NaN.
    """
    if x.is_cuda:
        return require_ext().pack_state8(x, signed)
    if x.dtype != torch.float32 or not _is_dense(x):
        raise RuntimeError("pack_state8: a dense float32 tensor")
    return _pack_torch(x, signed)


def unpack_state8(codes: torch.Tensor, scales: torch.Tensor, signed: bool,
                  dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The values that codes and scales stand for; bfloat16 holds them
    exactly."""
    if codes.is_cuda:
        return require_ext().unpack_state8(codes, scales, signed, dtype)
    if codes.dtype != torch.uint8 or not _is_dense(codes):
        raise RuntimeError("unpack_state8: codes must be dense bytes")
    if scales.dtype != torch.uint8 or scales.dim() != 1 or \
            scales.numel() != -(-codes.numel() // BLOCK8):
        raise RuntimeError("unpack_state8: scales must be one byte for 256 "
                           "codes")
    return _unpack_torch(codes, scales, signed, dtype)


def grad_norm(tensors) -> torch.Tensor:
    """2-norm over all values of a list of tensors, as one fp32 value on
    their device. Squares are summed in 64 bits. Differentiable."""
    tensors = list(tensors)
    if not tensors:
        raise RuntimeError("grad_norm: no tensors")
    if tensors[0].is_cuda:
        return require_ext().grad_norm(tensors)
    return torch.stack([t.double().square().sum()
                        for t in tensors]).sum().sqrt().float()


def _moved(state, value, beta, codes, lerp):
    """The state after `value`, rounded once to fp32 (csrc/hip/adamw.hip).
    codes: None for fp32 states, else how they are rounded to 8 bits."""
    if not lerp:
        return state * beta + value * (1.0 - beta)
    weight = float(torch.tensor(1.0 - beta, dtype=torch.float32))
    wide = state.double() + (value - state).double() * weight
    x = wide.float()
    if codes is None:
        return torch.where(state.isinf(), state + value, x)
    if codes == "random":
        return x
    bits = x.view(torch.int32)
    lost = (value - state).double() * weight + (state - x).double()
    up = (torch.sign(lost) * torch.sign(x)).to(torch.int32)
    middle = ((bits & 0xFFFFF) == 0x80000) & ~x.isnan()
    return torch.where(middle, bits + up, bits).view(torch.float32)


def _step_torch(p, g, m, v, clip, beta1, beta2, eps, decay, rate, inv_bc2,
                codes):
    """One tensor's step; m and v are fp32 and changed in place."""
    gf = g.float()
    if clip is not None:
        gf = gf * clip
    lerp = beta1 >= 0.5 and beta2 >= 0.5
    m.copy_(_moved(m, gf, beta1, codes, lerp))
    v.copy_(_moved(v, gf * gf, beta2, codes, lerp))
    p.copy_(p.float() * decay - m / (torch.sqrt(v) * inv_bc2 + eps) * rate)


@torch.no_grad()
def adamw_step(params, grads, exp_avgs, exp_avg_sqs, *,
               exp_avg_scales=None, exp_avg_sq_scales=None, step: int,
               lr: float, betas=(0.9, 0.999), eps: float = 1e-8,
               weight_decay: float = 0.0, grad_norm=None,
               max_grad_norm: float = 0.0, seed: int = None) -> None:
    """Updates params and their states in place.

    params: float32, bfloat16 or float16, dense, in any mixture; grads: in
    their parameter's type and shape. exp_avgs, exp_avg_sqs: float32 in the
    parameter's shape and strides; or uint8 codes in that layout with
    exp_avg_scales and exp_avg_sq_scales, one byte for 256 values (zeros in
    both for a state that begins). step: the number of this step, from 1.
    grad_norm: one float32 on the device (of grad_norm()); the gradients
    count as scaled to max_grad_norm where it is above that.
    seed: new 8-bit codes are rounded at random, without bias, by a hash of
    seed, step, the tensor's number in the lists and the value's place; the
    same call gives the same codes. None: they are rounded to nearest, which
    is for a step by itself. Over many steps give a seed: to nearest, a state
    that a step moves by less than half a code does not move at all, and with
    betas[1] above some 0.97 a second moment then never falls. fp32 states
    take no seed into account.

    step and lr are the host's, so the call is refused while a stream is
    captured into a graph. A tensor to write may share memory with no other.
    """
    beta1, beta2 = betas
    if not 0.0 <= beta1 < 1.0 or not 0.0 <= beta2 < 1.0:
        raise ValueError(f"adamw_step: betas {betas} outside [0, 1)")
    if step < 1:
        raise ValueError(f"adamw_step: step {step} below 1")
    if grad_norm is not None and not max_grad_norm > 0.0:
        raise ValueError("adamw_step: grad_norm without a max_grad_norm "
                         "above 0")
    if params and params[0].is_cuda:
        require_ext().adamw_step(
            params, grads, exp_avgs, exp_avg_sqs, exp_avg_scales,
            exp_avg_sq_scales, grad_norm, max_grad_norm, step, lr, beta1,
            beta2, eps, weight_decay,
            None if seed is None else int(seed) & (1 << 64) - 1)
        return
    eight = exp_avg_scales is not None
    if eight != (exp_avg_sq_scales is not None) or not (
            len(params) == len(grads) == len(exp_avgs) == len(exp_avg_sqs)) \
            or eight and not (len(params) == len(exp_avg_scales) ==
                              len(exp_avg_sq_scales)):
        raise RuntimeError("adamw_step: the lists have different lengths")
    clip = None
    if grad_norm is not None:
        clip = (torch.full_like(grad_norm, max_grad_norm) /
                (grad_norm + 1e-6)).clamp(max=1.0)
    random = eight and seed is not None
    keys = _keys(int(seed), int(step), len(params)) if random else None
    scalars = (clip, beta1, beta2, eps, 1.0 - lr * weight_decay,
               lr / (1.0 - beta1 ** step),
               1.0 / math.sqrt(1.0 - beta2 ** step),
               ("random" if random else "nearest") if eight else None)
    for i, (p, g, m, v) in enumerate(zip(params, grads, exp_avgs,
                                         exp_avg_sqs)):
        want = torch.uint8 if eight else torch.float32
        if p.dtype not in (torch.float32, torch.bfloat16, torch.float16):
            raise RuntimeError(f"adamw_step: parameter {i} is {p.dtype}")
        if g.dtype != p.dtype or m.dtype != want or v.dtype != want:
            raise RuntimeError(f"adamw_step: tensor {i}: the gradient must "
                               "have the parameter's type and the states "
                               f"must be {want}")
        if not g.shape == m.shape == v.shape == p.shape:
            raise RuntimeError(f"adamw_step: tensor {i}: sizes differ")
        if not eight:
            _step_torch(p, g, m, v, *scalars)
            continue
        mf = unpack_state8(m, exp_avg_scales[i], True)
        vf = unpack_state8(v, exp_avg_sq_scales[i], False)
        _step_torch(p, g, mf, vf, *scalars)
        for codes, scales, x, signed in (
                (m, exp_avg_scales[i], mf, True),
                (v, exp_avg_sq_scales[i], vf, False)):
            new, exps = _pack_torch(
                x, signed, _hashes(keys[i], p.numel()) if random else None)
            codes.copy_(new)
            scales.copy_(exps)
