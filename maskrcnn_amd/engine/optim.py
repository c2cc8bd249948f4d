"""AdamW over the framework's many-tensor step (ops/adamw.py).

The gradients' norm is clipped inside the step: max_grad_norm takes the place
of a clip_grad_norm_ before it, and the gradients stay as they are.
"""

from __future__ import annotations

import torch

from ..ops.adamw import (
    BLOCK8, adamw_step, grad_norm, pack_state8, unpack_state8,
)

_MOMENTS = (("exp_avg", "exp_avg_scale", True),
            ("exp_avg_sq", "exp_avg_sq_scale", False))


class AdamW(torch.optim.Optimizer):
    """AdamW with decoupled weight decay, states in 32 or 8 bits.

    params: as torch.optim's, float32, bfloat16 or float16, dense.
    state_bits: 32, or 8 for codes with a scale for 256 values, rounded at
    random (repeatably, by the step's number) so that they follow the fp32
    states in the mean.
    max_grad_norm: clips the norm over the gradients of all groups; the last
    step's norm is kept on the device as .grad_norm. A step may not be
    captured into a graph, as its number and rate are the host's.
    """

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8,
                 weight_decay=1e-2, state_bits=32, max_grad_norm=None):
        if state_bits not in (8, 32):
            raise ValueError(f"AdamW: state_bits {state_bits}, not 8 or 32")
        if lr < 0.0 or eps < 0.0 or weight_decay < 0.0:
            raise ValueError("AdamW: lr, eps and weight_decay must not be "
                             "negative")
        if not all(0.0 <= b < 1.0 for b in betas):
            raise ValueError(f"AdamW: betas {betas} outside [0, 1)")
        if max_grad_norm is not None and not max_grad_norm > 0.0:
            raise ValueError("AdamW: max_grad_norm must be above 0")
        self.state_bits = state_bits
        self.max_grad_norm = max_grad_norm
        self.grad_norm = None
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps,
                                      weight_decay=weight_decay))

    def __getstate__(self):
        return {**super().__getstate__(), "state_bits": self.state_bits,
                "max_grad_norm": self.max_grad_norm, "grad_norm": None}

    def _begin(self, p):
        state = self.state[p]
        state["step"] = 0
        dtype = torch.float32 if self.state_bits == 32 else torch.uint8
        blocks = -(-p.numel() // BLOCK8)
        for name, scale, _ in _MOMENTS:
            state[name] = torch.zeros_like(
                p, dtype=dtype, memory_format=torch.preserve_format)
            if self.state_bits == 8:
                state[scale] = torch.zeros(blocks, dtype=torch.uint8,
                                           device=p.device)

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        norm = None
        if self.max_grad_norm is not None:
            grads = [p.grad for group in self.param_groups
                     for p in group["params"] if p.grad is not None]
            if grads:
                norm = self.grad_norm = grad_norm(grads)
        for at, group in enumerate(self.param_groups):
            # Parameters that have missed steps have a number of their own;
            # a call takes those of one number and device.
            calls = {}
            for p in group["params"]:
                if p.grad is None:
                    continue
                state = self.state[p]
                if not state:
                    self._begin(p)
                state["step"] += 1
                calls.setdefault((state["step"], p.device), []).append(
                    (p, state))
            for (number, _), members in calls.items():
                states = [s for _, s in members]
                eight = self.state_bits == 8
                adamw_step(
                    [p for p, _ in members], [p.grad for p, _ in members],
                    [s["exp_avg"] for s in states],
                    [s["exp_avg_sq"] for s in states],
                    exp_avg_scales=[s["exp_avg_scale"] for s in states]
                    if eight else None,
                    exp_avg_sq_scales=[s["exp_avg_sq_scale"] for s in states]
                    if eight else None,
                    step=number, lr=group["lr"], betas=group["betas"],
                    eps=group["eps"], weight_decay=group["weight_decay"],
                    grad_norm=norm, max_grad_norm=self.max_grad_norm or 0.0,
                    seed=at if eight else None)
        return loss

    def _check_saved(self, p, saved):
        """Raises ValueError if `saved` is no state for p."""
        want = torch.float32 if self.state_bits == 32 else torch.uint8
        names = [n for m in _MOMENTS for n in m[:1 if want.is_floating_point
                                                else 2]]
        if "step" not in saved or any(
                n not in saved or saved[n].dtype != want for n in names):
            raise ValueError(f"AdamW: not states of {self.state_bits} bits")
        for name, scale, _ in _MOMENTS:
            if saved[name].shape != p.shape:
                raise ValueError(
                    f"AdamW: a saved {name} of {tuple(saved[name].shape)} "
                    f"for a parameter of {tuple(p.shape)}")
            if self.state_bits == 8 and (
                    not torch.ops.aten.is_non_overlapping_and_dense(
                        saved[name]) or
                    saved[scale].shape != (-(-p.numel() // BLOCK8),)):
                raise ValueError(f"AdamW: saved codes of {name} without "
                                 "their scales")

    def load_state_dict(self, state_dict):
        """Loads another AdamW's state of the same state_bits. (The base
        class would cast the states to their parameter's type.) A state that
        does not fit raises ValueError and changes nothing."""
        want = torch.float32 if self.state_bits == 32 else torch.uint8
        ids = [i for g in state_dict["param_groups"] for i in g["params"]]
        params = [p for g in self.param_groups for p in g["params"]]
        if len(ids) != len(params):
            raise ValueError(f"AdamW: a state of {len(ids)} parameters for "
                             f"{len(params)}")
        for i, p in zip(ids, params):
            if i in state_dict["state"]:
                self._check_saved(p, state_dict["state"][i])
        super().load_state_dict(state_dict)
        for i, p in zip(ids, params):
            if i not in state_dict["state"]:
                continue
            saved = state_dict["state"][i]
            state = self.state[p]
            state["step"] = int(saved["step"])
            for name, scale, signed in _MOMENTS:
                values = saved[name].to(p.device)
                if self.state_bits == 32:
                    state[name] = torch.empty_like(
                        p, dtype=want).copy_(values)
                    continue
                scales = saved[scale].to(p.device, copy=True)
                if values.stride() != p.stride():
                    # Scales belong to values that lie together: in another
                    # layout of the parameter other ones do.
                    full = unpack_state8(values, scales, signed)
                    values, scales = pack_state8(
                        torch.empty_like(p, dtype=torch.float32).copy_(full),
                        signed)
                elif values.data_ptr() == saved[name].data_ptr():
                    values = torch.empty_like(p, dtype=want).copy_(values)
                state[name], state[scale] = values, scales
