"""``DeviceAdam``: Adam / AdamW of GPU-resident tensors, all of them in one launch, with the moments
in 32 or in 8 bits.

The reference steps its GPU-resident experts and the gate with ``torch.optim.Adam`` / ``AdamW``
(MOLE/optim/mixed_optim.py:155-204); this is the same update (the arithmetic of
MOLE/cpp/define.hpp:543-579) over ``mole_adam_multi``.  With ``state_bits=8`` a moment takes one byte
an element and 4 bytes per 256 elements; see ``ops.adam_multi`` for how it is held.
"""
from __future__ import annotations

from typing import Dict, List, Tuple

import torch

from .. import ops

_E4M3_MAX = 448.0


def unpack_moment(codes: torch.Tensor, scale: torch.Tensor, square: bool) -> torch.Tensor:
    """fp32 values of an 8-bit moment (``square``: the second one)."""
    flat = codes.reshape(-1).float()
    flat = flat * scale.repeat_interleave(ops.ADAM_BLOCK)[:flat.numel()]
    return (flat.square_() if square else flat).view(codes.shape)


def pack_moment(values: torch.Tensor, square: bool) -> Tuple[torch.Tensor, torch.Tensor]:
    """Codes and scales of fp32 values, rounded to nearest: for states that come from elsewhere.  As in a
    step, a value that is NaN stays so, one that is infinite becomes its block's largest code (NaN in a block of
    zeros), and neither touches its neighbours."""
    flat = values.reshape(-1).float()
    if square:
        flat = flat.sqrt()
    n = flat.numel()
    blocks = torch.nn.functional.pad(flat, (0, -n % ops.ADAM_BLOCK)).view(-1, ops.ADAM_BLOCK)
    top = torch.where(blocks.isfinite(), blocks.abs(), 0.0).amax(1, keepdim=True)
    live = top >= 2.0 ** -100
    y = torch.where(live, blocks / torch.where(live, top, 1.0) * _E4M3_MAX, blocks * 0.0)
    if square:      # a second moment that is not zero is never held as zero
        y = torch.where((blocks > 0) & live, y.clamp(min=2.0 ** -9), y)
    codes = y.clamp_(-_E4M3_MAX, _E4M3_MAX).flatten()[:n].to(torch.float8_e4m3fn).view(values.shape)
    return codes, torch.where(live, top / _E4M3_MAX, 0.0).flatten()


class DeviceAdam(torch.optim.Optimizer):
    """Parameters are contiguous float32 or bfloat16 CUDA tensors with gradients of their type.
    ``adamw_mode`` as in ``CPUAdam``: decoupled weight decay, or decay added to the gradient.
    ``seed`` starts the random rounding of 8-bit moments."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0, adamw_mode=True,
                 state_bits=32, seed=0):
        if state_bits not in (8, 32):
            raise ValueError("the moments are held in 8 or 32 bits")
        if not (0.0 <= betas[0] < 1.0 and 0.0 <= betas[1] < 1.0):
            raise ValueError(f"betas {betas} outside [0, 1)")
        self.state_bits = state_bits
        self.seed = int(seed)
        super().__init__(params, {"lr": lr, "betas": tuple(betas), "eps": eps,
                                  "weight_decay": weight_decay, "adamw_mode": adamw_mode})

    def __getstate__(self):
        # the base class hands over its own three attributes only (copy, pickle)
        return {**super().__getstate__(), "state_bits": self.state_bits, "seed": self.seed}

    def _state_of(self, p: torch.Tensor) -> dict:
        state = self.state[p]
        if len(state) == 0:
            state["step"] = 0
            if self.state_bits == 32:
                for name in ("exp_avg", "exp_avg_sq"):
                    state[name] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
            else:
                for name in ("exp_avg", "exp_avg_sq"):
                    state[name] = torch.zeros(p.shape, dtype=torch.uint8,
                                              device=p.device).view(torch.float8_e4m3fn)
                    state[name + "_scale"] = torch.zeros(ops.adam_scales(p.numel()), device=p.device)
        return state

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        place = 0
        for group in self.param_groups:
            # one launch for all parameters of a device and type that have taken equally many steps
            calls: Dict[tuple, List[torch.Tensor]] = {}
            for p in group["params"]:
                if p.grad is None:
                    continue
                if p.grad.is_sparse:
                    raise RuntimeError("DeviceAdam takes dense gradients")
                calls.setdefault((p.device, p.dtype, int(self._state_of(p)["step"])), []).append(p)
            for (_, _, t), ps in calls.items():
                states = [self.state[p] for p in ps]
                scales = [None, None]
                if self.state_bits == 8:
                    scales = [[s["exp_avg_scale"] for s in states], [s["exp_avg_sq_scale"] for s in states]]
                ops.adam_multi(ps, [p.grad.contiguous() for p in ps], [s["exp_avg"] for s in states],
                               [s["exp_avg_sq"] for s in states], *scales, t=t + 1, lr=group["lr"],
                               betas=group["betas"], eps=group["eps"], weight_decay=group["weight_decay"],
                               adamw=group["adamw_mode"], seed=self.seed + 0x9E3779B9 * place)
                place += 1
                for s in states:
                    s["step"] = t + 1
        return loss

    # ---- checkpoint ---------------------------------------------------------------------------------
    def load_state_dict(self, state_dict):
        """Takes the state of a ``DeviceAdam`` of either width, or of ``torch.optim.Adam`` / ``AdamW``:
        moments that come in another form are converted."""
        # the base class would cast floating-point states to the parameter's type
        saved = state_dict["state"]
        for group in state_dict["param_groups"]:
            if group.get("amsgrad") or group.get("maximize"):
                raise ValueError("DeviceAdam has neither amsgrad nor maximize")
        super().load_state_dict({"state": {}, "param_groups": state_dict["param_groups"]})
        for group in self.param_groups:
            for name, value in self.defaults.items():
                group.setdefault(name, value)
        params = [p for g in self.param_groups for p in g["params"]]
        ids = [i for g in state_dict["param_groups"] for i in g["params"]]
        for i, p in zip(ids, params):
            if i in saved:
                self.state[p] = self._convert(p, saved[i])

    def _convert(self, p: torch.Tensor, src: dict) -> dict:
        out = {"step": int(src["step"])}
        for name in ("exp_avg", "exp_avg_sq"):
            x = src[name]
            if tuple(x.shape) != tuple(p.shape):
                raise ValueError(f"{name} has shape {tuple(x.shape)}, its parameter {tuple(p.shape)}")
            held8 = x.dtype == torch.float8_e4m3fn
            if held8 and self.state_bits == 8:
                out[name] = x.to(p.device).clone(memory_format=torch.contiguous_format)
                out[name + "_scale"] = src[name + "_scale"].to(p.device).clone()
                continue
            x = x.to(p.device)
            if held8:
                x = unpack_moment(x, src[name + "_scale"].to(p.device), name == "exp_avg_sq")
            if self.state_bits == 32:
                out[name] = x.float().clone(memory_format=torch.contiguous_format)
            else:
                out[name], out[name + "_scale"] = pack_moment(x, name == "exp_avg_sq")
        return out
