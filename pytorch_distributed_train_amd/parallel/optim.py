"""Fused SGD+momentum and AdamW over the flat parameter buffer.

FusedSGD:

Replaces torch's _fused_sgd / multi-tensor-apply path
with ONE kernel over ONE buffer: p <- p - lr * (mu*buf + g + wd*p), torch
SGD semantics (optim/sgd.py behavior, re-implemented):
    d_p = grad + wd * p
    buf = mu * buf + (1 - dampening) * d_p
    d_p = buf                      (or d_p + mu*buf if nesterov)
    p  -= lr * d_p

state_dict()/load_state_dict() expose torch.optim.SGD-compatible structure
(param_groups + per-param momentum_buffer) for checkpoint layout parity.
"""
from __future__ import annotations

import torch

from .flat import ALIGN, FlatParams, _aligned
from ..ops import functional as OF
from ..ops.backend import ext


class FusedSGD:
    def __init__(self, flat: FlatParams, lr: float, momentum: float = 0.0,
                 weight_decay: float = 0.0, dampening: float = 0.0,
                 nesterov: bool = False):
        if nesterov and (momentum <= 0 or dampening != 0):
            raise ValueError("nesterov needs momentum > 0, dampening = 0")
        self.flat = flat
        # on GPU lr lives in a device scalar the kernel dereferences, so a
        # hipGraph-captured step sees schedule updates (lr setter below)
        self._lr_dev = (torch.zeros(1, dtype=torch.float32,
                                    device=flat.master.device)
                        if flat.master.is_cuda else None)
        self.lr = lr
        self.momentum = momentum
        self.weight_decay = weight_decay
        self.dampening = dampening
        self.nesterov = nesterov
        self.momentum_buf = None
        if momentum != 0.0:
            self.momentum_buf = torch.zeros_like(flat.master)
        self._step_count = 0

    @property
    def lr(self) -> float:
        return self._lr

    @lr.setter
    def lr(self, value: float) -> None:
        self._lr = float(value)
        if self._lr_dev is not None:
            self._lr_dev.fill_(self._lr)

    @torch.no_grad()
    def step(self, grad_scale: float = 1.0) -> None:
        p, g = self.flat.master, self.flat.grad
        # torch.optim.SGD initializes the momentum buffer to a CLONE of d_p
        # on its first use (no (1-dampening) factor); with zero-initialized
        # flat storage that is equivalent to dampening=0 on the first step
        damp = self.dampening if self._step_count > 0 else 0.0
        if p.is_cuda:
            mom = self.momentum_buf if self.momentum_buf is not None \
                else torch.empty(0, device=p.device)
            ext().fused_sgd(p, g, mom, self.lr, self.momentum,
                            self.weight_decay, damp,
                            self.nesterov, grad_scale,
                            lr_dev=self._lr_dev)
        else:
            d_p = g if grad_scale == 1.0 else g * grad_scale
            if self.weight_decay != 0.0:
                d_p = d_p.add(p, alpha=self.weight_decay)
            if self.momentum != 0.0:
                buf = self.momentum_buf
                buf.mul_(self.momentum).add_(d_p, alpha=1 - damp)
                d_p = d_p.add(buf, alpha=self.momentum) if self.nesterov else buf
            p.add_(d_p, alpha=-self.lr)
        self._step_count += 1

    def zero_grad(self, set_to_none: bool = False) -> None:
        # set_to_none is ignored: flat gradient storage is zeroed in place
        self.flat.zero_grad()

    # -- torch.optim.SGD-compatible checkpoint structure ------------------
    def state_dict(self) -> dict:
        state = {}
        if self.momentum_buf is not None:
            for i in range(self.flat.num_params):
                off, n = self.flat.offsets[i], self.flat.sizes[i]
                state[i] = {"momentum_buffer":
                            self.momentum_buf[off:off + n]
                            .view(self.flat.shapes[i]).clone()}
        return {
            "state": state,
            "param_groups": [{
                "lr": self.lr, "momentum": self.momentum,
                "dampening": self.dampening,
                "weight_decay": self.weight_decay,
                "nesterov": self.nesterov,
                "params": list(range(self.flat.num_params)),
            }],
        }

    def load_state_dict(self, sd: dict) -> None:
        g = sd["param_groups"][0]
        self.lr = g["lr"]
        self.momentum = g["momentum"]
        self.dampening = g.get("dampening", 0.0)
        self.weight_decay = g.get("weight_decay", 0.0)
        self.nesterov = g.get("nesterov", False)
        if self.momentum != 0.0 and self.momentum_buf is None:
            self.momentum_buf = torch.zeros_like(self.flat.master)
        for i, s in sd["state"].items():
            i = int(i)
            off, n = self.flat.offsets[i], self.flat.sizes[i]
            buf = s.get("momentum_buffer")
            if buf is not None:
                self.momentum_buf[off:off + n].copy_(
                    buf.reshape(-1).to(self.momentum_buf.device,
                                       torch.float32))
                # restored buffers are past their first use: the next step
                # must apply the real dampening factor
                self._step_count = max(self._step_count, 1)


class FusedAdamW:
    """AdamW over the flat parameter buffer (functional.adamw_step): one
    pass over parameters, gradients and states, whatever the number of
    tensors.

    state_bits 32 keeps fp32 states, 8 keeps float8_e4m3fn ones with a scale
    per 64 elements (2.1 bytes a parameter instead of 8; flat storage is
    64-aligned, so no scale covers two parameters). decay(name, shape) ->
    bool says which parameters take weight decay (None: all). Step number
    and learning rate live on the device, so a hipGraph-captured step
    advances them on replay.

    state_dict() has torch.optim.AdamW's structure; with 8-bit states
    exp_avg and exp_avg_sq are the codes (of m and of sqrt(v)), beside
    exp_avg_scale and exp_avg_sq_scale. load_state_dict() takes either kind
    into either."""

    def __init__(self, flat: FlatParams, lr: float, betas=(0.9, 0.999),
                 eps: float = 1e-8, weight_decay: float = 0.01,
                 state_bits: int = 32, decay=None, seed: int = 0):
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits must be 8 or 32, not {state_bits}")
        b1, b2 = betas
        if not (0.0 <= b1 < 1.0 and 0.0 <= b2 < 1.0):
            raise ValueError(f"betas must be in [0, 1): {betas}")
        if eps < 0.0:
            raise ValueError(f"eps must not be negative: {eps}")
        self.flat = flat
        dev, n = flat.master.device, flat.total
        self._lr_dev = (torch.zeros(1, dtype=torch.float32, device=dev)
                        if flat.master.is_cuda else None)
        self.lr = lr
        self.betas = (float(b1), float(b2))
        self.eps = eps
        self.weight_decay = weight_decay
        self.state_bits = state_bits
        self.seed = int(seed)
        self.step_count = torch.zeros(1, dtype=torch.int64, device=dev)
        state = torch.float32 if state_bits == 32 else torch.float8_e4m3fn
        self.exp_avg = torch.zeros(n, dtype=torch.float32,
                                   device=dev).to(state)
        self.exp_avg_sq = self.exp_avg.clone()
        self.exp_avg_scale = self.exp_avg_sq_scale = None
        if state_bits == 8:
            self.exp_avg_scale = torch.zeros(n // ALIGN, device=dev)
            self.exp_avg_sq_scale = torch.zeros(n // ALIGN, device=dev)
        self._decay = None
        if decay is not None:
            on = torch.zeros(n // ALIGN, dtype=torch.uint8)
            for name, off, size, shape in zip(flat.names, flat.offsets,
                                              flat.sizes, flat.shapes):
                if decay(name, shape):
                    on[off // ALIGN:(off + _aligned(size)) // ALIGN] = 1
            self._decay = on.to(dev)

    @property
    def lr(self) -> float:
        return self._lr

    @lr.setter
    def lr(self, value: float) -> None:
        self._lr = float(value)
        if self._lr_dev is not None:
            self._lr_dev.fill_(self._lr)

    def step(self, grad_scale: float = 1.0) -> None:
        OF.adamw_step(self.flat.master, self.flat.grad, self.exp_avg,
                      self.exp_avg_sq, self.step_count,
                      self._lr if self._lr_dev is None else self._lr_dev,
                      beta1=self.betas[0], beta2=self.betas[1], eps=self.eps,
                      weight_decay=self.weight_decay, decay=self._decay,
                      grad_scale=grad_scale, m_scale=self.exp_avg_scale,
                      v_scale=self.exp_avg_sq_scale, seed=self.seed)

    def zero_grad(self, set_to_none: bool = False) -> None:
        # set_to_none is ignored: flat gradient storage is zeroed in place
        self.flat.zero_grad()

    # -- torch.optim.AdamW-compatible checkpoint structure ----------------
    def _blocks(self, i):
        off, n = self.flat.offsets[i], self.flat.sizes[i]
        return slice(off // ALIGN, (off + _aligned(n)) // ALIGN)

    def state_dict(self) -> dict:
        state = {}
        step = self.step_count.to(torch.float32).cpu()[0]
        for i in range(self.flat.num_params):
            off, n = self.flat.offsets[i], self.flat.sizes[i]
            shape = self.flat.shapes[i]
            state[i] = {
                "step": step.clone(),
                "exp_avg": self.exp_avg[off:off + n].view(shape).clone(),
                "exp_avg_sq":
                    self.exp_avg_sq[off:off + n].view(shape).clone()}
            if self.state_bits == 8:
                b = self._blocks(i)
                state[i]["exp_avg_scale"] = self.exp_avg_scale[b].clone()
                state[i]["exp_avg_sq_scale"] = \
                    self.exp_avg_sq_scale[b].clone()
        return {
            "state": state,
            "param_groups": [{
                "lr": self.lr, "betas": self.betas, "eps": self.eps,
                "weight_decay": self.weight_decay, "amsgrad": False,
                "maximize": False, "state_bits": self.state_bits,
                "seed": self.seed,
                "params": list(range(self.flat.num_params)),
            }],
        }

    @torch.no_grad()
    def load_state_dict(self, sd: dict) -> None:
        g = sd["param_groups"][0]
        if "betas" not in g:
            raise ValueError("not the state of an AdamW optimizer")
        if g.get("amsgrad") or g.get("maximize"):
            raise ValueError("amsgrad and maximize are not supported")
        if any(not 0 <= int(i) < self.flat.num_params for i in sd["state"]):
            raise ValueError(f"state of {len(sd['state'])} parameters for "
                             f"{self.flat.num_params}")
        self.lr = g["lr"]
        self.betas = tuple(float(b) for b in g["betas"])
        self.eps = g["eps"]
        self.weight_decay = g["weight_decay"]
        self.seed = int(g.get("seed", self.seed))
        dev = self.flat.master.device
        # parameters that the state does not hold have none
        self.step_count.zero_()
        for t in (self.exp_avg, self.exp_avg_sq, self.exp_avg_scale,
                  self.exp_avg_sq_scale):
            if t is not None:
                t.view(torch.uint8).zero_()
        for i, s in sd["state"].items():
            i = int(i)
            off, n = self.flat.offsets[i], self.flat.sizes[i]
            if int(s["step"]) > 0:
                self.step_count.fill_(int(s["step"]))
            for key, codes, scale in (
                    ("exp_avg", self.exp_avg, self.exp_avg_scale),
                    ("exp_avg_sq", self.exp_avg_sq, self.exp_avg_sq_scale)):
                x = s[key].reshape(-1).to(dev)
                has = s.get(key + "_scale")
                if has is not None and scale is not None:
                    codes[off:off + n].copy_(x)
                    scale[self._blocks(i)].copy_(has.to(dev))
                    continue
                wide = torch.zeros(_aligned(n), device=dev)
                wide[:n].copy_(x.float())
                if has is not None:  # 8 bits into 32
                    wide.mul_(has.to(dev).repeat_interleave(ALIGN))
                    if key == "exp_avg_sq":
                        wide.square_()
                if scale is None:
                    codes[off:off + n].copy_(wide[:n])
                else:  # 32 bits into 8
                    sq = key == "exp_avg_sq"
                    c, sc = OF.adamw_quantize(wide.sqrt() if sq else wide,
                                              positive=sq)
                    codes[off:off + n].copy_(c[:n])
                    scale[self._blocks(i)].copy_(sc)
