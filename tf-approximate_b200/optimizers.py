"""The optimizer step over all tensors of a network in one launch.  The reference leaves it to its host framework; here it runs on the
parameters of `layers.FakeApproxConv2D`, `layers.Dense` and any other torch parameters on one GPU."""
import ctypes as C

import numpy as np
import torch

from . import _lib
from .errors import InvalidArgumentError, raise_for_status

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_BLOCK = 256             # AXC_ADAMW_BLOCK
_TENSOR = np.dtype([("param", np.uint64), ("grad", np.uint64), ("count", np.int64), ("lr", np.float64), ("weight_decay", np.float64)])


class AdamW:
    """AdamW (decoupled weight decay) with moments in fp32 or in 8 bits.

    params: tensors of one type (float32, bfloat16 or float16) on one CUDA device, contiguous; or groups
    {"params": [...], "lr": ..., "weight_decay": ...} whose values stand in for the optimizer's own.  Parameters are updated in fp32
    and rounded once to their type.

    The moments of all parameters lie in one buffer each, every parameter's at a multiple of 256 values:
      state_bits=32   exp_avg, exp_avg_sq: fp32
      state_bits=8    exp_avg, exp_avg_sq_root: float8_e4m3fn, with exp_avg_scale and exp_avg_sq_root_scale, one fp32 value for each 256;
                      the second moment is held as its root, which is what the step divides by
    `step_count` counts the steps; a parameter without a gradient is left as it is, its moments too.  A step raises the version counter of
    the parameters that it changes.  One that is captured into a CUDA graph repeats its own step's rates and bias corrections when it is
    replayed."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, state_bits=32):
        groups = list(params)
        if groups and not isinstance(groups[0], dict):
            groups = [{"params": groups}]
        self.params, lrs, decays = [], [], []
        for g in groups:
            if not isinstance(g, dict) or "params" not in g:
                raise InvalidArgumentError("params are tensors, or dicts with the key 'params'")
            for p in ([g["params"]] if isinstance(g["params"], torch.Tensor) else g["params"]):
                self.params.append(p)
                lrs.append(g.get("lr", lr))
                decays.append(g.get("weight_decay", weight_decay))
        if not self.params:
            raise InvalidArgumentError("no parameters")
        if len({id(p) for p in self.params}) < len(self.params):
            raise InvalidArgumentError("a parameter is given twice")
        if state_bits not in (8, 32):
            raise InvalidArgumentError("state_bits must be 8 or 32")
        if not (0.0 <= betas[0] < 1.0 and 0.0 <= betas[1] < 1.0 and eps >= 0.0):
            raise InvalidArgumentError("betas must lie in [0, 1) and eps must not be negative")
        first = self.params[0]
        if not isinstance(first, torch.Tensor) or not first.is_cuda or first.dtype not in _TYPES:
            raise InvalidArgumentError("parameters must be float32, bfloat16 or float16 CUDA tensors")
        self.device, self.dtype, self.state_bits = first.device, first.dtype, state_bits
        self.betas, self.eps, self.step_count = tuple(betas), eps, 0
        for p in self.params:
            if not isinstance(p, torch.Tensor) or p.dtype is not self.dtype or p.device != self.device or not p.is_contiguous():
                raise InvalidArgumentError("every parameter must be a contiguous %s tensor on %s" % (self.dtype, self.device))
        spans = sorted((p.data_ptr(), p.data_ptr() + p.numel() * p.element_size()) for p in self.params if p.numel())
        if any(begin < end for (begin, _), (_, end) in zip(spans[1:], spans)):
            raise InvalidArgumentError("parameters share memory: a step would change it twice at the same time")
        self._counts = [p.numel() for p in self.params]
        n, blocks = len(self.params), C.c_int64()
        raise_for_status(_lib.load().axc_adamw_state_blocks((C.c_int64 * n)(*self._counts), n, C.byref(blocks)), "AdamW")
        self._table = np.zeros(n, dtype=_TENSOR)
        self._table["count"], self._table["lr"], self._table["weight_decay"] = self._counts, lrs, decays
        values = blocks.value * _BLOCK
        if state_bits == 32:
            self.exp_avg = torch.zeros(values, dtype=torch.float32, device=self.device)
            self.exp_avg_sq = torch.zeros(values, dtype=torch.float32, device=self.device)
        else:
            self.exp_avg = torch.zeros(values, dtype=torch.uint8, device=self.device).view(torch.float8_e4m3fn)
            self.exp_avg_sq_root = torch.zeros(values, dtype=torch.uint8, device=self.device).view(torch.float8_e4m3fn)
            self.exp_avg_scale = torch.zeros(blocks.value, dtype=torch.float32, device=self.device)
            self.exp_avg_sq_root_scale = torch.zeros(blocks.value, dtype=torch.float32, device=self.device)

    def set_lr(self, lr):
        """One learning rate for every parameter, from the next step on."""
        self._table["lr"] = lr

    def zero_grad(self):
        for p in self.params:
            p.grad = None

    def step(self, grads=None, grad_scale=1.0):
        """One step with `grads`, in the order of the parameters (default: their .grad; None: left as it is), times
        `grad_scale`.  A gradient has its parameter's shape, and any strides."""
        if len(self.params) != len(self._counts):
            raise InvalidArgumentError("the optimizer's parameters are those it was made with")
        if grads is not None and not isinstance(grads, list):
            grads = list(grads)
        eight = self.state_bits == 8
        _lib.binding().adamw_step(self.params, grads, self._table.ctypes.data, self.exp_avg, _TYPES[self.dtype], self.state_bits, self.step_count + 1,
                                  (self.betas[0], self.betas[1], self.eps, grad_scale), self.exp_avg_sq_root if eight else self.exp_avg_sq,
                                  self.exp_avg_scale if eight else None, self.exp_avg_sq_root_scale if eight else None)
        self.step_count += 1

    _STATES = ("exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_root", "exp_avg_sq_root_scale")

    def state_dict(self):
        """Copies of the moments, with what they belong to."""
        return {"step_count": self.step_count, "state_bits": self.state_bits, "counts": list(self._counts),
                **{k: getattr(self, k).clone() for k in self._STATES if hasattr(self, k)}}

    def load_state_dict(self, state):
        """Takes over a state of `state_dict`, as a whole or not at all."""
        names = [k for k in self._STATES if hasattr(self, k)]
        if not isinstance(state, dict) or not {"step_count", "state_bits", "counts", *names} <= state.keys():
            raise InvalidArgumentError("the state is not one of an optimizer with %d-bit moments" % self.state_bits)
        if state["state_bits"] != self.state_bits or list(state["counts"]) != self._counts:
            raise InvalidArgumentError("the state belongs to other parameters or has another number of bits")
        for k in names:
            mine, other = getattr(self, k), state[k]
            if not isinstance(other, torch.Tensor) or other.shape != mine.shape or other.dtype is not mine.dtype:
                raise InvalidArgumentError("the state's %s must be a %s tensor of shape %s" % (k, mine.dtype, tuple(mine.shape)))
        if int(state["step_count"]) < 0:
            raise InvalidArgumentError("a number of steps must not be negative")
        for k in names:
            getattr(self, k).copy_(state[k])
        self.step_count = int(state["step_count"])
