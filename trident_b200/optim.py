"""AdamW over many tensors at once, with optimizer states in 32 or in 8 bits.

One step is one kernel launch per parameter dtype (for up to 440 tensors each): the tensors' addresses
travel as kernel arguments, so a step needs no copies and no host synchronisation and can be captured in a
CUDA graph (a replay repeats the captured step number).
"""
import ctypes
from typing import Optional

import torch

from . import _lib
from .ops import _DTYPES, _call

_BLOCK = _lib.ADAMW_BLOCK
_SEED_STEP = 0x6A09E667  # fractional bits of sqrt(2): moves the rounding's seed from step to step


class AdamW:
    """m = b1 m + (1 - b1) g;  v = b2 v + (1 - b2) g^2;
    p = p (1 - lr wd) - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps), all in float32.

    params: contiguous CUDA tensors of float32, float16 or bfloat16 (dtypes may be mixed), updated in place.
    state_bits: 32 holds m and v as float32. 8 holds m and sqrt(v) as float8_e4m3fn with one float32 scale
        for each 256 values: 2 bytes a value in place of 8. m is rounded to nearest, sqrt(v) at random
        (by `seed` and the step) so that its mean is kept.
    master: keep float32 copies of 16-bit parameters, which are then their roundings. Without it an update
        below half a step of the 16-bit type is lost. (A float32 parameter is its own master copy.)
    state, step: lists of tensors (one for each parameter) to use in place of new states, and the number of
        steps behind them, to resume: "exp_avg" and "exp_avg_sq", or in 8 bits "exp_avg", "exp_avg_scale",
        "exp_avg_sq_root" and "exp_avg_sq_root_scale"; "master" where master copies are kept. `state`
        holds them afterwards under these names.
    """

    def __init__(self, params, lr: float = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 1e-2,
                 state_bits: int = 32, master: bool = False, seed: int = 0, state: Optional[dict] = None, step: int = 0):
        self.params = list(params)
        self.lr, self.betas, self.eps, self.weight_decay = float(lr), (float(betas[0]), float(betas[1])), float(eps), float(weight_decay)
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits must be 8 or 32, not {state_bits}")
        self.state_bits, self.master, self.seed, self.step_count = state_bits, bool(master), int(seed), int(step)
        if self.step_count < 0:
            raise ValueError(f"step={step}")
        if not self.params:
            raise ValueError("params is empty")
        self.dev = self.params[0].device
        for i, p in enumerate(self.params):
            if p.dtype not in _DTYPES or not p.is_cuda or p.device != self.dev or not p.is_contiguous():
                raise ValueError(f"parameter {i} must be a contiguous float32, float16 or bfloat16 tensor on one CUDA device")
        self.state = self._states(state)
        # one descriptor array per parameter dtype, filled once; a step writes the gradients' addresses
        self._groups = []
        for dtype in dict.fromkeys(p.dtype for p in self.params):
            at = [i for i, p in enumerate(self.params) if p.dtype == dtype]
            desc = (_lib.AdamWTensor * len(at))()
            for d, i in zip(desc, at):
                s = {k: v[i] for k, v in self.state.items()}
                d.param, d.n, d.m = self.params[i].data_ptr(), self.params[i].numel(), s["exp_avg"].data_ptr()
                if state_bits == 32:
                    d.v = s["exp_avg_sq"].data_ptr()
                else:
                    d.v, d.m_scale, d.v_scale = (s[k].data_ptr() for k in ("exp_avg_sq_root", "exp_avg_scale", "exp_avg_sq_root_scale"))
                if self.master and dtype != torch.float32:
                    d.master = s["master"].data_ptr()
            self._groups.append((dtype, [(i, d, self.params[i].shape, d.n) for i, d in zip(at, desc)], desc))
        self._config = _lib.AdamWConfig(state_bits=state_bits)
        self._partial = False  # a step has left tensors out by n = 0

    def _states(self, given) -> dict:
        P = self.params
        blocks = [((p.numel() + _BLOCK - 1) // _BLOCK,) for p in P]
        shapes = [tuple(p.shape) for p in P]
        if self.state_bits == 32:
            want = {"exp_avg": (torch.float32, shapes), "exp_avg_sq": (torch.float32, shapes)}
        else:
            want = {"exp_avg": (torch.float8_e4m3fn, shapes), "exp_avg_scale": (torch.float32, blocks),
                    "exp_avg_sq_root": (torch.float8_e4m3fn, shapes), "exp_avg_sq_root_scale": (torch.float32, blocks)}
        if self.master:
            want["master"] = (torch.float32, shapes)
        if given is None:
            new = {k: [torch.zeros(s, dtype=d, device=self.dev) for s in sizes] for k, (d, sizes) in want.items()}
            if self.master:
                new["master"] = [p.detach().float() for p in P]  # a float32 parameter is its own master
            return new
        if set(given) != set(want):
            raise ValueError(f"state must hold {sorted(want)}, not {sorted(given)}")
        for k, (d, sizes) in want.items():
            if len(given[k]) != len(P):
                raise ValueError(f"state[{k!r}] must hold {len(P)} tensors")
            for i, (t, s) in enumerate(zip(given[k], sizes)):
                if tuple(t.shape) != s or t.dtype != d or t.device != self.dev or not t.is_contiguous():
                    raise ValueError(f"state[{k!r}][{i}] must be a contiguous {d} tensor of shape {s} on {self.dev}")
        state = {k: list(given[k]) for k in want}
        if self.master:
            state["master"] = [p.detach() if p.dtype == torch.float32 else m for p, m in zip(P, state["master"])]
        return state

    def step(self, grads, grad_scale=None, lr: Optional[float] = None) -> None:
        """One step. grads: one tensor for each parameter, of its shape and of its dtype or float32 (the same
        choice for all parameters of a dtype), or None to leave that parameter and its states as they are.
        grad_scale: a float32 tensor of one element on the device that multiplies every gradient (a clipping
        coefficient, say). lr: this step's learning rate (default: self.lr)."""
        if len(grads) != len(self.params):
            raise ValueError(f"{len(grads)} gradients for {len(self.params)} parameters")
        if grad_scale is not None and (grad_scale.dtype != torch.float32 or grad_scale.numel() != 1 or grad_scale.device != self.dev):
            raise ValueError(f"grad_scale must be one float32 on {self.dev}")
        keep = []  # copies of gradients that were not contiguous
        calls = []
        index = self.dev.index
        for dtype, tensors, desc in self._groups:
            gdtype = None
            for i, d, shape, n in tensors:
                g = grads[i]
                if g is None:
                    d.n, self._partial = 0, True
                    continue
                if g.dtype is not gdtype:
                    if gdtype is not None:
                        raise ValueError(f"gradient {i} is {g.dtype}, others of {dtype} parameters are {gdtype}")
                    gdtype = g.dtype
                    if gdtype != dtype and gdtype != torch.float32:
                        raise ValueError(f"gradient {i} must be {dtype} or float32, not {gdtype}")
                if g.shape != shape or g.get_device() != index:
                    raise ValueError(f"gradient {i} must have its parameter's shape and device")
                if not g.is_contiguous():
                    g = g.contiguous()
                    keep.append(g)
                d.grad = g.data_ptr()
                if self._partial:
                    d.n = n
            if gdtype is not None:
                calls.append((_DTYPES[dtype], _DTYPES[gdtype], desc))
        t, c = self.step_count + 1, self._config
        c.step, c.lr = t, self.lr if lr is None else lr
        c.beta1, c.beta2 = self.betas
        c.eps, c.weight_decay = self.eps, self.weight_decay
        c.grad_scale = None if grad_scale is None else grad_scale.data_ptr()
        for k, (c.param_dtype, c.grad_dtype, desc) in enumerate(calls):
            c.rounding_seed = (self.seed + t * _SEED_STEP + k) & 0xFFFFFFFF
            _call(self.dev, _lib.lib().trident_adamw_step, desc, len(desc), ctypes.byref(c))
        self.step_count = t
