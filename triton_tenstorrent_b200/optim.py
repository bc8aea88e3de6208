"""AdamW over a list of CUDA tensors, with the moments in fp32 or in 8 bits: one kernel launch per step and parameter type (b200k_adamw,
include/b200k.h)."""
from __future__ import annotations

import math
import struct

import numpy as np
import torch

from . import _lib
from .ops import _DTYPES, _on, _stream

__all__ = ["AdamW"]

_BLOCK = 256                       # elements that share a scale of the 8-bit moments
_P, _G, _MASTER, _M, _V, _MS, _VS, _N, _INDEX = range(9)     # columns of the table: fields of b200k_adamw_tensor


class AdamW:
    """Updates `params` in place from their gradients:

        m <- b1 m + (1 - b1) g,  v <- b2 v + (1 - b2) g^2
        p <- p - lr weight_decay p - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)

    params          contiguous fp32, bf16 or fp16 CUDA tensors on one device that do not overlap (types may be mixed).  lr, eps and weight_decay hold for
                    all of them: parameters that are to have others (norm weights without decay, say) get an optimiser of their own
    lr              a number, or an fp32 CUDA tensor of one element that a captured step reads at each replay; like eps and weight_decay
                    it may be changed between steps (opt.lr = ...)
    state_bits      32: fp32 moments, 8 bytes a parameter.  8: one byte each for m and sqrt(v), with an fp32 scale per 256 elements;
                    stochastic rounding, reproducible from `seed`.  The scales are powers of two, unless load_state_dict took over a state with others
    master_weights  keep fp32 copies of the 16-bit parameters and update those; without them a 16-bit parameter loses every
                    update below half a unit in its last place

    The moments live in flat buffers in which parameter i begins at element offsets[i], a multiple of 256 (split() gives views in the
    parameters' shapes).  One step count serves all parameters and lives on the device, so that a captured step() can be replayed.  Steps of one
    optimiser follow one another: those on different streams have to be ordered by their caller.  copy.deepcopy and pickle give an optimiser with
    parameters and moments of its own (together with a module, in one call, its parameters are the copied module's)."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 1e-2, state_bits: int = 32,
                 master_weights: bool = False, seed: int = 0):
        self.params = list(params)
        if not self.params:
            raise ValueError("AdamW: no parameters")
        if state_bits not in (8, 32):
            raise ValueError(f"AdamW: state_bits must be 8 or 32, got {state_bits}")
        b1, b2 = (float(b) for b in betas)
        if not (0 <= b1 < 1 and 0 <= b2 < 1):
            raise ValueError(f"AdamW: betas must be in [0, 1), got {betas}")
        self._betas, self.lr, self.eps, self.weight_decay = (b1, b2), lr, eps, weight_decay
        self._check_hyper()
        self.state_bits, self.master_weights, self.seed = state_bits, bool(master_weights), int(seed) & 0xFFFFFFFF
        for i, p in enumerate(self.params):
            if not isinstance(p, torch.Tensor) or p.dtype not in _DTYPES:
                raise TypeError(f"AdamW: parameter {i} must be an fp32, bf16 or fp16 tensor")
            if p.is_inference():
                raise ValueError(f"AdamW: parameter {i} is an inference tensor")
            if not p.is_cuda or p.device != self.params[0].device:
                raise ValueError(f"AdamW: parameter {i} must live on the same CUDA device as the first one (got {p.device})")
            if not p.is_contiguous():
                raise ValueError(f"AdamW: parameter {i} is not contiguous")
        spans = sorted((p.data_ptr(), p.data_ptr() + p.numel() * p.element_size()) for p in self.params if p.numel())
        if any(a[1] > b[0] for a, b in zip(spans, spans[1:])):
            raise ValueError("AdamW: parameters overlap in memory, or one is listed twice")
        self.device = self.params[0].device
        self.offsets, total = [], 0
        for p in self.params:
            self.offsets.append(total)
            total += -(-p.numel() // _BLOCK) * _BLOCK
        self.total = total
        if state_bits == 32:
            self._m, self._v = (torch.zeros(total, device=self.device) for _ in range(2))
            self._ms = self._vs = None
        else:
            self._m, self._v = (torch.zeros(total, device=self.device, dtype=torch.uint8) for _ in range(2))
            self._ms, self._vs = (torch.zeros(total // _BLOCK, device=self.device) for _ in range(2))
        self._peak_scales = False
        self.master = None
        if self.master_weights and any(p.dtype != torch.float32 for p in self.params):
            self.master = torch.zeros(total, device=self.device)
            for i, view in enumerate(self.split(self.master)):
                view.copy_(self.params[i].detach())
        self._state = torch.empty(5, device=self.device, dtype=torch.float64)
        self._set_step(0)
        self._shapes = [p.shape for p in self.params]
        self._low = [i for i, p in enumerate(self.params) if p.dtype != torch.float32]
        self._lay_table()
        kinds = {p.dtype for p in self.params}
        self._dtype = kinds.pop() if len(kinds) == 1 and all(p.numel() for p in self.params) else None     # the one type, if there is one

    @property
    def betas(self):
        """(b1, b2), fixed at construction: the device counts their powers from step to step."""
        return self._betas

    def _lay_table(self):
        """The columns of the table that stay from step to step: addresses of this object's own moments, scales and master copies, and the sizes."""
        table = np.zeros((len(self._shapes), 9), dtype=np.int64)
        at = np.array(self.offsets, dtype=np.int64)
        width = self._m.element_size()
        table[:, _M], table[:, _V] = self._m.data_ptr() + at * width, self._v.data_ptr() + at * width
        if self.state_bits == 8:
            table[:, _MS], table[:, _VS] = self._ms.data_ptr() + at // _BLOCK * 4, self._vs.data_ptr() + at // _BLOCK * 4
        if self.master is not None:
            table[self._low, _MASTER] = self.master.data_ptr() + at[self._low] * 4
        table[:, _N] = [shape.numel() for shape in self._shapes]
        table[:, _INDEX] = np.arange(len(self._shapes))
        self._table = table
        self._dims = np.array([n for shape in self._shapes for n in (len(shape), *shape)], dtype=np.int64)     # what step() compares the tensors with
        self._addresses = self._dims.ctypes.data, table.ctypes.data

    # A copy (copy.deepcopy, pickle) has buffers of its own: the addresses are taken anew.
    def __getstate__(self):
        return {k: v for k, v in self.__dict__.items() if k not in ("_table", "_dims", "_addresses")}

    def __setstate__(self, held):
        self.__dict__.update(held)
        self._lay_table()

    def _check_hyper(self):
        if isinstance(self.lr, torch.Tensor):
            if self.lr.dtype != torch.float32 or self.lr.numel() != 1 or not self.lr.is_cuda:
                raise ValueError("AdamW: a tensor lr must be one fp32 element on the GPU")
        elif not 0 <= self.lr < math.inf:
            raise ValueError(f"AdamW: lr must be >= 0, got {self.lr}")
        if not 0 <= self.eps < math.inf or not 0 <= self.weight_decay < math.inf:
            raise ValueError(f"AdamW: eps and weight_decay must be >= 0, got {self.eps}, {self.weight_decay}")
        if 0 < self.eps < 2.0 ** -126:
            raise ValueError(f"AdamW: eps must be 0 or at least 2^-126 (a normal fp32), got {self.eps}")

    def _set_step(self, t: int):
        b1, b2 = self.betas
        raw = struct.pack("<ddqdfI", b1 ** t, b2 ** t, t, 1 / (1 - b1 ** (t + 1)), 1 / math.sqrt(1 - b2 ** (t + 1)), 0)
        self._state.copy_(torch.frombuffer(bytearray(raw), dtype=torch.float64))

    def step_count(self) -> int:
        """Steps taken so far (waits for the device)."""
        return int(self._state.view(torch.int64)[2])

    def split(self, flat: torch.Tensor):
        """Views of a flat buffer (moments, master copy) in the shapes of the parameters."""
        return [flat[a:a + p.numel()].view(p.shape) for a, p in zip(self.offsets, self.params)]

    def moments(self):
        """(m, v) as flat fp32 tensors: the buffers themselves with state_bits = 32, the values that the codes stand for with 8."""
        if self.state_bits == 32:
            return self._m, self._v
        m, v = (torch.empty(self.total, device=self.device) for _ in range(2))
        with _on(self.device):
            _lib.check(_lib.load().b200k_adamw_moments(self._m.data_ptr(), self._ms.data_ptr(), self._v.data_ptr(), self._vs.data_ptr(),
                                                       m.data_ptr(), v.data_ptr(), self.total // _BLOCK, _stream()))
        return m, v

    def zero_grad(self):
        for p in self.params:
            p.grad = None

    def step(self, grads=None, grad_scale=1.0):
        """One update.  grads: one gradient per parameter in the parameter's type or in fp32, or None for a parameter that is left
        alone (with its moments) in this step; by default the parameters' .grad.  grad_scale multiplies every gradient: a number, or
        an fp32 CUDA tensor of one element (loss scaling, clipping by a norm)."""
        params = self.params
        if grads is not None:
            grads = grads if type(grads) is list else list(grads)
            if len(grads) != len(params):
                raise ValueError(f"AdamW: {len(params)} gradients expected, got {len(grads)}")
        self._check_hyper()
        scale, scale_ptr = 1.0, 0
        if isinstance(grad_scale, torch.Tensor):
            if grad_scale.dtype != torch.float32 or grad_scale.numel() != 1 or grad_scale.device != self.device:
                raise ValueError(f"AdamW: a tensor grad_scale must be one fp32 element on {self.device}")
            scale_ptr = grad_scale.data_ptr()
        else:
            scale = float(grad_scale)
        lr, lr_ptr = self.lr, 0
        if isinstance(lr, torch.Tensor):
            if lr.device != self.device:
                raise ValueError(f"AdamW: lr must be on {self.device}")
            lr, lr_ptr = 0.0, lr.data_ptr()
        # The usual case first: every gradient there, one type each, nothing to copy
        dtype, wide = self._dtype, -1
        if dtype is not None:
            wide = _lib.tensor_list().fill_rows(params, grads, len(self._shapes), *self._addresses, 9, self.device.index, _DTYPES[dtype])
        if wide >= 0:
            launches, touched = [(dtype, torch.float32 if wide else dtype, self._table)], params
        else:
            launches, touched, grads = self._sort([p.grad for p in params] if grads is None else grads)
            if not touched:
                return
        entry = _lib.load().b200k_adamw
        b1, b2 = self.betas
        with _on(self.device):
            stream = _stream()
            for k, (dtype, gdtype, rows) in enumerate(launches):
                _lib.check(entry(rows.ctypes.data, len(rows), _DTYPES[dtype], _DTYPES[gdtype], self.state_bits + self._peak_scales * _lib.ADAMW_PEAK_SCALES, self._state.data_ptr(), lr, lr_ptr,
                                 b1, b2, self.eps, self.weight_decay, scale, scale_ptr, self.seed, int(k == len(launches) - 1), stream))
        # a backward pass that still needs an old value must fail instead of using the new one
        torch.autograd.graph.increment_version(touched)

    def _sort(self, grads):
        """The general case of step(): ([(parameter type, gradient type, table)], the parameters that take part, the gradients with copies of
        those that are not contiguous)."""
        grads, rows, touched = list(grads), {}, []
        at = self.device.index
        for i, (p, g, shape) in enumerate(zip(self.params, grads, self._shapes)):
            if g is None or shape.numel() == 0:
                continue
            if g.dtype is not p.dtype and g.dtype is not torch.float32:
                raise TypeError(f"AdamW: gradient {i} must be {p.dtype} or torch.float32, got {g.dtype}")
            if g.shape != shape or g.get_device() != at or g.layout is not torch.strided:
                raise ValueError(f"AdamW: gradient {i} must be a dense {tuple(shape)} tensor on {self.device}, got {tuple(g.shape)} on {g.device}")
            if p.shape != shape or not p.is_contiguous() or p.get_device() != at:
                raise ValueError(f"AdamW: parameter {i} is no longer a contiguous {tuple(shape)} tensor on {self.device}")
            if not g.is_contiguous():
                g = grads[i] = g.contiguous()
            rows.setdefault((p.dtype, g.dtype), []).append((i, p.data_ptr(), g.data_ptr()))
            touched.append(p)
        launches = []
        for (dtype, gdtype), mine in rows.items():
            pointers = np.array(mine, dtype=np.int64)
            table = self._table[pointers[:, 0]]
            table[:, _P:_G + 1] = pointers[:, 1:]
            launches.append((dtype, gdtype, table))
        return launches, touched, grads

    def state_dict(self) -> dict:
        """The state as tensors (copies): step, the moments as they are held, and the master copy.  lr, betas, eps, weight_decay and seed are not part of it:
        a run that is to go on as it was is given the same ones."""
        held = {"step": self.step_count(), "exp_avg": self._m.clone()}
        if self.state_bits == 32:
            held["exp_avg_sq"] = self._v.clone()
        else:
            held.update(exp_avg_scale=self._ms.clone(), exp_avg_sq_root=self._v.clone(), exp_avg_sq_root_scale=self._vs.clone())
        if self.master is not None:
            held["master"] = self.master.clone()
        return held

    def load_state_dict(self, held: dict):
        """Takes over what state_dict() of an optimiser over the same list of shapes gave.  The scales of 8-bit moments say by which rule they were made:
        powers of two, or each block's largest magnitude / the largest code's value; the steps to come go by the same one."""
        want = {"exp_avg": self._m}
        want.update({"exp_avg_sq": self._v} if self.state_bits == 32 else
                    {"exp_avg_scale": self._ms, "exp_avg_sq_root": self._v, "exp_avg_sq_root_scale": self._vs})
        if self.master is not None:
            want["master"] = self.master
        if set(held) != {"step", *want}:
            raise ValueError(f"AdamW: the state must have {sorted({'step', *want})}, got {sorted(held)}")
        for name, t in want.items():
            if held[name].dtype != t.dtype or held[name].shape != t.shape:
                raise ValueError(f"AdamW: {name} must be {t.dtype} {tuple(t.shape)}, got {held[name].dtype} {tuple(held[name].shape)}")
        if not 0 <= int(held["step"]) < 1 << 63:
            raise ValueError(f"AdamW: step must be >= 0 and below 2^63, got {held['step']}")
        for name, t in want.items():
            t.copy_(held[name])
        if self.state_bits == 8:         # a power of two has the mantissa 1/2; blocks of zeros may have the scale zero by either rule
            mantissa = torch.frexp(torch.cat([self._ms, self._vs])).mantissa
            self._peak_scales = bool(((mantissa != 0.5) & (mantissa != 0)).any())
        self._set_step(int(held["step"]))
