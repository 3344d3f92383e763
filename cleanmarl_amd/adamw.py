"""AdamW over a list of tensors (the optimiser of policies that are the caller's own model).

The learners of this package keep one flat fp32 vector per network and step it behind the pass that makes its gradient
(cm_optimizer_step); a model has hundreds of tensors of several types.  MultiAdamW steps all of them with a few launches, states in 32 bits
or in 8 (e4m3 codes with one scale for each 256 elements), with global-norm clipping and an optional low-precision copy of each
parameter (cleanmarl/mappo_multienvs.py:584-594 with optimizer = AdamW).
"""
import ctypes as C

import numpy as np
import torch

from . import _native as N

BLOCK = 256
_DTYPES = {torch.float32: N.DTYPE_F32, torch.float16: N.DTYPE_F16, torch.bfloat16: N.DTYPE_BF16}
_ENTRY = np.dtype([("param", np.uint64), ("grad", np.uint64), ("copy", np.uint64), ("n", np.int64), ("block", np.int64),
                   ("param_dtype", np.int32), ("grad_dtype", np.int32), ("copy_dtype", np.int32), ("reserved", np.int32)])  # cm_adamw_tensor_t

_contiguous, _address, _index, _shape, _type = torch.Tensor.is_contiguous, torch.Tensor.data_ptr, torch.Tensor.get_device, torch.Tensor.shape.__get__, torch.Tensor.dtype.__get__


def _tensor(t, what, like=None):
    if t.dtype not in _DTYPES:
        raise ValueError(f"{what}: float32, float16 or bfloat16, got {t.dtype}")
    if not t.is_contiguous():
        raise ValueError(f"{what}: need a contiguous tensor, got shape {tuple(t.shape)} with strides {tuple(t.stride())}")
    if like is not None and (t.shape != like.shape or t.device != like.device):
        raise ValueError(f"{what}: need shape {tuple(like.shape)} on {like.device}, got {tuple(t.shape)} on {t.device}")
    return t


class MultiAdamW:
    """params: tensors of one GPU, each float32, float16 or bfloat16 and contiguous, no two sharing memory.

    state_bits 32 or 8 (a NaN code in root_avg_sq stands for infinity: an element whose second moment has left fp32).  max_norm > 0 clips all gradients by their global norm (``norm[0]`` is the norm of the last step, ``norm[1]`` the
    factor applied).  copies: per parameter a tensor (or None) that receives its new value in another type.  capturable: the step
    counter lives on the device, so that a captured step() counts on at every replay; a captured step reads the gradients
    at the addresses they had and keeps the learning rate, decay, eps and max_norm it was captured with.

    A step counts as an in-place operation on the parameters and copies it writes: a backward pass that needs one of them as it was before raises
    (a replayed graph's steps go uncounted, as those of torch's operations do)."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, state_bits=32, max_norm=0.0, copies=None, capturable=False):
        self.params = list(params)
        if not self.params:
            raise ValueError("params: an empty list")
        self.device = self.params[0].device  # the tensor's own: it carries an index
        if self.device.type != "cuda":
            raise ValueError(f"params are on {self.device}: the kernels have no CPU form")
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits: 8 or 32, got {state_bits}")
        if not (0.0 <= betas[0] < 1.0 and 0.0 <= betas[1] < 1.0 and eps >= 0.0):
            raise ValueError(f"betas must lie in [0, 1) and eps must not be negative, got {betas}, {eps}")
        self.copies = list(copies) if copies is not None else [None] * len(self.params)
        if len(self.copies) != len(self.params):
            raise ValueError(f"copies: {len(self.copies)} for {len(self.params)} params")
        for i, (p, c) in enumerate(zip(self.params, self.copies)):
            _tensor(p, f"params[{i}]", like=p if p.device == self.device else torch.empty(p.shape, device="meta"))
            if c is not None:
                _tensor(c, f"copies[{i}]", like=p)
        spans = sorted((t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()) for t in self.params + [c for c in self.copies if c is not None] if t.numel())
        if any(a[1] > b[0] for a, b in zip(spans, spans[1:])):
            raise ValueError("params / copies: two of them share memory")
        self.lr, self.betas, self.eps, self.weight_decay, self.max_norm = lr, tuple(betas), eps, weight_decay, max_norm
        self.state_bits, self.capturable, self.steps = state_bits, capturable, 0
        lib = N.load()
        blocks = [int(lib.cm_adamw_state_blocks(p.numel())) for p in self.params]
        self.starts = [int(b) for b in np.cumsum([0] + blocks)]  # first state block of each tensor, and the number of blocks
        total = max(1, self.starts[-1]) * BLOCK
        state = dict(dtype=torch.float32 if state_bits == 32 else torch.float8_e4m3fn, device=self.device)
        self._m, self._v = torch.zeros(total, **state), torch.zeros(total, **state)
        self.scale = torch.zeros(total // BLOCK, 2, device=self.device) if state_bits == 8 else None
        self.norm = torch.zeros(2, device=self.device)
        # what does not change from step to step; addresses are read at every step
        self._shapes, self._dtypes = [p.shape for p in self.params], [p.dtype for p in self.params]
        self._has_copies = any(c is not None for c in self.copies)
        self._fixed = np.zeros(len(self.params), _ENTRY)
        self._fixed["n"], self._fixed["block"] = [p.numel() for p in self.params], self.starts[:-1]
        self._fixed["param_dtype"] = [_DTYPES[p.dtype] for p in self.params]
        self._fixed["copy_dtype"] = [0 if c is None else _DTYPES[c.dtype] for c in self.copies]
        self.step_dev = torch.zeros(1, dtype=torch.int32, device=self.device) if capturable else None

    # the arenas: tensor i's states are elements [256 * starts[i], 256 * starts[i] + numel)
    @property
    def exp_avg(self):
        return self._m

    @property
    def exp_avg_sq(self):
        if self.state_bits == 8:
            raise AttributeError("8-bit states hold the root of the second moment: root_avg_sq")
        return self._v

    @property
    def root_avg_sq(self):
        if self.state_bits == 32:
            raise AttributeError("32-bit states hold the second moment: exp_avg_sq")
        return self._v

    def step(self, grads=None, grad_scale=1.0):
        """One step on ``grads`` (per parameter a tensor or None; default: each parameter's .grad, of which there has to be one).  A parameter without a
        gradient is left alone, its states too; the bias correction counts this optimiser's steps.  Gradients are read, multiplied by grad_scale on the way, never written."""
        params, index = self.params, self.device.index
        if grads is None:
            grads = [p.grad for p in params]
            if all(g is None for g in grads):
                raise ValueError("no parameter has a gradient: a tensor detached from a parameter (p.data) never gets one; hand over the parameters themselves, or grads")
        grads = list(grads)
        if len(grads) != len(params):
            raise ValueError(f"grads: {len(grads)} for {len(params)} params")
        have = [i for i, g in enumerate(grads) if g is not None]
        some = len(have) != len(params)
        if some:
            params, grads, copies = ([t[i] for i in have] for t in (params, grads, self.copies))
        else:
            copies = self.copies
        table = self._fixed[have] if some else self._fixed.view(np.uint8).copy().view(_ENTRY)  # (bytes: records are copied one by one, 12 us for 228)
        shapes, kinds = ([t[i] for i in have] for t in (self._shapes, self._dtypes)) if some else (self._shapes, self._dtypes)
        # the whole list at once (there may be hundreds of tensors); only a list that is not as it should be is looked through
        # (228 small tensors: 0.16 ms on the host with a generator for each check, 0.14 with these)
        types = list(map(_type, grads))
        if not (list(map(_shape, params)) == shapes == list(map(_shape, grads)) and list(map(_type, params)) == kinds and all(map(_contiguous, params))
                and all(map(_contiguous, grads)) and {index}.issuperset(map(_index, params)) and {index}.issuperset(map(_index, grads)) and _DTYPES.keys() >= set(types)):
            for i, p, g, shape, kind in zip(have, params, grads, shapes, kinds):
                if p.shape != shape or p.dtype != kind or p.device != self.device or not p.is_contiguous():
                    raise ValueError(f"params[{i}] has another device, type, shape or layout than at the start")
                _tensor(g, f"grads[{i}]", like=p)
        table["param"] = np.fromiter(map(_address, params), np.uint64, len(have))
        table["grad"] = np.fromiter(map(_address, grads), np.uint64, len(have))
        table["grad_dtype"] = np.fromiter(map(_DTYPES.__getitem__, types), np.int32, len(have))
        if self._has_copies:
            at = [i for i, c in enumerate(copies) if c is not None]
            there = [copies[i] for i in at]
            if not (list(map(_shape, there)) == [shapes[i] for i in at] and list(map(_DTYPES.get, map(_type, there))) == table["copy_dtype"][at].tolist()
                    and all(map(_contiguous, there)) and {index}.issuperset(map(_index, there))):
                raise ValueError("copies: one has another device, type, shape or layout than at the start")
            table["copy"][at] = np.fromiter(map(_address, there), np.uint64, len(at))
        lib = N.load()
        with N.on_device(index):
            clip = self.max_norm is not None and self.max_norm > 0
            nbytes = lib.cm_adamw_workspace_bytes(len(have)) if clip else 0
            ws = torch.empty(max(1, nbytes), dtype=torch.uint8, device=self.device) if clip else None
            if self.capturable:
                self.step_dev.add_(1)
            o = N.AdamW(self._m.data_ptr(), self._v.data_ptr(), None if self.scale is None else self.scale.data_ptr(), self.starts[-1],
                        self.lr, self.betas[0], self.betas[1], self.eps, self.weight_decay, self.max_norm if clip else 0.0, grad_scale,
                        self.norm.data_ptr(), None if ws is None else ws.data_ptr(), nbytes,
                        None if self.step_dev is None else self.step_dev.data_ptr(), self.steps + 1, self.state_bits)
            rc = lib.cm_adamw_multi_step(table.ctypes.data, len(have), C.byref(o), N.raw_stream(index))
            if rc and self.capturable:
                self.step_dev.sub_(1)  # a step that was refused is none
            N.check(rc, "cm_adamw_multi_step")
        torch.autograd.graph.increment_version(params)  # written behind torch's back: a graph that saved one of them has to notice
        if self._has_copies:
            torch.autograd.graph.increment_version(there)
        self.steps += 1

    def load_state(self, exp_avg, second, scale=None, step=0):
        """Copies states in: exp_avg and exp_avg_sq (32 bits), or exp_avg, root_avg_sq and scale (8 bits), laid out like the arenas."""
        for mine, theirs, what in ((self._m, exp_avg, "exp_avg"), (self._v, second, "second"), (self.scale, scale, "scale")):
            if (mine is None) != (theirs is None) or (mine is not None and (mine.shape != theirs.shape or mine.dtype != theirs.dtype)):
                raise ValueError(f"{what}: does not fit the states of this optimiser")
            if mine is not None:
                mine.copy_(theirs)
        self._set_steps(int(step))

    def _set_steps(self, step):
        self.steps = step
        if self.step_dev is not None:
            self.step_dev.fill_(step)

    def state_dict(self):
        steps = self.steps if self.step_dev is None else int(self.step_dev.item())
        return dict(exp_avg=self._m.clone(), second=self._v.clone(), scale=None if self.scale is None else self.scale.clone(), step=steps)

    def load_state_dict(self, d):
        self.load_state(d["exp_avg"], d["second"], d["scale"], d["step"])
