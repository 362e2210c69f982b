"""Fused AdamW: `FusedAdamW` over a model's flat parameter buffer (one kernel launch per step), `MultiTensorAdamW` over any
list of separate tensors, with states in 32 or in 8 bits.

Same update rule and defaults as the optimizer the reference wires through LightningCLI
(train/main.py:13-14, train/configs/spectralv2.yaml:99-111): decoupled weight decay, no amsgrad.
"""
import array
from operator import attrgetter

import torch

from . import _lib
from ._lib import _D, _I, _P, ptr

_lib.register({
    "noise_adamw_multi_begin": [_P, _P, _P, _I, _D, _D, _D, _P],
    "noise_adamw_multi": [_P, _P, _P, _P, _P, _I, _I, _I, _I, _P, _P, _P, _P, _P, _D, _D, _D, _D, _D, _D, _P],
})


class FusedAdamW:
    def __init__(self, model, lr=1e-4, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2):
        self.model = model
        self.lr, self.betas, self.eps, self.weight_decay = float(lr), (float(betas[0]), float(betas[1])), float(eps), float(weight_decay)
        self._m = self._v = self._step = None

    def _state(self):
        flat, grads = self.model.bind_grads()
        if self._m is None or self._m.device != flat.device or self._m.numel() != flat.numel():
            self._m = torch.zeros_like(flat)
            self._v = torch.zeros_like(flat)
            self._step = torch.zeros((), dtype=torch.int64, device=flat.device)
        return flat, grads

    def zero_grad(self, set_to_none=False):
        _, grads = self._state()
        grads.zero_()

    def step(self, grad_scale=1.0):
        flat, grads = self._state()
        _lib.require_cuda(flat)
        _lib.call("noise_adamw_step", ptr(flat), ptr(grads), ptr(self._m), ptr(self._v), ptr(self._step), flat.numel(),
                  self.lr, self.betas[0], self.betas[1], self.eps, self.weight_decay, float(grad_scale), _lib.stream(),
                  nbytes=28 * flat.numel())
        self.model.model.weights_changed()     # the kernel wrote the parameters through a raw pointer

    def state_dict(self):
        self._state()
        return {"exp_avg": self._m.clone(), "exp_avg_sq": self._v.clone(), "step": self._step.clone(),
                "lr": self.lr, "betas": self.betas, "eps": self.eps, "weight_decay": self.weight_decay}

    def load_state_dict(self, sd):
        self._state()
        self._m.copy_(sd["exp_avg"])
        self._v.copy_(sd["exp_avg_sq"])
        self._step.copy_(sd["step"])
        self.lr, self.betas, self.eps, self.weight_decay = sd["lr"], tuple(sd["betas"]), sd["eps"], sd["weight_decay"]


class MultiTensorAdamW:
    """AdamW over separate parameter tensors (fp32, bf16 or fp16, contiguous, apart in memory, on one GPU), a few launches per step for the
    whole list.

    Gradients have their parameter's type; an fp32 parameter also takes bf16 or fp16 gradients.  A parameter whose
    gradient is None is left as it is and its step count does not advance.  The arithmetic is fp32 and a 16-bit parameter is
    rounded once, to nearest: no fp32 master copy is kept.

    `state_bits=32` keeps both moments in fp32 (8 bytes per value); `state_bits=8` keeps the first moment and the root of
    the second as e4m3 values with one fp32 scale per 256 values of a tensor (2.03 bytes per value).  A block of 256 in
    which a gradient is not finite gets NaN states.

    `state` holds the flat state buffers (no copies): tensor i owns the values [offsets[i], offsets[i] + numel) of each,
    every offset a multiple of 256, and scale [offsets[i] / 256 ...] of the scale buffers.
    """
    BLOCK = 256
    MOST = 1 << 33      # values of one tensor: what one launch covers

    def __init__(self, params, lr=1e-4, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, state_bits=32):
        self.params = list(params)
        if not self.params:
            raise ValueError("MultiTensorAdamW got an empty parameter list")
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits is 32 or 8, got {state_bits}")
        hyper = self._hyper(lr, betas, eps, weight_decay)
        _lib.require_cuda(*self.params)
        if len({id(p) for p in self.params}) < len(self.params):
            raise ValueError("a parameter appears twice in the list")
        dev = self.params[0].device
        for i, p in enumerate(self.params):
            if p.device != dev:
                raise ValueError(f"parameters live on different devices: {dev} and {p.device}")
            if p.dtype not in _lib.DTYPES:
                raise TypeError(f"parameter {i} is {p.dtype}: float32, bfloat16 or float16 expected")
            if not p.is_contiguous():
                raise ValueError(f"parameter {i} of shape {tuple(p.shape)} is not contiguous")
            if p.numel() > self.MOST:
                raise ValueError(f"parameter {i} has {p.numel()} values: at most {self.MOST} are supported")
        self._apart(self.params)
        self.lr, self.betas, self.eps, self.weight_decay = hyper
        self.state_bits = state_bits
        n = len(self.params)
        self._numel = [p.numel() for p in self.params]
        self.offsets, total = [], 0
        for k in self._numel:
            self.offsets.append(total)
            total += (k + self.BLOCK - 1) // self.BLOCK * self.BLOCK
        total = max(total, self.BLOCK)
        z = dict(device=dev, dtype=torch.float32)      # whatever the default type is
        if state_bits == 8:
            # the bytes of +0 are zero
            small = lambda: torch.zeros(total, dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn)
            scales = lambda: torch.zeros(total // self.BLOCK, **z)
            self.state = {"exp_avg": small(), "exp_avg_scale": scales(), "exp_avg_sq_root": small(), "exp_avg_sq_root_scale": scales()}
        else:
            self.state = {"exp_avg": torch.zeros(total, **z), "exp_avg_sq": torch.zeros(total, **z)}
        self.step_count = torch.zeros(n, dtype=torch.int64, device=dev)
        self._coef = torch.empty(n, 2, **z)
        self._device = self.params[0].get_device()
        self._shapes = [p.shape for p in self.params]
        self._types = [p.dtype for p in self.params]
        # what a step hands to the kernel when every parameter has a gradient
        self._addresses = array.array("Q", map(torch.Tensor.data_ptr, self.params))
        self._whole = (array.array("l", self._numel), array.array("l", self.offsets), array.array("i", range(n)),
                       array.array("Q", [0xffffffffffffffff] * ((n + 63) // 64)))

    def zero_grad(self, set_to_none=True):
        for p in self.params:
            if set_to_none:
                p.grad = None
            elif p.grad is not None:
                p.grad.zero_()

    @torch.no_grad()
    def step(self, grad_scale=1.0, grads=None):
        """One update from `grads` (one tensor or None per parameter), the parameters' own `.grad` when omitted.
        `grad_scale` multiplies every gradient (1 / world size of a summed data-parallel gradient)."""
        params, n, grad_scale = self.params, len(self.params), float(grad_scale)
        grads = list(map(attrgetter("grad"), params)) if grads is None else list(grads)
        if len(grads) != n:
            raise ValueError(f"{len(grads)} gradients for {n} parameters")
        live = [i for i, g in enumerate(grads) if g is not None]
        if not live:
            return
        whole = len(live) == n
        numel, off, index, mask = self._whole
        shapes, types, addresses = self._shapes, self._types, self._addresses
        if not whole:
            params, grads, shapes, types = ([a[i] for i in live] for a in (params, grads, shapes, types))
            numel, off, addresses = (array.array(a.typecode, [a[i] for i in live]) for a in (numel, off, addresses))
            index, mask = array.array("i", live), array.array("Q", bytes(len(mask) * 8))
            for i in live:
                mask[i >> 6] |= 1 << (i & 63)
        addresses = self._check(live, params, grads, shapes, types, numel, addresses)
        gtypes = list(map(attrgetter("dtype"), grads))
        kinds = set(zip(types, gtypes))
        for pd, gd in kinds:
            if gd != pd and not (pd == torch.float32 and gd in _lib.DTYPES):
                raise TypeError(f"a {pd} parameter cannot take a {gd} gradient")
        lists = [addresses, array.array("Q", map(torch.Tensor.data_ptr, grads)), numel, off, index]
        s = self.state
        if self.state_bits == 8:
            bufs = (s["exp_avg"], s["exp_avg_scale"], s["exp_avg_sq_root"], s["exp_avg_sq_root_scale"])
        else:
            bufs = (s["exp_avg"], None, s["exp_avg_sq"], None)
        bufs = [ptr(b) for b in bufs]
        with _lib.on_device(self.step_count):
            st = _lib.stream()
            _lib.call("noise_adamw_multi_begin", ptr(self.step_count), ptr(self._coef), mask.buffer_info()[0], n, self.lr, *self.betas, st)
            for pd, gd in kinds:
                part = lists
                if len(kinds) > 1:
                    mine = [j for j in range(len(params)) if types[j] == pd and gtypes[j] == gd]
                    part = [array.array(a.typecode, [a[j] for j in mine]) for a in lists]
                state_bytes = 4 if self.state_bits == 8 else 16
                _lib.call("noise_adamw_multi", *(a.buffer_info()[0] for a in part), len(part[0]), _lib.DTYPES[pd], _lib.DTYPES[gd],
                          self.state_bits, ptr(self._coef), *bufs, self.lr, *self.betas, self.eps, self.weight_decay, grad_scale, st,
                          nbytes=sum(part[2]) * (state_bytes + 2 * pd.itemsize + gd.itemsize) if _lib.PROFILE is not None else 0)
        _lib.written(*params)      # the models' checks for stale weights go by the version counters, too

    def _check(self, live, params, grads, shapes, types, numel, addresses):
        """The parameters' addresses, after the checks.  Whole-list comparisons first: a step of many small tensors is as fast
        as the loops over them are."""
        T = torch.Tensor
        here = [self._device] * len(live)
        if list(map(attrgetter("shape"), grads)) != shapes or list(map(T.get_device, grads)) != here:
            for i, g, shape in zip(live, grads, shapes):
                if g.shape != shape or g.get_device() != self._device:
                    raise ValueError(f"gradient {i} is {tuple(g.shape)} on {g.device}, its parameter {tuple(shape)} on {self.step_count.device}")
        if not all(map(T.is_contiguous, grads)):
            grads[:] = [g.contiguous() for g in grads]
        now = array.array("Q", map(T.data_ptr, params))
        # types and sizes whatever the addresses: a rebound parameter may have got its old address again
        if (not all(map(T.is_contiguous, params)) or list(map(attrgetter("dtype"), params)) != types
                or list(map(T.numel, params)) != list(numel)
                or (now != addresses and (list(map(attrgetter("shape"), params)) != shapes or list(map(T.get_device, params)) != here))):
            raise RuntimeError("a parameter was moved, resized, converted or transposed after the optimizer was built")
        if now != addresses:
            self._apart(params)
        return now

    @staticmethod
    def _hyper(lr, betas, eps, weight_decay):
        if not (lr >= 0 and eps >= 0 and weight_decay >= 0 and len(betas) == 2 and all(0 <= b < 1 for b in betas)):
            raise ValueError(f"need lr, eps, weight_decay >= 0 and betas in [0, 1): got {lr}, {eps}, {weight_decay}, {betas}")
        return float(lr), (float(betas[0]), float(betas[1])), float(eps), float(weight_decay)

    @staticmethod
    def _apart(params):
        """Refuses parameters that share memory: one launch updates them side by side, in no order."""
        spans = sorted((p.data_ptr(), p.data_ptr() + p.numel() * p.element_size()) for p in params if p.numel())
        if any(a[1] > b[0] for a, b in zip(spans, spans[1:])):
            raise ValueError("two parameters share memory")

    def state_dict(self):
        return {**{k: v.clone() for k, v in self.state.items()}, "step": self.step_count.clone(), "state_bits": self.state_bits,
                "sizes": list(self._numel), "lr": self.lr, "betas": self.betas, "eps": self.eps, "weight_decay": self.weight_decay}

    def load_state_dict(self, sd):
        """Everything is checked before the first value is copied.  `sizes`, the parameters' sizes in their order, says which
        tensor owns which part of the buffers; a checkpoint without it (from before it was kept) is held to the totals only."""
        if sd.get("state_bits") != self.state_bits:
            raise ValueError(f"a checkpoint with {sd.get('state_bits')}-bit states cannot be loaded into {self.state_bits}-bit ones")
        for k, v in {**self.state, "step": self.step_count}.items():
            if k not in sd or sd[k].shape != v.shape or sd[k].dtype != v.dtype:
                raise ValueError(f"state {k!r} must be {v.dtype} {tuple(v.shape)}")
        if list(sd.get("sizes", self._numel)) != self._numel:
            raise ValueError("the checkpoint is of parameters of other sizes or in another order")
        missing = [k for k in ("lr", "betas", "eps", "weight_decay") if k not in sd]
        if missing:
            raise ValueError(f"the checkpoint lacks {', '.join(missing)}")
        hyper = self._hyper(sd["lr"], sd["betas"], sd["eps"], sd["weight_decay"])
        for k, v in self.state.items():
            v.view(torch.uint8).copy_(sd[k].view(torch.uint8))      # the bytes, of 8-bit values too
        self.step_count.copy_(sd["step"])
        self.lr, self.betas, self.eps, self.weight_decay = hyper
