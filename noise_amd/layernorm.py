"""LayerNorm over the last axis of token tensors (the operator of train/models.py:90, :116, :214) for fp32, bf16 and fp16
activations of any width, forward and backward on the kernels of csrc/layernorm.hip.

    y = layer_norm(x, weight, bias)                           # differentiable
    y, mean, rstd = layer_norm_fwd(x, weight, bias)           # explicit passes: the statistics are fp32, one per row
    dx, dweight, dbias = layer_norm_bwd(dy, x, mean, rstd, weight)

`x` is (..., D) with unit stride on the last axis and evenly spaced rows (a column slice of a wider tensor is read in
place; anything else is copied first).  `weight` and `bias` are (D,), fp32 or of x's type, and may each be None.
Statistics and sums are fp32; y and dx have x's type, the parameter gradients the parameters'.
"""
import torch

from . import _lib
from ._lib import _F, _I, _L, _P, ptr

_lib.register({
    "noise_layer_norm_fwd": [_P, _L, _P, _P, _F, _P, _P, _P, _L, _I, _I, _I, _P],
    "noise_layer_norm_bwd": [_P, _L, _P, _L, _P, _P, _P, _P, _P, _P, _P, _L, _I, _I, _I, _P],
    "noise_layer_norm_bwd_rows": [_L, _I],
})


def _rows(t, D):
    """t (..., D) as (tensor, row stride): the tensor itself when its rows are evenly spaced, a packed copy otherwise."""
    if t.is_contiguous():
        return t, D
    if t.stride(-1) == 1 or D == 1:
        try:
            flat = t.view(-1, D)
        except RuntimeError:
            flat = None
        if flat is not None and (flat.stride(1) == 1 or D == 1):
            return flat, flat.stride(0)
    return t.contiguous(), D


def _check(x, weight, bias):
    _lib.no_tangents(x, weight, bias)
    _lib.require_cuda(x, weight, bias)
    if x.dtype not in _lib.DTYPES:
        raise TypeError(f"layer_norm takes float32, bfloat16 or float16 activations, got {x.dtype}")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"layer_norm needs at least one value per row, got {tuple(x.shape)}")
    D = x.shape[-1]
    if D > 1 << 24 or x.numel() // D >= 1 << 31:      # the width travels as a 32-bit number
        raise ValueError(f"layer_norm takes rows of at most 2^24 values and fewer than 2^31 of them, got {tuple(x.shape)}")
    wdtype = None
    for name, p in (("weight", weight), ("bias", bias)):
        if p is None:
            continue
        if p.shape != (D,):
            raise ValueError(f"{name} must be ({D},), got {tuple(p.shape)}")
        if p.dtype not in (torch.float32, x.dtype) or (wdtype is not None and p.dtype != wdtype):
            raise TypeError(f"weight and bias must both be float32 or both {x.dtype}, got {name} in {p.dtype}")
        wdtype = p.dtype
    return D, (torch.float32 if wdtype is None else wdtype)


def layer_norm_fwd(x, weight=None, bias=None, eps=1e-6):
    """(y, mean, rstd): y like x (packed), mean and rstd fp32 of x.shape[:-1]."""
    D, wdtype = _check(x, weight, bias)
    with _lib.on_device(x, weight, bias):
        xr, ld = _rows(x, D)
        y = x.new_empty(x.shape)
        mean, rstd = (x.new_empty(x.shape[:-1], dtype=torch.float32) for _ in range(2))
        rows = x.numel() // D
        if rows:
            w = weight.contiguous() if weight is not None else None
            b = bias.contiguous() if bias is not None else None
            _lib.call("noise_layer_norm_fwd", ptr(xr), ld, ptr(w), ptr(b), eps, ptr(y), ptr(mean), ptr(rstd), rows, D,
                      _lib.DTYPES[x.dtype], _lib.DTYPES[wdtype], _lib.stream(), nbytes=2 * x.numel() * x.element_size())
        return y, mean, rstd


def layer_norm_bwd(dy, x, mean, rstd, weight=None, need_params=True):
    """(dx, dweight, dbias) for the gradient dy of layer_norm_fwd's y; `weight` None and need_params: the gradients of a
    weight of ones and a bias of zeros, in fp32.  need_params False leaves both None and saves their reduction."""
    D, wdtype = _check(x, weight, None)
    _lib.no_tangents(dy, mean, rstd)
    _lib.require_cuda(dy, mean, rstd)
    if dy.shape != x.shape or dy.dtype != x.dtype:
        raise ValueError(f"dy must be {tuple(x.shape)} in {x.dtype}, got {tuple(dy.shape)} in {dy.dtype}")
    for name, s in (("mean", mean), ("rstd", rstd)):
        if s.shape != x.shape[:-1] or s.dtype != torch.float32:
            raise ValueError(f"{name} must be float32 {tuple(x.shape[:-1])}, got {s.dtype} {tuple(s.shape)}")
    with _lib.on_device(x, dy, mean, rstd, weight):
        xr, ldx = _rows(x, D)
        gr, ldg = _rows(dy, D)
        dx = x.new_empty(x.shape)
        rows = x.numel() // D
        dw = db = slab = None
        if need_params:
            dw, db = (x.new_empty(D, dtype=wdtype) for _ in range(2))
            if rows == 0:
                dw.zero_()
                db.zero_()
            else:
                slab = x.new_empty(_lib.lib.noise_layer_norm_bwd_rows(rows, D) * 2 * D, dtype=torch.float32)
        if rows:
            mean, rstd = mean.contiguous(), rstd.contiguous()
            w = weight.contiguous() if weight is not None else None
            _lib.call("noise_layer_norm_bwd", ptr(gr), ldg, ptr(xr), ldx, ptr(mean), ptr(rstd), ptr(w), ptr(dx), ptr(dw), ptr(db),
                      ptr(slab), rows, D, _lib.DTYPES[x.dtype], _lib.DTYPES[wdtype], _lib.stream(),
                      nbytes=3 * x.numel() * x.element_size())
        return dx, dw, db


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, mean, rstd = layer_norm_fwd(x, weight, bias, eps)
        ctx.save_for_backward(x, mean, rstd, weight)
        ctx.bias_dtype = None if bias is None else bias.dtype
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, mean, rstd, weight = ctx.saved_tensors
        need_w, need_b = ctx.needs_input_grad[1], ctx.needs_input_grad[2]
        dx, dw, db = layer_norm_bwd(dy, x, mean, rstd, weight, need_params=need_w or need_b)
        if need_b and db.dtype != ctx.bias_dtype:
            db = db.to(ctx.bias_dtype)      # a bias without a weight
        return dx, dw if need_w else None, db if need_b else None, None


def layer_norm(x, weight=None, bias=None, eps=1e-6):
    """LayerNorm of x (..., D) over its last axis; back-propagates into x, weight and bias."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias)):
        return _LayerNorm.apply(x, weight, bias, eps)
    return layer_norm_fwd(x, weight, bias, eps)[0]
