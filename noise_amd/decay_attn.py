"""Decay attention: causal linear attention with a decay for each head, on the kernels of csrc/decay_attn.hip.

    S_t = exp(log_decay) S_{t-1} + k_t (x) v_t          o_t = scale * q_t S_t

Next to the softmax attention of the models' bottleneck (train/models.py:14-36), which needs every token of a clip at
once, this one carries a state of fixed size: whole clips run in chunks, a stream runs token by token from the same state.

    o, state = decay_attention(q, k, v, log_decay)                            # clips; differentiable in q, k, v and state
    o, state = decay_attention(q, k, v, log_decay, state, lengths=lengths)    # the next piece of a padded batch
    o = decay_attention_step(q, k, v, log_decay, state)                       # one token per stream, state updated in place
    o, end = decay_attention_fwd(...)                                         # explicit passes
    dq, dk, dv, d_state = decay_attention_bwd(do, q, k, v, log_decay, state, lengths, d_state=d_end)

q and k are (B, T, H, Dk), v is (B, T, H, Dv) with head sizes of 1 to 128, all fp32, bf16 or fp16 with any strides (views of one
packed projection are read in place; a last axis without unit stride is copied first).  `log_decay` is (H,) fp32, at most 0
(-inf: no memory), and takes no gradient (one that requires it is refused while gradients are recorded).  States are
(B, H, Dk, Dv) fp32.  `lengths` (B,) int32 or int64 on the GPU (below zero means 0, above T means T): the tokens of clip b at
and behind lengths[b] are neither read nor added to the state, their rows of o and of the gradients are zero, and the state
returned is the one behind the last real token.  `scale` defaults to Dk ** -0.5.

Numbers: states are carried in fp32 accuracy whatever the tokens' type, and in 16-bit types o, dq, dk and dv are rounded to the type
once: the weights inside a chunk and the state as it meets q enter the products with at least 15 bits of fraction.  In fp16 that
holds within 2^18 of the largest value that 16 neighbouring columns of a state may hold by its bound, the decayed sum of
max |k| max |v|, and one bit less for each factor of two beyond.  A token that is not finite reaches what the formulas say: its
column and later tokens, or all columns where it is one of k or q; an infinity may come out as a NaN.
"""
import ctypes

import torch

from . import _lib
from ._lib import _F, _I, _L, _P, ptr

_lib.register({
    "noise_decay_attn_fwd": [_P] * 10 + [_F] + [_I] * 6 + [_P],
    "noise_decay_attn_bwd": [_P] * 14 + [_F] + [_I] * 6 + [_P],
    "noise_decay_attn_step": [_P] * 7 + [_F] + [_I] * 5 + [_P],
    "noise_decay_attn_workspace": [_I] * 7,
})
_lib.lib.noise_decay_attn_workspace.restype = _L

MAX_HEAD = 128
MAX_TOKENS, MAX_PAIRS = 1 << 30, 1 << 22      # of clips; single tokens take twice the pairs


def _unit(t):
    """t itself when its last axis has unit stride, a packed copy otherwise."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _tokens(t):
    """(t, its strides) as the walk reads them: unit stride in a row, rows apart and within reach; a packed copy otherwise (a
    broadcast token axis, overlapping windows).  The stride of an axis of one token says nothing."""
    t = _unit(t)
    b, s, h, _ = t.stride()
    if t.shape[1] == 1:
        s = t.shape[-1]
    if not t.shape[-1] <= s < 1 << 22:
        t = t.contiguous()
        b, s, h, _ = t.stride()
    return t, (b, s, h)


def _check(q, k, v, log_decay, state, tokens):
    _lib.no_tangents(q, k, v, log_decay, state)
    _lib.require_cuda(q, k, v, log_decay, state)
    qs, vs, dims = q.shape, v.shape, 4 if tokens else 3
    if len(qs) != dims or k.shape != qs or len(vs) != dims or vs[:-1] != qs[:-1]:
        raise ValueError(f"q, k must be {'(B, T, H, Dk)' if tokens else '(B, H, Dk)'} and v the same with Dv: got {tuple(q.shape)}, "
                         f"{tuple(k.shape)}, {tuple(v.shape)}")
    if q.dtype not in _lib.DTYPES or k.dtype != q.dtype or v.dtype != q.dtype:
        raise TypeError(f"q, k, v must share one of float32, bfloat16, float16: got {q.dtype}, {k.dtype}, {v.dtype}")
    B, H, dk, dv = qs[0], qs[-2], qs[-1], vs[-1]
    if B * H > (MAX_PAIRS if tokens else 2 * MAX_PAIRS) or tokens and qs[1] > MAX_TOKENS:      # sizes travel as 32-bit numbers
        raise ValueError(f"too many tokens or (clip, head) pairs for one call: {tuple(qs)}")
    if not (1 <= dk <= MAX_HEAD and 1 <= dv <= MAX_HEAD):
        raise ValueError(f"head sizes of 1 to {MAX_HEAD} are supported, got {dk} and {dv}")
    if log_decay.shape != (H,) or log_decay.dtype != torch.float32:
        raise ValueError(f"log_decay must be float32 ({H},), got {log_decay.dtype} {tuple(log_decay.shape)}")
    _check_state("state", state, (B, H, dk, dv))
    return B, H, dk, dv


def _check_state(name, state, shape):
    if state is not None and (state.shape != shape or state.dtype != torch.float32):
        raise ValueError(f"{name} must be float32 {shape}, got {state.dtype} {tuple(state.shape)}")


def _check_lengths(lengths, B, T):
    if lengths is None:
        return None
    _lib.require_cuda(lengths)
    if tuple(lengths.shape) != (B,) or lengths.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"lengths must be ({B},) integers, got {lengths.dtype} {tuple(lengths.shape)}")
    if lengths.dtype == torch.int64:
        lengths = lengths.clamp(0, T)       # the kernels' own limits, before the type loses the high bits
    return lengths.to(torch.int32).contiguous()


def _workspace(q, dv, backward):
    B, T, H, dk = q.shape
    n = _lib.lib.noise_decay_attn_workspace(B, T, H, dk, dv, _lib.DTYPES[q.dtype], backward)
    return q.new_empty(n, dtype=torch.float32) if n else None


def decay_attention_fwd(q, k, v, log_decay, state=None, lengths=None, scale=None):
    """(o, state behind the last token): o (B, T, H, Dv) in q's type, the state a new fp32 tensor."""
    B, H, dk, dv = _check(q, k, v, log_decay, state, True)
    lengths = _check_lengths(lengths, B, q.shape[1])
    scale = dk ** -0.5 if scale is None else float(scale)
    with _lib.on_device(q, k, v, log_decay, state, lengths):
        if q.numel() == 0:      # no token: the state as it was
            end = q.new_empty(B, H, dk, dv, dtype=torch.float32)
            end.copy_(state) if state is not None else end.zero_()
            return torch.empty(v.shape, device=v.device, dtype=v.dtype), end
        end = q.new_empty(B, H, dk, dv, dtype=torch.float32)
        x0 = state.contiguous() if state is not None else None
        T, g, ws = q.shape[1], log_decay.contiguous(), _workspace(q, dv, 0)
        (q, sq), (k, sk), (v, sv) = _tokens(q), _tokens(k), _tokens(v)
        o = q.new_empty(B, T, H, dv)
        strides = (_L * 12)(*sq, *sk, *sv, T * H * dv, H * dv, dv)
        _lib.call("noise_decay_attn_fwd", ptr(q), ptr(k), ptr(v), ptr(o), strides, ptr(g), ptr(lengths), ptr(x0), ptr(end), ptr(ws),
                  scale, B, T, H, dk, dv, _lib.DTYPES[q.dtype], _lib.stream(), nbytes=2 * q.element_size() * (q.numel() + v.numel()))
        return o, end


def decay_attention_bwd(do, q, k, v, log_decay, state=None, lengths=None, scale=None, d_state=None):
    """(dq, dk, dv, gradient of `state`) for the gradients `do` of o and `d_state` of the returned state (None: zero)."""
    B, H, dk, dv = _check(q, k, v, log_decay, state, True)
    lengths = _check_lengths(lengths, B, q.shape[1])
    _lib.no_tangents(do, d_state)
    _lib.require_cuda(do, d_state)
    if do.shape != v.shape or do.dtype != v.dtype:
        raise ValueError(f"do must be {tuple(v.shape)} in {v.dtype}, got {tuple(do.shape)} in {do.dtype}")
    _check_state("d_state", d_state, (B, H, dk, dv))
    scale = dk ** -0.5 if scale is None else float(scale)
    with _lib.on_device(q, do, k, v, log_decay, state, lengths, d_state):
        d0 = q.new_empty(B, H, dk, dv, dtype=torch.float32)
        if q.numel() == 0:
            d0.copy_(d_state) if d_state is not None else d0.zero_()
            return torch.empty_like(q), torch.empty_like(k), torch.empty_like(v), d0
        g = log_decay.contiguous()
        x0 = state.contiguous() if state is not None else None
        x1 = d_state.contiguous() if d_state is not None else None
        T, ws = q.shape[1], _workspace(q, dv, 1)
        (do, so), (q, sq), (k, sk), (v, sv) = _tokens(do), _tokens(q), _tokens(k), _tokens(v)
        gq, gk, gv = q.new_empty(B, T, H, dk), q.new_empty(B, T, H, dk), q.new_empty(B, T, H, dv)
        narrow, wide = (T * H * dk, H * dk, dk), (T * H * dv, H * dv, dv)
        strides = (_L * 21)(*so, *sq, *sk, *sv, *narrow, *narrow, *wide)
        _lib.call("noise_decay_attn_bwd", ptr(do), ptr(q), ptr(k), ptr(v), ptr(gq), ptr(gk), ptr(gv), strides, ptr(g), ptr(lengths),
                  ptr(x0), ptr(x1), ptr(d0), ptr(ws), scale, B, T, H, dk, dv, _lib.DTYPES[q.dtype], _lib.stream(),
                  nbytes=q.element_size() * (4 * q.numel() + 3 * v.numel()))
        return gq, gk, gv, d0


class _DecayAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, log_decay, state, lengths, scale):
        ctx.save_for_backward(q, k, v, log_decay, state, lengths)
        ctx.scale = scale
        return decay_attention_fwd(q, k, v, log_decay, state, lengths, scale)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, do, d_end):
        q, k, v, log_decay, state, lengths = ctx.saved_tensors
        dq, dk, dv, d_state = decay_attention_bwd(do, q, k, v, log_decay, state, lengths, ctx.scale, d_end)
        return dq, dk, dv, None, d_state if state is not None else None, None, None


def decay_attention(q, k, v, log_decay, state=None, lengths=None, scale=None):
    """(o, state behind the last token); back-propagates into q, k, v and state."""
    if log_decay.requires_grad and torch.is_grad_enabled():
        raise ValueError("log_decay takes no gradient: detach it")
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, v, state)):
        return _DecayAttention.apply(q, k, v, log_decay, state, lengths, scale)
    return decay_attention_fwd(q, k, v, log_decay, state, lengths, scale)


def decay_attention_step(q, k, v, log_decay, state, scale=None, out=None):
    """One token per stream: q, k (B, H, Dk), v (B, H, Dv); `state` (B, H, Dk, Dv) fp32, packed, is updated in place.  Returns
    o (B, H, Dv) (`out` when given; it may be q, k or v, but no other part of an argument).  No gradient."""
    if state is None:
        raise ValueError("decay_attention_step needs the streams' state")
    B, H, dk, dv = _check(q, k, v, log_decay, state, False)
    if not state.is_contiguous():
        raise ValueError("state must be packed: it is updated in place")
    if torch.is_grad_enabled() and any(t.requires_grad for t in (q, k, v, state)):
        raise RuntimeError("decay_attention_step has no backward pass: call it under torch.no_grad() or detach its inputs")
    if out is None:
        out = q.new_empty(B, H, dv)
    elif tuple(out.shape) != (B, H, dv) or out.dtype != q.dtype or not out.is_contiguous():
        raise ValueError(f"out must be a packed {q.dtype} {(B, H, dv)}, got {out.dtype} {tuple(out.shape)}")
    scale = dk ** -0.5 if scale is None else float(scale)
    with _lib.on_device(q, k, v, log_decay, state, out):
        if B * H:
            q, k, v, g = _unit(q), _unit(k), _unit(v), log_decay.contiguous()
            strides = (_L * 6)(*q.stride()[:2], *k.stride()[:2], *v.stride()[:2])
            _lib.call("noise_decay_attn_step", ptr(q), ptr(k), ptr(v), strides, ptr(g), ptr(state), ptr(out),
                      scale, B, H, dk, dv, _lib.DTYPES[q.dtype], _lib.stream(), nbytes=8 * state.numel())
    _lib.written(state, out)
    return out
