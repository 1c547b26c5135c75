"""Log-probabilities of chosen tokens, and entropies, out of a model's logits (csrc/logprob.cu).

One pass over the logits forward (a running maximum with its sums) and one backward; logits stay in their type, everything else
is fp32.  Reference behaviour: data_pipeline/trainer/rl_training.py:95-191 (soft-cap, scale, temperature, in this order).
"""
from __future__ import annotations

import functools
import math

import torch

from . import _lib

_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_PLAIN = (torch.Tensor, torch.nn.Parameter)


def on_this_gpu(*tensors) -> bool:
    """Plain CUDA tensors of the current device (or None), outside functorch transforms and forward-mode differentiation."""
    for t in tensors:
        if t is not None and (type(t) not in _PLAIN or not t.is_cuda or t.get_device() != torch._C._cuda_getDevice()):
            return False
    return not torch._C._are_functorch_transforms_active() and torch.autograd.forward_ad._current_level < 0


def native(logits: torch.Tensor, labels: torch.Tensor) -> bool:
    return logits.dtype in _DTYPES and on_this_gpu(logits, labels) and logits.numel() > 0 and logits.shape[-1] < 1 << 31


def plain(logits, labels, factor: float, cap: float, ignore_index: int | None, entropy: bool):
    """The same in PyTorch operations, in fp32 (fp64 logits: fp64)."""
    z = logits if logits.dtype == torch.float64 else logits.float()
    if cap:
        z = cap * torch.tanh(z / cap)
    log_p = torch.log_softmax(z * factor, dim=-1)
    known = (labels >= 0) & (labels < logits.shape[-1])
    logp = log_p.gather(-1, labels.where(known, 0).long().unsqueeze(-1)).squeeze(-1).where(known, math.nan)
    used = torch.ones_like(known) if ignore_index is None else labels != ignore_index
    logp = logp.where(used, 0.0)
    if not entropy:
        return logp
    p = log_p.exp()
    return logp, -(p * log_p.where(p > 0, 0.0)).sum(-1).where(used, 0.0)


def _rows(logits: torch.Tensor):
    """The logits as (tensor, rows, rows of an inner run, its strides): up to three dimensions are read where they lie."""
    if logits.stride(-1) != 1 and logits.shape[-1] > 1:
        logits = logits.contiguous()
    if logits.dim() > 3:
        logits = logits.reshape(-1, *logits.shape[-2:])
    shape, stride = logits.shape, logits.stride()
    if logits.dim() == 3:
        return logits, shape[0] * shape[1], shape[1], stride[0], stride[1]
    if logits.dim() == 2:
        return logits, shape[0], shape[0], 0, stride[0]
    return logits, 1, 1, 0, 0


def _tail(rows, V, factor, cap, ignore_index, lenient=False):
    n, inner, outer_stride, inner_stride = rows
    ignore = -(1 << 63) if ignore_index is None else ignore_index
    return (n, inner, outer_stride, inner_stride, V, factor, cap, ignore, lenient, _lib.stream_ptr())


_fns: dict = {}


@functools.lru_cache(maxsize=None)
def _workspace():
    from ctypes import c_int, c_longlong
    fn = _lib.load("logprob").ts_logprob_workspace
    fn.argtypes, fn.restype = [c_longlong, c_int, c_int], c_longlong
    return fn


def _call(name: str, *args) -> None:
    fn = _fns.get(name)
    if fn is None:
        from ctypes import c_float, c_int, c_longlong, c_void_p
        fn = getattr(_lib.load("logprob"), name)
        shape = [c_longlong] * 4 + [c_int, c_float, c_float, c_longlong, c_int, c_void_p]
        fn.argtypes = [c_void_p, c_int] + [c_void_p] * 5 + ([c_longlong] if name == "ts_logprob_bwd" else []) + shape
        _fns[name] = fn
    _lib.check(fn(*args), name)


def _forward(logits, labels, factor, cap, ignore_index, entropy: bool, keep: bool):
    x, *rows = _rows(logits)
    f32 = dict(dtype=torch.float32, device=logits.device)
    logp = torch.empty(labels.shape, **f32)
    H = torch.empty(labels.shape, **f32) if entropy else None
    kept = torch.empty(labels.numel(), 4, **f32) if keep else None
    need = _workspace()(labels.numel(), x.shape[-1], _DTYPES[x.dtype])
    work = torch.empty(need, dtype=torch.uint8, device=logits.device) if need else None
    _call("ts_logprob_fwd", _lib.ptr(x), _DTYPES[x.dtype], _lib.ptr(labels), _lib.ptr(logp), _lib.ptr(H), _lib.ptr(kept),
          _lib.ptr(work), *_tail(rows, x.shape[-1], factor, cap, ignore_index))
    return logp, H, kept


def rows_forward(logits: torch.Tensor, labels: torch.Tensor, logp: torch.Tensor, kept: torch.Tensor | None, ignore_index: int) -> None:
    """logp [n] = log softmax(logits [n, V])[labels], kept [n, 4] for `rows_backward_`, of CUDA rows that are dense within themselves.
    Labels outside the vocabulary count as ignored."""
    n, V = logits.shape
    need = _workspace()(n, V, _DTYPES[logits.dtype])
    work = torch.empty(need, dtype=torch.uint8, device=logits.device) if need else None
    _call("ts_logprob_fwd", _lib.ptr(logits), _DTYPES[logits.dtype], _lib.ptr(labels), _lib.ptr(logp), None, _lib.ptr(kept), _lib.ptr(work),
          *_tail((n, n, 0, logits.stride(0)), V, 1.0, 0.0, ignore_index, True))


def rows_backward_(logits: torch.Tensor, labels: torch.Tensor, kept: torch.Tensor, g: torch.Tensor, ignore_index: int) -> None:
    """The logits become the gradient of (g * logp).sum()."""
    n, V = logits.shape
    _call("ts_logprob_bwd", _lib.ptr(logits), _DTYPES[logits.dtype], _lib.ptr(labels), _lib.ptr(kept), _lib.ptr(g), None, _lib.ptr(logits),
          logits.stride(0), *_tail((n, n, 0, logits.stride(0)), V, 1.0, 0.0, ignore_index, True))


class _TokenLogProbs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, labels, factor, cap, ignore_index, entropy):
        logp, H, kept = _forward(logits, labels, factor, cap, ignore_index, entropy, True)
        ctx.save_for_backward(logits, labels, kept)
        ctx.how = (factor, cap, ignore_index, entropy)
        ctx.set_materialize_grads(False)
        return (logp, H) if entropy else logp

    @staticmethod
    def backward(ctx, g, h=None):
        logits, labels, kept = ctx.saved_tensors
        factor, cap, ignore_index, entropy = ctx.how
        none = (None,) * 5
        if g is None and h is None:
            return None, *none
        if torch.is_grad_enabled():                      # this gradient will be differentiated itself
            out = plain(logits, labels, factor, cap, ignore_index, entropy)
            pairs = [(o, d) for o, d in zip(out if entropy else (out,), (g, h)) if d is not None]
            (grad,) = torch.autograd.grad([o for o, _ in pairs], logits, [d for _, d in pairs], create_graph=True)
            return grad, *none
        x, *rows = _rows(logits)
        grad = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
        g, h = (None if d is None else d.float().contiguous() for d in (g, h))
        _call("ts_logprob_bwd", _lib.ptr(x), _DTYPES[x.dtype], _lib.ptr(labels), _lib.ptr(kept), _lib.ptr(g), _lib.ptr(h),
              _lib.ptr(grad), x.shape[-1], *_tail(rows, x.shape[-1], factor, cap, ignore_index))
        return grad, *none


def token_log_probs(logits: torch.Tensor, labels: torch.Tensor, factor: float = 1.0, cap: float = 0.0,
                    ignore_index: int | None = -100, entropy: bool = False):
    """log softmax(factor * cap tanh(logits / cap))[labels] in fp32 (and the distribution's entropy)."""
    if labels.shape != logits.shape[:-1]:
        raise ValueError(f"labels of shape {tuple(labels.shape)} for logits of shape {tuple(logits.shape)}")
    if labels.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"labels are int64 or int32, not {labels.dtype}")
    if not logits.is_floating_point():
        raise TypeError(f"logits are floating point, not {logits.dtype}")
    if logits.shape[-1] == 0:
        raise ValueError("logits of an empty vocabulary")
    if not native(logits, labels):
        return plain(logits, labels, factor, cap, ignore_index, entropy)
    labels = labels.to(torch.int64).contiguous()
    if torch.is_grad_enabled() and logits.requires_grad:
        labels = labels.clone() if labels.is_inference() else labels      # (such tensors cannot be kept for a backward pass)
        return _TokenLogProbs.apply(logits, labels, factor, cap, ignore_index, entropy)
    logp, H, _ = _forward(logits, labels, factor, cap, ignore_index, entropy, False)
    return (logp, H) if entropy else logp
