"""Losses over token log-probabilities with their gradients: the clipped policy loss with a KL term, and the losses of (chosen,
rejected) pairs (csrc/posttrain.cu).

Loss and gradient come out of the same pass: the backward pass leaves the gradient alone where one flows into the loss, multiplies
an fp32 gradient by what does otherwise, and computes a 16-bit one again, which is then rounded once.  Reference behaviour: data_pipeline/trainer/rl_training.py:297-430 and
data_pipeline/trainer/loss/sota_losses.py:1151-1400.
"""
from __future__ import annotations

import math
from typing import NamedTuple

import torch
import torch.nn.functional as F

from . import _lib
from .logprob import _DTYPES, on_this_gpu

_MASKS = {torch.bool: 0, torch.uint8: 0, torch.int32: 1, torch.int64: 2, torch.float32: 3, torch.bfloat16: 4, torch.float16: 5}
REDUCTIONS = {"sequence": 0, "token": 1, "constant": 2}
KINDS = {"sigmoid": 0, "robust": 1, "hinge": 2, "ipo": 3}


class PolicyStats(NamedTuple):
    """Means over the unmasked tokens, on the device: the KL estimate e^d - 1 - d with d = ref - logp (zero without a reference),
    the share of tokens whose objective was clipped, and the probability ratio to the old policy."""
    kl: torch.Tensor
    clip_fraction: torch.Tensor
    ratio: torch.Tensor


_fns: dict = {}


def _fn(name: str):
    fn = _fns.get(name)
    if fn is None:
        from ctypes import c_double as d, c_int as i, c_longlong as n, c_void_p as p
        lib = _lib.load("posttrain")
        types = {"ts_policy_loss": [i, p, n, p, n, p, n, p, i, p, n, i, n, n, d, d, d, d, d, i, d, p, p, p, p, i, p, p],
                 "ts_preference_loss": [i, p, n, p, n, p, n, i, n, n, d, d, d, d, i, i, p, p, p, p, i, p, p],
                 "ts_scale_by": [p, p, n, p], "ts_policy_workspace": [n, n]}
        for k, t in types.items():
            _fns[k] = getattr(lib, k)
            _fns[k].argtypes = t
        _fns["ts_policy_workspace"].restype = n
        fn = _fns[name]
    return fn


def _rows_of(x: torch.Tensor) -> torch.Tensor:
    return x if x.stride(1) == 1 or x.shape[1] == 1 else x.contiguous()


def _masked(x: torch.Tensor, used: torch.Tensor) -> torch.Tensor:
    return x.where(used, 0.0)


class _Loss(torch.autograd.Function):
    """A loss whose kernel has already written its gradient.  The first backward pass hands that gradient out; one after it
    (retain_graph) or one captured without its forward computes it again, for the first buffer may have been changed since."""

    @staticmethod
    def forward(ctx, logp, kernel, plain, *constants):
        loss, rest, ctx.grad = kernel(logp, *constants, grad=True)
        ctx.save_for_backward(logp, *constants)
        ctx.kernel, ctx.plain = kernel, plain
        ctx.captured = torch.cuda.is_current_stream_capturing()
        ctx.mark_non_differentiable(rest)
        ctx.set_materialize_grads(False)
        return loss, rest

    @staticmethod
    def backward(ctx, g, _):
        logp, *constants = ctx.saved_tensors          # (refuses a freed graph, and inputs that were changed since)
        none = (None,) * (2 + len(constants))
        if g is None:
            return None, *none
        if torch.is_grad_enabled():                   # this gradient will be differentiated itself
            return torch.autograd.grad(ctx.plain(logp, *constants)[0], logp, g, create_graph=True)[0], *none
        grad, ctx.grad = ctx.grad, None
        if ctx.captured != torch.cuda.is_current_stream_capturing():
            grad = None
        if grad is not None and grad.dtype == torch.float32:
            _lib.check(_fn("ts_scale_by")(_lib.ptr(grad), _lib.ptr(g), grad.numel(), _lib.stream_ptr()), "ts_scale_by")
        else:
            grad = ctx.kernel(logp, *constants, grad=True if grad is None else grad, factor=g)[2]
        return grad.to(logp.dtype), *none


def _run(logp, kernel, plain, *constants):
    constants = tuple(None if t is None else t.detach() for t in constants)
    if not native(logp, *constants):
        return plain(logp, *constants)
    if torch.is_grad_enabled() and logp.requires_grad:
        return _Loss.apply(logp, kernel, plain, *constants)
    return kernel(logp, *constants)[:2]


def native(logp, *others) -> bool:
    """Whether the kernels take these log-probabilities: [rows, T], on the current device, with some tokens."""
    return logp.dim() == 2 and logp.numel() > 0 and logp.dtype in _DTYPES and on_this_gpu(logp, *(t for t in others if t is not None))


def _one_type(*tensors):
    """Rows that are dense within themselves, all in the first one's type, or all in fp32 where they differ."""
    same = all(t is None or t.dtype == tensors[0].dtype for t in tensors)
    return [t if t is None else _rows_of(t if same else t.float()) for t in tensors]


def _mask_of(mask):
    return _rows_of(mask if mask.dtype in _MASKS else mask.float())


def _strided(t):
    return (_lib.ptr(t), 0 if t is None else t.stride(0))


def _outputs(p, rest: int, grad, factor):
    """(loss, other results, gradient buffer in the type that is computed in): no results where a gradient is formed again."""
    new = lambda *shape: torch.empty(shape, dtype=torch.float32, device=p.device)      # noqa: E731
    buffer = torch.empty(p.shape, dtype=p.dtype, device=p.device) if grad is True else grad
    return (new(), new(rest), buffer) if factor is None else (None, None, buffer)


# ------------------------------------------------------------------------------------------------ clipped policy loss
def policy_plain(logp, old_logp, advantages, mask, ref_logp, low, high, beta, reduction, length):
    """The same in PyTorch operations.  Masked tokens are replaced before anything is computed from them: whatever they hold
    reaches neither the loss nor a gradient."""
    used, m = mask != 0, mask.to(torch.float64 if logp.dtype == torch.float64 else torch.float32)
    m = _masked(m, used)
    logp, old = _masked(logp, used).to(m.dtype), _masked(old_logp, used).to(m.dtype)
    a = advantages if advantages.dim() == 2 else advantages.unsqueeze(1)
    a = _masked(a.to(m.dtype).expand(logp.shape), used)
    ratio = torch.exp(logp - old)
    gain = torch.minimum(ratio * a, ratio.clamp(1 - low, 1 + high) * a)
    clipped = ((a > 0) & (ratio > 1 + high)) | ((a < 0) & (ratio < 1 - low))
    token, kl = -gain, torch.zeros_like(gain)
    if ref_logp is not None:
        d = _masked(ref_logp, used).to(m.dtype) - logp
        kl = torch.expm1(d) - d
        token = token + beta * kl
    total = m.sum().clamp(min=1)
    if reduction == "sequence":
        loss = ((token * m).sum(1) / m.sum(1).clamp(min=1)).sum() / max(1, m.shape[0])
    elif reduction == "token":
        loss = (token * m).sum() / total
    else:
        loss = (token * m).sum() / max(1, m.shape[0] * length)
    with torch.no_grad():
        stats = torch.stack([(x.detach() * m).sum() / total for x in (kl, clipped.to(m.dtype), ratio)])
    return loss, stats


def policy_loss(logp, old_logp, advantages, mask, ref_logp=None, low=0.2, high=0.2, beta=0.0, reduction="sequence", length=None):
    """(loss, [kl, share of clipped tokens, ratio]); arguments checked by the caller."""
    length = length or logp.shape[1]

    def kernel(logp, old, advantages, mask, ref, grad=None, factor=None):
        p, old, ref = _one_type(logp.detach(), old, ref)
        mask, advantages = _mask_of(mask), advantages.float().contiguous()
        loss, stats, g = _outputs(p, 3, grad, factor)
        B, T = p.shape
        work = torch.empty(_fn("ts_policy_workspace")(B, T), dtype=torch.float64, device=p.device)
        rc = _fn("ts_policy_loss")(
            _DTYPES[p.dtype], *_strided(p), *_strided(old), *_strided(ref), _lib.ptr(advantages), int(advantages.dim() == 2),
            *_strided(mask), _MASKS[mask.dtype], B, T, math.log1p(-low) if low < 1 else -math.inf, math.log1p(high), 1 - low, 1 + high,
            beta, REDUCTIONS[reduction], 1.0 / (B * length), _lib.ptr(g), _lib.ptr(loss), _lib.ptr(stats), _lib.ptr(factor),
            int(grad is True), _lib.ptr(work), _lib.stream_ptr())
        _lib.check(rc, "ts_policy_loss")
        return loss, stats, g

    def plain(logp, old, advantages, mask, ref):
        return policy_plain(logp, old, advantages, mask, ref, low, high, beta, reduction, length)

    return _run(logp, kernel, plain, old_logp, advantages, mask, ref_logp)


# ------------------------------------------------------------------------------------------------ pairs
def preference_plain(logp, ref_logp, mask, beta, kind, smoothing, gamma, normalized, nll):
    """The same in PyTorch operations, in fp64: scores are long sums whose difference decides."""
    P = logp.shape[0] // 2
    used, out = mask != 0, torch.float64 if logp.dtype == torch.float64 else torch.float32
    m = _masked(mask.double(), used)
    v = _masked(logp, used).double()
    own = (v * m).sum(1)
    score = own if ref_logp is None else own - (_masked(ref_logp, used).double() * m).sum(1)
    count = m.sum(1).clamp(min=1)
    if normalized:
        score = score / count
    x = score[:P] - score[P:]
    q = beta * x - gamma
    up, down = F.softplus(-q, threshold=1e3), F.softplus(q, threshold=1e3)
    if kind == "sigmoid":
        loss = (1 - smoothing) * up + smoothing * down
    elif kind == "robust":
        loss = ((1 - smoothing) * up - smoothing * down) / (1 - 2 * smoothing)
    elif kind == "hinge":
        loss = torch.relu(1 - q)
    else:
        loss = (x - 0.5 / beta) ** 2
    if nll:
        loss = loss - nll * own[:P] / count[:P]
    loss = loss.sum() / max(1, P)
    return loss.to(out), (beta * score).detach().to(out)


def preference_loss(logp, ref_logp, mask, beta=0.1, kind="sigmoid", smoothing=0.0, gamma=0.0, normalized=False, nll=0.0):
    """(loss, rewards of all rows); arguments checked by the caller."""
    def kernel(logp, ref, mask, grad=None, factor=None):
        p, ref = _one_type(logp.detach(), ref)
        R, T = p.shape
        mask = _mask_of(mask)
        loss, rewards, g = _outputs(p, R, grad, factor)
        work = torch.empty(R // 2, dtype=torch.float64, device=p.device)
        rc = _fn("ts_preference_loss")(
            _DTYPES[p.dtype], *_strided(p), *_strided(ref), *_strided(mask), _MASKS[mask.dtype], R // 2, T, beta, gamma, smoothing, nll,
            KINDS[kind], int(normalized), _lib.ptr(g), _lib.ptr(loss), _lib.ptr(rewards), _lib.ptr(factor), int(grad is True), _lib.ptr(work), _lib.stream_ptr())
        _lib.check(rc, "ts_preference_loss")
        return loss, rewards, g

    def plain(logp, ref, mask):
        return preference_plain(logp, ref, mask, beta, kind, smoothing, gamma, normalized, nll)

    return _run(logp, kernel, plain, ref_logp, mask)
