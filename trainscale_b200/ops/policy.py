"""Losses over token log-probabilities with their gradients: the clipped policy loss with a KL term, and the losses of (chosen,
rejected) pairs (csrc/posttrain.cu).

Loss and gradient come out of the same pass: the backward pass leaves the gradient alone where one flows into the loss, multiplies
an fp32 gradient by what does otherwise, and computes a 16-bit one again, which is then rounded once.  Reference behaviour:
data_pipeline/trainer/rl_training.py:297-430 and data_pipeline/trainer/loss/sota_losses.py:1151-1400.
"""
from __future__ import annotations

import functools
import math
import struct
from typing import NamedTuple

import torch
import torch.nn.functional as F

from . import _lib
from .logprob import _DTYPES, _address, _stream, fp32, gradient, on_this_gpu, ordinary

_MASKS = {torch.bool: 0, torch.uint8: 0, torch.int32: 1, torch.int64: 2, torch.float32: 3, torch.bfloat16: 4, torch.float16: 5}
REDUCTIONS = {"sequence": 0, "token": 1, "constant": 2}
KINDS = {"sigmoid": 0, "robust": 1, "hinge": 2, "ipo": 3}
_POLICY_CALL = struct.Struct("=14q5dqd6q")       # PolicyCall and PairsCall of csrc/posttrain.cu
_PAIRS_CALL = struct.Struct("=10q4d8q")


class PolicyStats(NamedTuple):
    """Means over the unmasked tokens, on the device: the KL estimate e^d - 1 - d with d = ref - logp (zero without a reference),
    the share of tokens whose objective was clipped, and the probability ratio to the old policy."""
    kl: torch.Tensor
    clip_fraction: torch.Tensor
    ratio: torch.Tensor


@functools.lru_cache(maxsize=None)
def _library():
    from ctypes import c_char_p, c_longlong, c_void_p
    lib = _lib.load("posttrain")
    lib.ts_policy_loss.argtypes = lib.ts_preference_loss.argtypes = [c_char_p, c_void_p]
    lib.ts_scale_by.argtypes = [c_void_p, c_void_p, c_longlong, c_void_p]
    lib.ts_policy_workspace.argtypes, lib.ts_policy_workspace.restype = [c_longlong, c_longlong], c_longlong
    return lib


def _place(x: torch.Tensor | None) -> tuple[int, int]:
    """Address and elements between rows."""
    return (0, 0) if x is None else (x.data_ptr(), x.stride(0))


def _rows_of(x: torch.Tensor) -> torch.Tensor:
    return x if x.stride(1) == 1 or x.shape[1] == 1 else x.contiguous()


def _one_type(first, *more):
    """Rows that are dense within themselves, all in the first one's type, or all in fp32 where they differ."""
    out = [first, *more]
    for t in more:
        if t is not None and t.dtype != first.dtype:
            out = [u if u is None else u.float() for u in out]
            break
    return [t if t is None else _rows_of(t) for t in out]


def _mask_of(mask: torch.Tensor) -> torch.Tensor:
    return _rows_of(mask if mask.dtype in _MASKS else mask.float())


def _gradient(p: torch.Tensor) -> torch.Tensor:
    return torch.empty_like(p, memory_format=torch.contiguous_format)


def _changed(tensors) -> tuple:
    return tuple([None if t is None or t.is_inference() else t._version for t in tensors])


class _Loss(torch.autograd.Function):
    """A loss whose kernel has already written its gradient.  The first backward pass hands that gradient out; one after it
    (retain_graph) or one captured without its forward computes it again, for the first buffer may have been changed since.

    `op(logp, *constants)` launches the kernel: it gives (loss, other results, gradient), with `grad` a buffer for the gradient or True
    for a new one, and the gradient alone, times `factor`, where that is given."""

    @staticmethod
    def forward(ctx, logp, op, *constants):
        loss, rest, ctx.grad = op(logp, *constants, grad=True)
        ctx.save_for_backward(logp)
        ctx.op, ctx.constants, ctx.versions, ctx.dtype = op, constants, _changed(constants), logp.dtype
        ctx.captured = torch._C._cuda_isCurrentStreamCapturing()
        if rest is not None:
            ctx.mark_non_differentiable(rest)
        ctx.set_materialize_grads(False)
        return loss, rest

    @staticmethod
    def backward(ctx, g, _):
        constants = ctx.constants
        none = (None,) * (1 + len(constants))
        if g is None:
            return None, *none
        kernel = ordinary(g)
        grad, ctx.grad = ctx.grad, None
        if ctx.captured != torch._C._cuda_isCurrentStreamCapturing():
            grad = None
        if grad is not None and grad.dtype is torch.float32 and kernel:
            _lib.check(_library().ts_scale_by(grad.data_ptr(), g.data_ptr(), grad.numel(), _stream()), "ts_scale_by")
        else:
            (logp,) = ctx.saved_tensors               # (refuses a freed graph, and log-probabilities changed since)
            if _changed(constants) != ctx.versions:
                raise RuntimeError("an input of a policy or preference loss was changed in place before its gradient was computed")
            if not kernel:
                return gradient(lambda x: ctx.op.plain(x, *constants)[0], logp, (g,)), *none
            grad = ctx.op(logp, *constants, grad=True if grad is None else grad, factor=g)[2]
        return grad if grad.dtype is ctx.dtype else grad.to(ctx.dtype), *none


def native(logp, *others) -> bool:
    """Whether the kernels take these log-probabilities: [rows, T], on the current device, with some tokens and no more than a launch
    counts."""
    shape = logp.shape
    return (len(shape) == 2 and logp.dtype in _DTYPES and 0 < shape[0] < 1 << 28 and 0 < shape[1] < 1 << 30
            and on_this_gpu(logp, *others))


def _run(op, logp, *constants):
    """(loss, other results): the constants get no gradient."""
    constants = tuple([t.detach() if t is not None and t.requires_grad else t for t in constants])
    if not native(logp, *constants):
        return op.plain(logp, *constants)
    if torch.is_grad_enabled() and logp.requires_grad:
        return _Loss.apply(logp, op, *constants)
    return op(logp, *constants)[:2]


def _masked(x: torch.Tensor, used: torch.Tensor) -> torch.Tensor:
    return x.where(used, 0.0)


# ------------------------------------------------------------------------------------------------ clipped policy loss
class PolicyLoss:
    """policy_loss(logp, old_logp, advantages, mask, ref_logp): see `rl.clipped_policy_loss`, which checks the arguments."""

    def __init__(self, low: float, high: float, beta: float, reduction: str, length: int | None, stats: bool):
        self.low, self.high, self.beta, self.reduction, self.length, self.stats = low, high, beta, reduction, length, stats

    def __call__(self, logp, old, advantages, mask, ref, grad=None, factor=None):
        p, old, ref = _one_type(logp, old, ref)
        mask = _mask_of(mask)
        if advantages.dtype is not torch.float32 or not advantages.is_contiguous():
            advantages = advantages.float().contiguous()
        B, T = p.shape
        lib, low, high = _library(), self.low, self.high
        loss = stats = work = None
        if factor is None:
            loss = fp32(p)
            if self.stats:
                stats = fp32(p, 3)
        out = _gradient(p) if grad is True else grad
        need = lib.ts_policy_workspace(B, T)
        if need:
            work = fp32(p, 2 * need)
        call = _POLICY_CALL.pack(
            _DTYPES[p.dtype], *_place(p), *_place(old), *_place(ref), advantages.data_ptr(), advantages.dim() == 2, *_place(mask),
            _MASKS[mask.dtype], B, T, math.log1p(-low) if low < 1 else -math.inf, math.log1p(high), 1 - low, 1 + high, self.beta,
            REDUCTIONS[self.reduction], 1.0 / (B * (self.length or T)), _address(out), _address(loss), _address(stats), _address(factor),
            grad is True, _address(work))
        _lib.check(lib.ts_policy_loss(call, _stream()), "ts_policy_loss")
        return loss, stats, out

    def plain(self, logp, old_logp, advantages, mask, ref_logp):
        """The same in PyTorch operations.  Masked tokens are replaced before anything is computed from them: whatever they hold
        reaches neither the loss nor a gradient."""
        used, m = mask != 0, mask.to(torch.float64 if logp.dtype == torch.float64 else torch.float32)
        m = _masked(m, used)
        logp, old = _masked(logp, used).to(m.dtype), _masked(old_logp, used).to(m.dtype)
        a = advantages if advantages.dim() == 2 else advantages.unsqueeze(1)
        a = _masked(a.to(m.dtype).expand(logp.shape), used)
        with torch.no_grad():
            moved = logp.double() - old.double()      # (fp32 could round it to the other side of a bound)
            clipped = ((a > 0) & (moved > math.log1p(self.high))) | ((a < 0) & (moved < (math.log1p(-self.low) if self.low < 1 else -math.inf)))
            idle = clipped | ((a == 0) & ~moved.isnan())
        # (0 * inf: a ratio that has no say may overflow, and so would its derivative: it is not taken)
        ratio = torch.exp((logp - old).where(~idle, 0.0))
        bound = torch.full_like(a, 1 - self.low).masked_fill(a > 0, 1 + self.high)
        token, kl = -a * bound.where(clipped, ratio), torch.zeros_like(logp)
        if ref_logp is not None:
            d = _masked(ref_logp, used).to(m.dtype) - logp
            kl = torch.expm1(d) - d
            if self.beta:                             # (0 * inf: a reference that is only looked at has no say)
                token = token + self.beta * kl
        total = m.sum().clamp(min=1)
        if self.reduction == "sequence":
            loss = ((token * m).sum(1) / m.sum(1).clamp(min=1)).sum() / max(1, m.shape[0])
        elif self.reduction == "token":
            loss = (token * m).sum() / total
        else:
            loss = (token * m).sum() / max(1, m.shape[0] * (self.length or m.shape[1]))
        with torch.no_grad():
            stats = torch.stack([(x.detach() * m).sum() / total for x in (kl, clipped.to(m.dtype), torch.exp(logp - old))])
        return loss, stats


def policy_loss(logp, old_logp, advantages, mask, ref_logp=None, low=0.2, high=0.2, beta=0.0, reduction="sequence", length=None,
                stats=False):
    """(loss, [kl, share of clipped tokens, ratio] if `stats`)."""
    return _run(PolicyLoss(low, high, beta, reduction, length, stats), logp, old_logp, advantages, mask, ref_logp)


# ------------------------------------------------------------------------------------------------ pairs
class PairLoss:
    """pair_loss(logp, ref_logp, mask): see `rl.preference_loss`, which checks the arguments."""

    def __init__(self, beta: float, kind: str, smoothing: float, gamma: float, normalized: bool, nll: float):
        self.beta, self.kind, self.smoothing, self.gamma, self.normalized, self.nll = beta, kind, smoothing, gamma, normalized, nll

    def __call__(self, logp, ref, mask, grad=None, factor=None):
        p, ref = _one_type(logp, ref)
        mask = _mask_of(mask)
        R, T = p.shape
        loss = rewards = None
        if factor is None:
            loss, rewards = fp32(p), fp32(p, R)
        out = _gradient(p) if grad is True else grad
        work = fp32(p, R)                             # R / 2 fp64 values
        call = _PAIRS_CALL.pack(
            _DTYPES[p.dtype], *_place(p), *_place(ref), *_place(mask), _MASKS[mask.dtype], R // 2, T, self.beta, self.gamma,
            self.smoothing, self.nll, KINDS[self.kind], self.normalized, _address(out), _address(loss), _address(rewards),
            _address(factor), grad is True, work.data_ptr())
        _lib.check(_library().ts_preference_loss(call, _stream()), "ts_preference_loss")
        return loss, rewards, out

    def plain(self, logp, ref_logp, mask):
        """The same in PyTorch operations, in fp64: scores are long sums whose difference decides."""
        P = logp.shape[0] // 2
        used, out = mask != 0, torch.float64 if logp.dtype == torch.float64 else torch.float32
        m = _masked(mask.double(), used)
        own = (_masked(logp, used).double() * m).sum(1)
        score = own if ref_logp is None else own - (_masked(ref_logp, used).double() * m).sum(1)
        count = m.sum(1).clamp(min=1)
        if self.normalized:
            score = score / count
        x = score[:P] - score[P:]
        q = self.beta * x - self.gamma
        eps, up = self.smoothing, F.softplus(-q, threshold=1e3)
        down = F.softplus(q, threshold=1e3) if eps else 0.0       # (0 * inf: a token of no probability)
        if self.kind == "sigmoid":
            loss = (1 - eps) * up + eps * down
        elif self.kind == "robust":
            loss = ((1 - eps) * up - eps * down) / (1 - 2 * eps)
        elif self.kind == "hinge":
            loss = torch.relu(1 - q)
        else:
            loss = (x - 0.5 / self.beta) ** 2
        if self.nll:
            loss = loss - self.nll * own[:P] / count[:P]
        return (loss.sum() / max(1, P)).to(out), (self.beta * score).detach().to(out)


def preference_loss(logp, ref_logp, mask, beta=0.1, kind="sigmoid", smoothing=0.0, gamma=0.0, normalized=False, nll=0.0):
    """(loss, rewards of all rows)."""
    return _run(PairLoss(beta, kind, smoothing, gamma, normalized, nll), logp, ref_logp, mask)
