"""Log-probabilities of chosen tokens, and entropies, out of a model's logits (csrc/logprob.cu).

One pass over the logits forward (a running maximum with its sums) and one backward; logits stay in their type, everything else
is fp32.  Reference behaviour: data_pipeline/trainer/rl_training.py:95-191 (soft-cap, scale, temperature, in this order).
"""
from __future__ import annotations

import functools
import math
import struct

import torch
from torch._C import _are_functorch_transforms_active, _len_torch_dispatch_stack
from torch._C._functorch import is_legacy_batchedtensor
from torch.autograd import forward_ad

from . import _lib

_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_PLAIN = (torch.Tensor, torch.nn.Parameter)
_CALL = struct.Struct("=14q2d2q")                # LogprobCall of csrc/logprob.cu
_NEVER = -(1 << 63)                              # no label: nothing is ignored


def on_this_gpu(*tensors) -> bool:
    """Plain CUDA tensors of the current device (or None), while operations only run (`_lib.eager`)."""
    if not _lib.eager():
        return False
    for t in tensors:
        if t is not None and (type(t) not in _PLAIN or not t.is_cuda or t.get_device() != torch._C._cuda_getDevice()):
            return False
    return True


def native(logits: torch.Tensor, labels: torch.Tensor) -> bool:
    """Whether the kernels take these: 16- or 32-bit logits on the current device, some of them, and no more rows than a launch counts."""
    return (logits.dtype in _DTYPES and on_this_gpu(logits, labels) and 0 < labels.numel() < 1 << 28 and 0 < logits.shape[-1] < 1 << 31)


def plain(logits, labels, factor: float, cap: float, ignore_index: int | None, entropy: bool):
    """The same in PyTorch operations, in fp32 (fp64 logits: fp64)."""
    z = logits if logits.dtype == torch.float64 else logits.float()
    if cap:
        z = cap * torch.tanh(z / cap)
    z = z * factor
    log_p = torch.log_softmax(z, dim=-1)
    known = (labels >= 0) & (labels < logits.shape[-1])
    chosen, top = labels.where(known, 0).long().unsqueeze(-1), z.detach().amax(-1)
    logp = log_p.gather(-1, chosen).squeeze(-1)
    # (beside a logit of +inf the others have no probability, as in the kernel; log_softmax says NaN)
    logp = logp.where(top != math.inf, z.gather(-1, chosen).squeeze(-1) - top).where(known, math.nan)
    used = torch.ones_like(known) if ignore_index is None else labels != ignore_index
    logp = logp.where(used, 0.0)
    if not entropy:
        return logp
    p = log_p.exp()
    return logp, -(p * log_p.where(p > 0, 0.0)).sum(-1).where(used, 0.0)


def _rows(logits: torch.Tensor):
    """The logits as a tensor, and (rows, rows of an inner run, its strides): up to three dimensions are read where they lie."""
    if logits.stride(-1) != 1 and logits.shape[-1] > 1:
        logits = logits.contiguous()
    if logits.dim() > 3:
        logits = logits.reshape(-1, *logits.shape[-2:])
    shape, stride = logits.shape, logits.stride()
    if len(shape) == 3:
        return logits, (shape[0] * shape[1], shape[1], stride[0], stride[1])
    return logits, (shape[0], shape[0], 0, stride[0]) if len(shape) == 2 else (1, 1, 0, 0)


@functools.lru_cache(maxsize=None)
def _library():
    from ctypes import c_char_p, c_int, c_longlong, c_void_p
    lib = _lib.load("logprob")
    lib.ts_logprob_fwd.argtypes = lib.ts_logprob_bwd.argtypes = [c_char_p, c_void_p]
    lib.ts_logprob_workspace.argtypes, lib.ts_logprob_workspace.restype = [c_longlong, c_longlong, c_int], c_longlong
    lib.few_rows = lib.ts_logprob_few_rows()         # fewer never need a workspace
    return lib


def _address(t: torch.Tensor | None) -> int:
    return 0 if t is None else t.data_ptr()


def _stream() -> int:
    return torch._C._cuda_getCurrentRawStream(torch._C._cuda_getDevice())


def fp32(x: torch.Tensor, *shape: int) -> torch.Tensor:
    """A new fp32 tensor where `x` is (spelling the type out costs a microsecond)."""
    return x.new_empty(shape) if x.dtype is torch.float32 else x.new_empty(shape, dtype=torch.float32)


def _run_forward(x, rows, labels, logp, H, kept, factor=1.0, cap=0.0, ignore_index=None, lenient=False) -> None:
    lib, V, kind = _library(), x.shape[-1], _DTYPES[x.dtype]
    need = lib.ts_logprob_workspace(rows[0], V, kind) if rows[0] >= lib.few_rows else 0
    work = fp32(x, need // 4) if need else None
    call = _CALL.pack(x.data_ptr(), kind, labels.data_ptr(), logp.data_ptr(), _address(H), _address(kept), _address(work), 0, 0, *rows, V,
                      factor, cap, _NEVER if ignore_index is None else ignore_index, lenient)
    _lib.check(lib.ts_logprob_fwd(call, _stream()), "ts_logprob_fwd")


def _run_backward(x, rows, labels, kept, g, h, grad, pitch, factor=1.0, cap=0.0, ignore_index=None, lenient=False) -> None:
    call = _CALL.pack(x.data_ptr(), _DTYPES[x.dtype], labels.data_ptr(), _address(g), _address(h), kept.data_ptr(), 0, grad.data_ptr(), pitch,
                      *rows, x.shape[-1], factor, cap, _NEVER if ignore_index is None else ignore_index, lenient)
    _lib.check(_library().ts_logprob_bwd(call, _stream()), "ts_logprob_bwd")


def _forward(logits, labels, how, entropy: bool, keep: bool):
    x, rows = _rows(logits)
    logp = fp32(x, *labels.shape)
    H = fp32(x, *labels.shape) if entropy else None
    kept = fp32(x, rows[0], 4) if keep else None
    _run_forward(x, rows, labels, logp, H, kept, *how)
    return logp, H, kept


def rows_forward(logits: torch.Tensor, labels: torch.Tensor, logp: torch.Tensor, kept: torch.Tensor | None, ignore_index: int) -> None:
    """logp [n] = log softmax(logits [n, V])[labels], kept [n, 4] for `rows_backward_`, of rows on the current GPU that are dense within
    themselves.  Labels outside the vocabulary count as ignored."""
    n, pitch = logits.shape[0], logits.stride(0)
    _run_forward(logits, (n, n, 0, pitch), labels, logp, None, kept, ignore_index=ignore_index, lenient=True)


def rows_backward_(logits: torch.Tensor, labels: torch.Tensor, kept: torch.Tensor, g: torch.Tensor, ignore_index: int) -> None:
    """The logits become the gradient of (g * logp).sum()."""
    n, pitch = logits.shape[0], logits.stride(0)
    _run_backward(logits, (n, n, 0, pitch), labels, kept, g, None, logits, pitch, ignore_index=ignore_index, lenient=True)


def ordinary(grad: torch.Tensor | None) -> bool:
    """Whether a backward pass only runs, once, for this gradient: not for several at once (is_grads_batched, jacobian(vectorize=True)),
    recorded or transformed, nor differentiated itself.  (Traces and compiled functions have no kernel's node to run; one call here, for
    it costs more in autograd's thread than elsewhere.)"""
    return not (torch.is_grad_enabled() or _len_torch_dispatch_stack() or _are_functorch_transforms_active() or forward_ad._current_level >= 0
                or (grad is not None and is_legacy_batchedtensor(grad)))


def gradient(form, x: torch.Tensor, upstream) -> torch.Tensor:
    """The gradient in `x` of results of PyTorch operations, form(x), where some of `upstream` flows into them: for a backward pass
    that is recorded or transformed, runs for several gradients at once, or will be differentiated itself."""
    again = torch.is_grad_enabled()
    with torch.enable_grad():
        x = x if again else x.detach().requires_grad_()
        out = form(x)
        pairs = [(o, d) for o, d in zip(out if isinstance(out, tuple) else (out,), upstream) if d is not None]
        return torch.autograd.grad([o for o, _ in pairs], x, [d for _, d in pairs], create_graph=again)[0]


class _TokenLogProbs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, labels, how, entropy):
        logp, H, kept = _forward(logits, labels, how, entropy, True)
        ctx.save_for_backward(logits, labels, kept)
        ctx.how, ctx.entropy = how, entropy
        ctx.set_materialize_grads(False)
        return (logp, H) if entropy else logp

    @staticmethod
    def backward(ctx, g, h=None):
        logits, labels, kept = ctx.saved_tensors
        if g is None and h is None:
            return None, None, None, None
        if not (ordinary(g) and ordinary(h)):
            return gradient(lambda x: plain(x, labels, *ctx.how, ctx.entropy), logits, (g, h)), None, None, None
        x, rows = _rows(logits)
        grad = torch.empty_like(logits, memory_format=torch.contiguous_format)
        g, h = (None if d is None else d.float().contiguous() for d in (g, h))
        _run_backward(x, rows, labels, kept, g, h, grad, x.shape[-1], *ctx.how)
        return grad, None, None, None


def token_log_probs(logits: torch.Tensor, labels: torch.Tensor, factor: float = 1.0, cap: float = 0.0,
                    ignore_index: int | None = -100, entropy: bool = False):
    """log softmax(factor * cap tanh(logits / cap))[labels] in fp32 (and the distribution's entropy)."""
    shape, kind = logits.shape, labels.dtype
    if labels.shape != shape[:-1]:
        raise ValueError(f"labels of shape {tuple(labels.shape)} for logits of shape {tuple(shape)}")
    if kind is not torch.int64 and kind is not torch.int32:
        raise TypeError(f"labels are int64 or int32, not {kind}")
    if not logits.is_floating_point():
        raise TypeError(f"logits are floating point, not {logits.dtype}")
    if shape[-1] == 0:
        raise ValueError("logits of an empty vocabulary")
    how = (factor, cap, ignore_index)
    if not native(logits, labels):
        return plain(logits, labels, *how, entropy)
    if kind is not torch.int64 or not labels.is_contiguous():
        labels = labels.to(torch.int64).contiguous()
    if logits.requires_grad and torch.is_grad_enabled():
        labels = labels.clone() if labels.is_inference() else labels      # (such tensors cannot be kept for a backward pass)
        return _TokenLogProbs.apply(logits, labels, how, entropy)
    logp, H, _ = _forward(logits, labels, how, entropy, False)
    return (logp, H) if entropy else logp
