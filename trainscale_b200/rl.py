"""RL / preference-training utilities and the preference trainer (DPO / SimPO / ORPO / KTO / CPO).

Utilities after data_pipeline/trainer/rl_training.py:95-671 (`selective_log_softmax`, `chunked_log_softmax`,
`compute_advantages` (group-normalised), `grpo_loss`, `drgrpo_loss`, `dapo_loss`, `left_pack_padding`, `GRPOCompute`,
`RewardModel`).  The reference ships the data stage and the losses but no preference training loop
(data_pipeline/trainer/loss/sota_losses.py:1151, preprocessing/prompt_engine.py:1929); `PreferenceTrainer` is that
loop: policy (and a frozen reference copy) under the flat engine, chosen and rejected sequences concatenated into
one forward, per-token log-probs from the fused lm_head + log-prob kernel (logits never materialised).

`token_log_probs`, `clipped_policy_loss` and `preference_loss` are the kernels under them (csrc/logprob.cu, csrc/posttrain.cu):
logits to log-probabilities and entropies, log-probabilities to a policy loss, and to the loss of (chosen, rejected) pairs.  On the
CPU, and for what the kernels do not take, they are PyTorch operations with the same meaning.
"""
from __future__ import annotations

import copy
import math
from typing import Any, Dict

import torch
import torch.nn as nn
import torch.nn.functional as F
from torch.nn.modules.module import _has_any_global_hook

from .losses import CPOLoss, DPOLoss, KTOLoss, ORPOLoss, SimPOLoss
from .ops import cross_entropy as ce_ops
from .ops import logprob as lp_ops
from .ops import policy as policy_ops
from .ops.policy import PolicyStats
from .utils.refargs import ANY, reference_kwargs


def _takes_transforms(temperature, cap, scale) -> bool:
    """Whether `token_log_probs` takes these: finite, and their product within the range of fp32."""
    if not (0 < temperature < math.inf and 0 <= cap < math.inf and 0 <= scale < math.inf):
        return False
    factor = (scale or 1.0) / temperature
    return 1e-30 < factor < 1e30 and factor * (cap or 1.0) < 1e30


def token_log_probs(logits: torch.Tensor, labels: torch.Tensor, *, temperature: float = 1.0, logit_softcapping: float = 0.0,
                    logit_scale: float = 0.0, ignore_index: int | None = -100, return_entropy: bool = False):
    """log p(labels) under `logits` [..., V] in fp32, shape of `labels` [...]; differentiable in the logits.

    Transforms of the logits, in this order: soft-cap c tanh(z / c), scale, divide by the temperature (0 switches the first two off).
    Rows whose label is `ignore_index` give 0 and no gradient, and are not read; a label outside the vocabulary gives NaN.
    `return_entropy`: (log-probabilities, entropy of each row's distribution), both differentiable; logits of -inf are tokens of no
    probability.  bf16, fp16 and fp32 logits with rows that are dense within themselves (also of a slice such as `logits[:, :-1]`) are
    read in place, once in each direction."""
    if not (0 < temperature < math.inf and 0 <= logit_softcapping < math.inf and 0 <= logit_scale < math.inf):
        raise ValueError(f"the temperature is finite and positive, the cap and the scale are finite and not negative; not {temperature}, "
                         f"{logit_softcapping} and {logit_scale}")
    if not _takes_transforms(temperature, logit_softcapping, logit_scale):
        raise ValueError(f"a logit scale of {logit_scale}, a cap of {logit_softcapping} and a temperature of {temperature} leave the range "
                         "of fp32")
    factor = (logit_scale or 1.0) / temperature
    return lp_ops.token_log_probs(logits, labels, factor, float(logit_softcapping), ignore_index, return_entropy)


@reference_kwargs(input_ids="index")
def selective_log_softmax(logits: torch.Tensor, index: torch.Tensor, temperature: float = 1.0,
                          logit_softcapping: float = 0.0, logit_scale: float = 0.0) -> torch.Tensor:
    """log_softmax(logits)[..., index] without keeping the full log-softmax.  Optional transforms of the logits, in
    this order: soft-cap c tanh(z / c), scale, divide by the temperature.  The transforms happen in the type of the logits;
    `token_log_probs` makes them in fp32 whatever that is, and is what computes this on the GPU where the two agree.  There an index
    outside the vocabulary gives NaN for its row; elsewhere it is an error."""
    how = (temperature, logit_softcapping or 0.0, logit_scale or 0.0)
    if (_numbers(*how) and (logits.dtype == torch.float32 or how == (1.0, 0.0, 0.0)) and index.dtype == torch.int64
            and index.shape == logits.shape[:-1] and _takes_transforms(*how) and lp_ops.native(logits, index)):
        return token_log_probs(logits, index, temperature=how[0], logit_softcapping=how[1], logit_scale=how[2], ignore_index=None)
    if logit_softcapping:
        logits = logit_softcapping * torch.tanh(logits / logit_softcapping)
    if logit_scale:
        logits = logits * logit_scale
    if temperature != 1.0:
        logits = logits / temperature
    sel = logits.gather(-1, index.unsqueeze(-1)).squeeze(-1).float()
    return sel - torch.logsumexp(logits.float(), dim=-1)


@reference_kwargs(hidden_states="hidden", input_ids="labels")
def chunked_log_softmax(hidden: torch.Tensor, lm_head: torch.Tensor, labels: torch.Tensor, chunk_tokens: int = 4096,
                        ignore_index: int = -100, *, num_chunks: int | None = None, temperature: float = 1.0,
                        logit_softcapping: float = 0.0, logit_scale: float = 0.0) -> torch.Tensor:
    """Per-token log p(label) from hidden states, chunked over tokens: only [B, L] values are kept.  `num_chunks`
    (the reference's knob) sets the chunk size to tokens / num_chunks.  Temperature and logit scale act on the hidden
    states (the head is linear); soft-capping is not linear and takes the chunked PyTorch path."""
    tokens = labels.numel()
    if num_chunks:
        chunk_tokens = max(1, -(-tokens // int(num_chunks)))
    if logit_softcapping:
        h2, y = hidden.reshape(-1, hidden.shape[-1]), labels.reshape(-1)
        out = []
        for a in range(0, tokens, chunk_tokens):
            z = h2[a:a + chunk_tokens].float() @ lm_head.float().t()
            out.append(selective_log_softmax(z, y[a:a + chunk_tokens].clamp(min=0), temperature, logit_softcapping,
                                             logit_scale) * (y[a:a + chunk_tokens] != ignore_index))
        return torch.cat(out).view(labels.shape)
    factor = (logit_scale or 1.0) / temperature
    if factor != 1.0:
        hidden = hidden * factor
    return ce_ops.fused_linear_token_logprobs(hidden, lm_head, labels, ignore_index, chunk_tokens)


def compute_advantages(rewards: torch.Tensor, group_size: int | str | None = None, eps: float = 1e-4, scale: bool = True,
                       *, baseline: str | None = None) -> torch.Tensor:
    """Group-normalised advantages: rewards [N] with consecutive groups of `group_size` samples per prompt.

    The reference's form `compute_advantages(rewards [B, G], baseline="mean" | "max" | "min" | "none", eps)` subtracts the
    per-row baseline and divides by the standard deviation of ALL advantages (data_pipeline/trainer/rl_training.py:241);
    it is selected by `baseline=` or by a string in the second position, and returns the [B, G] shape."""
    if isinstance(group_size, str) or baseline is not None or group_size is None:
        kind = baseline if baseline is not None else (group_size or "mean")
        r = rewards.float()
        base = {"mean": lambda: r.mean(-1, keepdim=True), "max": lambda: r.max(-1, keepdim=True).values,
                "min": lambda: r.min(-1, keepdim=True).values}.get(kind, lambda: 0.0)()
        a = r - base
        std = a.std() if a.numel() > 1 else a.new_zeros(())
        return a / std if float(std) > eps else a
    r = rewards.float().view(-1, group_size)
    a = r - r.mean(1, keepdim=True)
    if scale:
        a = a / (r.std(1, keepdim=True) + eps)
    return a.reshape(-1)


def _masked_mean(x, mask, dim=None):
    return (x * mask).sum(dim) / mask.sum(dim).clamp(min=1)


def _seq_mean(x, mask):
    return (x * mask).sum(-1) / mask.sum(-1).clamp(min=1)


def _reference_rl_loss(kind: str, policy_log_probs, ref_log_probs, third, mask, beta=0.04, epsilon=0.1, temperature=1.0):
    """The reference's sequence-level formulations (data_pipeline/trainer/rl_training.py:297-430), returning
    (loss, metrics).  grpo: -E[A * mean log pi] + beta * KL-per-token; drgrpo: PPO-style clipping of the sequence-level
    ratio pi / pi_ref; dapo: policy gradient weighted by softmax(rewards / temperature) over each group."""
    lp, lr = _seq_mean(policy_log_probs, mask), _seq_mean(ref_log_probs, mask)
    log_ratio = policy_log_probs - ref_log_probs
    metrics = {}
    if kind == "grpo":
        pg = -(third * lp).mean()
        kl_tok = log_ratio * mask
        kl = beta * kl_tok.sum(-1).mean() / mask.sum(-1).clamp(min=1).mean()
        metrics["kl_div"] = float((kl_tok.mean()).detach())
    elif kind == "drgrpo":
        ratio = torch.exp(_seq_mean(log_ratio, mask))
        adv = third.reshape(-1)
        pg = -torch.minimum(ratio.reshape(-1) * adv, ratio.clamp(1 - epsilon, 1 + epsilon).reshape(-1) * adv).mean()
        kl_seq = _seq_mean(log_ratio, mask)
        kl = beta * kl_seq.mean()
        metrics.update(kl_div=float((kl_seq.mean()).detach()), ratio_mean=float((ratio.mean()).detach()))
    else:
        soft = torch.softmax(third.float() / temperature, dim=-1)
        pg = -(soft * lp).sum(-1).mean()
        kl = beta * _seq_mean(log_ratio, mask).mean()
        metrics["soft_advantages_entropy"] = float(-(soft * soft.clamp_min(1e-30).log()).sum(-1).mean().detach())
    loss = pg + kl
    metrics.update(pg_loss=float((pg).detach()), kl_loss=float((kl).detach()), total_loss=float((loss).detach()))
    return loss, metrics


def clipped_policy_loss(logp: torch.Tensor, old_logp: torch.Tensor, advantages: torch.Tensor, mask: torch.Tensor,
                        ref_logp: torch.Tensor | None = None, *, clip: float = 0.2, clip_high: float | None = None, beta: float = 0.0,
                        reduction: str = "sequence", max_len: int | None = None, return_stats: bool = False):
    """Clipped policy loss with a KL term over token log-probabilities [B, T]:

        r = e^(logp - old_logp);  token = -min(r A, clamp(r, 1 - clip, 1 + clip_high) A) + beta (e^d - 1 - d),  d = ref_logp - logp

    `advantages`: [B], or [B, T].  `mask` [B, T]: tokens count with its value; where it is zero nothing is read into the loss, not even
    inf or NaN.  `reduction`: "sequence" (mean over the rows of the mean over their tokens), "token" (mean over all tokens) or
    "constant" (sum over B * max_len; max_len is T by default); a mask that leaves nothing counts as one token.
    `old_logp`, `advantages` and `ref_logp` are constants.  `return_stats`: (loss, `PolicyStats`), on the device.
    On the GPU the loss and the gradient of fp32, bf16 or fp16 log-probabilities leave one kernel together, behind one that counts the
    mask where there are more than 8192 tokens; four tokens of a thread are summed in fp32, those sums in fp64."""
    shape = logp.shape
    if len(shape) != 2:
        raise ValueError(f"log-probabilities are [sequences, tokens], not {tuple(shape)}")
    if old_logp.shape != shape or mask.shape != shape or (ref_logp is not None and ref_logp.shape != shape):
        raise ValueError(f"old_logp {tuple(old_logp.shape)}, mask {tuple(mask.shape)} and ref_logp "
                         f"{None if ref_logp is None else tuple(ref_logp.shape)} have the shape of the log-probabilities, {tuple(shape)}")
    if advantages.shape != shape[:1] and advantages.shape != shape:
        raise ValueError(f"advantages of shape {tuple(advantages.shape)} for log-probabilities of shape {tuple(shape)}")
    if reduction not in policy_ops.REDUCTIONS:
        raise ValueError(f"unknown reduction {reduction!r}; one of {sorted(policy_ops.REDUCTIONS)}")
    high = clip if clip_high is None else clip_high
    if not (0 <= clip < math.inf and 0 <= high < math.inf):
        raise ValueError(f"clip ranges are finite and not negative, not {clip} and {high}")
    if not math.isfinite(beta):
        raise ValueError(f"beta is {beta}")
    if beta and ref_logp is None:
        raise ValueError("a KL term needs ref_logp")
    if max_len is not None and max_len <= 0:
        raise ValueError(f"max_len is {max_len}")
    loss, stats = policy_ops.policy_loss(logp, old_logp, advantages, mask, ref_logp, clip, high, beta, reduction, max_len, return_stats)
    return (loss, PolicyStats(*stats.unbind())) if return_stats else loss


def _numbers(*values) -> bool:
    """Plain numbers: a tensor of one may want a gradient, or be filled in by a captured graph."""
    return all(isinstance(v, (int, float)) for v in values)


def _takes_policy_kernel(logp, old_logp, ref_logp, advantages, mask, *numbers) -> bool:
    """Whether `clipped_policy_loss` stands for the PyTorch form of a group-relative loss: fp32 on the GPU, a gradient for the
    policy's log-probabilities alone, clip ranges and a weight of the KL term (`numbers`) that are finite and not negative."""
    others = [t for t in (old_logp, ref_logp, advantages, mask) if t is not None]
    return (_numbers(*numbers) and all(0 <= v < math.inf for v in numbers)
            and all(torch.is_tensor(t) for t in (logp, *others)) and policy_ops.native(logp, *others)
            and all(t.dtype == torch.float32 for t in (logp, old_logp, advantages) if t is not None) and mask.dtype != torch.float64
            and (ref_logp is None or ref_logp.dtype == torch.float32) and advantages.shape == logp.shape[:1]
            and old_logp.shape == mask.shape == logp.shape and (ref_logp is None or ref_logp.shape == logp.shape)
            and not (torch.is_grad_enabled() and any(t.requires_grad for t in others)))


def preference_loss(policy_logps: torch.Tensor, ref_logps: torch.Tensor | None, mask: torch.Tensor, *, beta: float = 0.1,
                    loss_type: str = "sigmoid", label_smoothing: float = 0.0, gamma: float = 0.0, length_normalized: bool = False,
                    nll_weight: float = 0.0):
    """Loss of preference pairs straight from token log-probabilities [2 P, T], the chosen sequences first: returns
    (loss, rewards of the chosen [P], rewards of the rejected [P]).

    A sequence's score is the sum of mask * (policy - reference), divided by its tokens with `length_normalized`; the rewards are beta
    times the scores, and the loss is the mean over the pairs of a function of x, the difference of the two scores:
    "sigmoid" -log sigma(beta x - gamma) with `label_smoothing`, "robust" (its unbiased form under flipped labels), "hinge"
    max(0, 1 - beta x + gamma) or "ipo" (x - 1 / (2 beta))^2; "hinge" and "ipo" have no smoothed form and are the same whatever
    `label_smoothing` says.  `nll_weight` adds the chosen sequences' mean negative log-likelihood.
    Without `ref_logps` the loss is reference-free; reference log-probabilities are constants.  Tokens of mask zero are not read into
    the loss, not even inf or NaN.  Scores and what follows from them are fp64."""
    if policy_logps.dim() != 2 or policy_logps.shape[0] % 2:
        raise ValueError(f"log-probabilities are [2 * pairs, tokens], not {tuple(policy_logps.shape)}")
    for name, t in (("ref_logps", ref_logps), ("mask", mask)):
        if t is not None and t.shape != policy_logps.shape:
            raise ValueError(f"{name} of shape {tuple(t.shape)} for log-probabilities of shape {tuple(policy_logps.shape)}")
    if loss_type not in policy_ops.KINDS:
        raise ValueError(f"unknown preference loss {loss_type!r}; one of {sorted(policy_ops.KINDS)}")
    if not (math.isfinite(beta) and beta > 0 and math.isfinite(gamma) and math.isfinite(nll_weight)):
        raise ValueError(f"beta is finite and positive, gamma and nll_weight are finite, not {beta}, {gamma} and {nll_weight}")
    if not 0 <= label_smoothing <= 1 or (loss_type == "robust" and label_smoothing >= 0.5):
        raise ValueError(f"label_smoothing is {label_smoothing}: it lies in [0, 1], below 0.5 for the robust loss")
    if gamma and loss_type == "ipo":
        raise ValueError("ipo has no margin gamma")
    P = policy_logps.shape[0] // 2
    loss, rewards = policy_ops.preference_loss(policy_logps, ref_logps, mask, float(beta), loss_type, float(label_smoothing), float(gamma),
                                               bool(length_normalized), float(nll_weight))
    return (loss, *rewards.view(2, P).unbind())


def grpo_loss(logp: torch.Tensor = None, old_logp: torch.Tensor = None, ref_logp: torch.Tensor | None = None,
              advantages: torch.Tensor = None, mask: torch.Tensor = None, clip: float = 0.2, beta: float = 0.01, *,
              policy_log_probs=None, ref_log_probs=None):
    """Clipped surrogate per token, averaged per sequence then over the batch, plus the k3 KL estimator.
    Called with the reference's keywords (`policy_log_probs=, ref_log_probs=, advantages=, mask=, beta=`) it computes
    the reference's sequence-level loss instead and returns (loss, metrics): see `_reference_rl_loss`."""
    if policy_log_probs is not None:
        return _reference_rl_loss("grpo", policy_log_probs, ref_log_probs, advantages, mask, beta)
    if _takes_policy_kernel(logp, old_logp, ref_logp, advantages, mask, clip, beta):
        beta = beta if ref_logp is not None else 0.0
        return clipped_policy_loss(logp, old_logp, advantages, mask, ref_logp if beta else None, clip=clip, beta=beta)
    ratio = torch.exp(logp - old_logp)
    a = advantages.unsqueeze(-1)
    obj = torch.minimum(ratio * a, ratio.clamp(1 - clip, 1 + clip) * a)
    per_tok = -obj
    if ref_logp is not None and beta > 0:
        d = ref_logp - logp
        per_tok = per_tok + beta * (torch.exp(d) - d - 1)
    return _masked_mean(per_tok, mask, dim=-1).mean()


def drgrpo_loss(logp=None, old_logp=None, advantages=None, mask=None, clip: float = 0.2, max_len: int | None = None, *,
                policy_log_probs=None, ref_log_probs=None, beta: float = 0.04, epsilon: float = 0.1):
    """Dr. GRPO: no std scaling in the advantage and a constant length normaliser (removes the length bias).
    With the reference's keywords (`policy_log_probs=, ref_log_probs=, ..., beta=, epsilon=`): its formulation,
    returning (loss, metrics)."""
    if policy_log_probs is not None:
        return _reference_rl_loss("drgrpo", policy_log_probs, ref_log_probs, advantages, mask, beta, epsilon)
    if _takes_policy_kernel(logp, old_logp, None, advantages, mask, clip) and (max_len is None or _numbers(max_len) and max_len > 0):
        return clipped_policy_loss(logp, old_logp, advantages, mask, clip=clip, reduction="constant", max_len=max_len)
    ratio = torch.exp(logp - old_logp)
    a = advantages.unsqueeze(-1)
    obj = torch.minimum(ratio * a, ratio.clamp(1 - clip, 1 + clip) * a)
    L = max_len or mask.shape[-1]
    return -((obj * mask).sum(-1) / L).mean()


def dapo_loss(logp=None, old_logp=None, advantages=None, mask=None, clip_low: float = 0.2, clip_high: float = 0.28, *,
              policy_log_probs=None, ref_log_probs=None, rewards=None, beta: float = 0.04, temperature: float = 1.0):
    """DAPO: decoupled clip range and token-level normalisation over the whole batch.  With the reference's keywords
    (`policy_log_probs=, ref_log_probs=, rewards=, mask=, beta=, temperature=`): its soft-advantage formulation,
    returning (loss, metrics)."""
    if policy_log_probs is not None:
        return _reference_rl_loss("dapo", policy_log_probs, ref_log_probs, rewards, mask, beta, temperature=temperature)
    if _takes_policy_kernel(logp, old_logp, None, advantages, mask, clip_low, clip_high):
        return clipped_policy_loss(logp, old_logp, advantages, mask, clip=clip_low, clip_high=clip_high, reduction="token")
    ratio = torch.exp(logp - old_logp)
    a = advantages.unsqueeze(-1)
    obj = torch.minimum(ratio * a, ratio.clamp(1 - clip_low, 1 + clip_high) * a)
    return -(obj * mask).sum() / mask.sum().clamp(min=1)


@reference_kwargs(input_ids="ids")
def left_pack_padding(ids: torch.Tensor, mask: torch.Tensor | int | None = None, pad_id: int = 0, *,
                      pad_token_id: int | None = None):
    """Move real tokens to the left of every row (stable), padding to the right: returns (ids, mask).

    The reference's function of this name, `left_pack_padding(input_ids, pad_token_id)`, goes the other way: it moves
    the PADDING to the left (real tokens end flush right, as its attention path wants) and returns the ids alone
    (data_pipeline/trainer/rl_training.py:434).  That form is selected by an integer second argument or `pad_token_id=`."""
    if pad_token_id is not None or isinstance(mask, int):
        pad = pad_token_id if pad_token_id is not None else mask
        real = ids != pad
        order = torch.argsort(real.int(), dim=1, stable=True)          # padding first, tokens keep their order
        return ids.gather(1, order)
    order = torch.argsort((mask == 0).int(), dim=1, stable=True)
    return ids.gather(1, order).masked_fill(mask.gather(1, order) == 0, pad_id), mask.gather(1, order)


class GRPOCompute:
    def __init__(self, group_size: int = 8, clip: float = 0.2, beta: float = 0.01, variant: str = "grpo",
                 model: nn.Module | None = None, reward_clip: float | None = None, chunk_tokens: int = 4096, *,
                 ref_model: nn.Module | None = None, config=None):
        """`GRPOCompute(model, ref_model, config)` is the reference's form: `config` (an RL configuration object)
        supplies num_generations (group size), clip_range, kl_coef (beta), algorithm (variant) and reward_clip."""
        if isinstance(group_size, nn.Module):                 # positional (model, ref_model, config)
            model, group_size = group_size, 8
            if isinstance(clip, nn.Module) or clip is None:
                ref_model, clip = clip, 0.2
            if not isinstance(beta, (int, float)):
                config, beta = beta, 0.01
        if config is not None:
            group_size = int(getattr(config, "num_generations", group_size))
            clip = float(getattr(config, "clip_range", clip))
            beta = float(getattr(config, "kl_coef", beta))
            variant = str(getattr(getattr(config, "algorithm", variant), "value", getattr(config, "algorithm", variant))).lower()
            reward_clip = getattr(config, "reward_clip", reward_clip)
        self.group_size, self.clip, self.beta, self.variant = group_size, clip, beta, variant
        self.model, self.ref_model, self.reward_clip, self.chunk_tokens = model, ref_model, reward_clip, chunk_tokens

    def compute_log_probs(self, input_ids: torch.Tensor, attention_mask: torch.Tensor | None = None,
                          model: nn.Module | None = None) -> torch.Tensor:
        """log p(token t+1 | tokens <= t) for every position, [B, S-1] (0 where the target is padding), without ever
        forming [B, S, V] logits: the decoder's hidden states go through the chunked fused head
        (data_pipeline/trainer/rl_training.py:509-552)."""
        model = model if model is not None else self.model
        if model is None:
            raise ValueError("compute_log_probs needs a model (argument or constructor)")
        out = model(input_ids=input_ids, return_logits=False)
        labels = input_ids[:, 1:]
        if attention_mask is not None:
            labels = labels.masked_fill(attention_mask[:, 1:] == 0, -100)
        return chunked_log_softmax(out.hidden_states[:, :-1], model.head_weight, labels, self.chunk_tokens)

    def compute_grpo_loss(self, policy_log_probs, ref_log_probs, rewards, mask, old_log_probs=None):
        """(loss, {"reward_mean", "reward_std", "advantage_abs_mean", "kl"}) for the configured variant.  Without
        `old_log_probs` the policy's own (detached) values are the behaviour policy: one optimisation step per batch."""
        if self.reward_clip:
            rewards = rewards.clamp(-self.reward_clip, self.reward_clip)
        old = policy_log_probs.detach() if old_log_probs is None else old_log_probs
        adv = compute_advantages(rewards, self.group_size, scale=self.variant != "drgrpo")
        kl = None
        if (_takes_policy_kernel(policy_log_probs, old, ref_log_probs, adv, mask, self.clip, self.beta)
                and type(self).__call__ is GRPOCompute.__call__):
            kw = {"drgrpo": dict(reduction="constant"), "dapo": dict(reduction="token", clip_high=0.28)}.get(
                self.variant, dict(beta=self.beta if ref_log_probs is not None else 0.0))
            loss, seen = clipped_policy_loss(policy_log_probs, old, adv, mask, ref_log_probs, clip=self.clip, return_stats=True, **kw)
            kl = seen.kl                              # (out of the pass that made the loss)
        else:
            loss = self(policy_log_probs, old, ref_log_probs, rewards, mask)
        stats = {"reward_mean": float(rewards.float().mean()), "reward_std": float(rewards.float().std()),
                 "advantage_abs_mean": float(adv.abs().mean())}
        if ref_log_probs is not None:
            d = (ref_log_probs - policy_log_probs).detach() if kl is None else None
            stats["kl"] = float(_masked_mean(torch.exp(d) - d - 1, mask) if kl is None else kl)
        return loss, stats

    def __call__(self, logp, old_logp, ref_logp, rewards, mask):
        adv = compute_advantages(rewards, self.group_size, scale=self.variant != "drgrpo")
        if self.variant == "drgrpo":
            return drgrpo_loss(logp, old_logp, adv, mask, self.clip)
        if self.variant == "dapo":
            return dapo_loss(logp, old_logp, adv, mask, self.clip)
        return grpo_loss(logp, old_logp, ref_logp, adv, mask, self.clip, self.beta)


class RewardModel(nn.Module):
    """Decoder backbone + scalar head read at the last real token."""

    def __init__(self, backbone=None, *, model=None, reward_fn=None):
        """`RewardModel(backbone)`: a framework decoder gets a scalar value head.  `model=` / `reward_fn=` are the
        reference's form (data_pipeline/trainer/rl_training.py:607): any classifier whose last-position logit is the
        score, or a function (input_ids, attention_mask, **kw) -> [B]; with neither, rewards are zero."""
        super().__init__()
        self.reward_fn, self.scorer = reward_fn, None
        backbone = backbone if backbone is not None else model
        self.backbone = backbone
        if backbone is not None and hasattr(getattr(backbone, "config", None), "hidden_size") and hasattr(backbone, "model"):
            h = backbone.config.hidden_size
            p = next(backbone.parameters())
            self.value_head = nn.Linear(h, 1, bias=False, dtype=p.dtype, device=p.device)
        else:
            self.scorer, self.backbone = backbone, None

    def forward(self, input_ids, attention_mask=None, **kwargs):
        if self.backbone is None:
            if self.scorer is not None:
                out = self.scorer(input_ids=input_ids, attention_mask=attention_mask)
                logits = out.logits if hasattr(out, "logits") else out
                return logits[:, -1].reshape(logits.shape[0], -1)[:, 0].float() if logits.dim() > 1 else logits.float()
            if self.reward_fn is not None:
                return self.reward_fn(input_ids, attention_mask, **kwargs)
            return torch.zeros(input_ids.shape[0], device=input_ids.device)
        h = self.backbone.model(input_ids)
        if attention_mask is None:
            last = torch.full((h.shape[0],), h.shape[1] - 1, device=h.device)
        else:
            last = attention_mask.long().sum(1).clamp(min=1) - 1
        return self.value_head(h[torch.arange(h.shape[0], device=h.device), last]).squeeze(-1).float()


class PreferenceTrainer:
    """Preference optimisation on batches with chosen_/rejected_ input_ids, attention_mask and labels."""

    def __init__(self, policy, engine=None, ref_model=None, loss: str = "dpo", beta: float = 0.1, **loss_kw):
        self.policy, self.engine, self.kind = policy, engine, loss
        self.ref = ref_model
        if self.ref is not None:
            self.ref.eval()
            for p in self.ref.parameters():
                p.requires_grad_(False)
        self.loss_fn = {"dpo": lambda: DPOLoss(beta, **loss_kw), "simpo": lambda: SimPOLoss(beta, **loss_kw),
                        "orpo": lambda: ORPOLoss(**loss_kw), "kto": lambda: KTOLoss(beta, **loss_kw),
                        "cpo": lambda: CPOLoss(beta, **loss_kw)}[loss]()

    @staticmethod
    def make_reference(policy):
        """Frozen copy of the policy taken before the engine re-points its parameters at flat buffers."""
        ref = copy.deepcopy(policy)
        for p in ref.parameters():
            p.requires_grad_(False)
        return ref.eval()

    def _token_logps(self, model, ids, mask, labels, grad: bool):
        """Log-probabilities of the next tokens, and where there is one."""
        ctx = torch.enable_grad() if grad else torch.no_grad()
        with ctx:
            h = model.model(ids)
            w = model.head_weight
            lab = labels.masked_fill(mask == 0, -100)
            tgt = torch.full_like(lab, -100)
            tgt[:, :-1] = lab[:, 1:]
            return ce_ops.fused_linear_token_logprobs(h, w if grad else w.detach(), tgt), tgt != -100

    def _seq_logps(self, model, ids, mask, labels, grad: bool):
        lp, valid = self._token_logps(model, ids, mask, labels, grad)
        return lp.sum(-1), valid.sum(-1)

    def _sums_plainly(self) -> bool:
        return type(self)._seq_logps is PreferenceTrainer._seq_logps and "_seq_logps" not in self.__dict__

    def _pair_kernel(self) -> dict | None:
        """The loss as arguments of `preference_loss`; None for those that are not a function of one pair's scores, and for a loss module
        that is not just what the constructor makes: a subclass, another module, one with hooks, a replaced forward or a learned beta."""
        f, kind = self.loss_fn, self.kind
        if type(f) is not {"dpo": DPOLoss, "simpo": SimPOLoss, "cpo": CPOLoss}.get(kind) or (
                "forward" in f.__dict__ or f._forward_hooks or f._forward_pre_hooks or f._backward_hooks or f._backward_pre_hooks
                or _has_any_global_hook()):
            return None
        if kind == "dpo" and f.loss_type in policy_ops.KINDS and (f.loss_type != "robust" or f.label_smoothing < 0.5):
            kw = dict(loss_type=f.loss_type, label_smoothing=f.label_smoothing if f.loss_type in ("sigmoid", "robust") else 0.0)
        elif kind == "simpo":
            kw = dict(label_smoothing=f.eps, gamma=f.gamma, length_normalized=True)
        elif kind == "cpo":
            kw = dict(label_smoothing=f.eps, nll_weight=f.alpha)
        else:
            return None
        kw["beta"] = f.beta
        numbers = [v for k, v in kw.items() if k not in ("loss_type", "length_normalized")]
        if not all(isinstance(v, (int, float)) and math.isfinite(v) for v in numbers):
            return None
        return kw if f.beta > 0 and 0 <= kw["label_smoothing"] <= 1 else None

    def compute_loss(self, batch: Dict[str, torch.Tensor]):
        B = batch["chosen_input_ids"].shape[0]
        ids = torch.cat((batch["chosen_input_ids"], batch["rejected_input_ids"]))
        mask = torch.cat((batch["chosen_attention_mask"], batch["rejected_attention_mask"]))
        labels = torch.cat((batch["chosen_labels"], batch["rejected_labels"]))
        metrics = {}
        # (a trainer that sums in its own way has no token log-probabilities to give)
        kernel = self._pair_kernel() if self._sums_plainly() else None
        if kernel is not None:
            tokens, valid = self._token_logps(self.policy, ids, mask, labels, True)
            if not policy_ops.native(tokens, valid):
                kernel, lp, n = None, tokens.sum(-1), valid.sum(-1)
        else:
            lp, n = self._seq_logps(self.policy, ids, mask, labels, True)
        if kernel is not None:
            ref = None
            if self.kind == "dpo" and self.ref is not None and not self.loss_fn.reference_free:
                ref, _ = self._token_logps(self.ref, ids, mask, labels, False)
            loss, cr, rjr = preference_loss(tokens, ref, valid, **kernel)
            if self.kind != "cpo":
                metrics["reward_accuracy"] = (cr > rjr).float().mean()
            if self.kind == "dpo":
                metrics["reward_margin"] = (cr - rjr).mean()
            return loss, metrics
        pc, pr, nc, nr = lp[:B], lp[B:], n[:B], n[B:]
        if self.kind == "dpo":
            rc = rr = None
            if self.ref is not None and not self.loss_fn.reference_free:
                rl, _ = self._seq_logps(self.ref, ids, mask, labels, False)
                rc, rr = rl[:B], rl[B:]
            loss, cr, rjr = self.loss_fn(pc, pr, rc, rr)
            metrics = {"reward_accuracy": (cr > rjr).float().mean(), "reward_margin": (cr - rjr).mean()}
        elif self.kind == "simpo":
            loss, cr, rjr = self.loss_fn(pc, pr, nc.float(), nr.float())
            metrics = {"reward_accuracy": (cr > rjr).float().mean()}
        elif self.kind == "orpo":
            nll = -(pc / nc.clamp(min=1)).mean()
            loss, ratio = self.loss_fn(pc / nc.clamp(min=1), pr / nr.clamp(min=1), nll)
            metrics = {"log_odds_ratio": ratio.mean()}
        elif self.kind == "cpo":
            loss = self.loss_fn(pc, pr, -(pc / nc.clamp(min=1)).mean())
        else:   # kto on paired data: chosen = desirable, rejected = undesirable
            rl = torch.zeros_like(lp)
            if self.ref is not None:
                rl, _ = self._seq_logps(self.ref, ids, mask, labels, False)
            tag = torch.cat((torch.ones(B), torch.zeros(B))).to(lp.device)
            loss, _ = self.loss_fn(lp, rl, tag)
        return loss, metrics

    def train_step(self, batch: Dict[str, torch.Tensor], lr: float | None = None):
        loss, metrics = self.compute_loss(batch)
        if self.engine is not None:
            self.engine.micro_step = max(1, self.engine.cfg.gradient_accumulation_steps) - 1
            self.engine.backward(loss)
            gn = self.engine.step(lr)
        else:
            loss.backward()
            gn = None
        return loss.detach(), metrics, gn


# ------------------------------------------------------------------------------------------------ reward / batch helpers
def clip_rewards(rewards: torch.Tensor, clip_value: float | None = 10.0) -> torch.Tensor:
    """Clamp rewards to [-clip_value, clip_value] (data_pipeline/trainer/rl_training.py:272)."""
    return rewards if clip_value is None else rewards.clamp(-clip_value, clip_value)


def apply_length_penalty(rewards: torch.Tensor, lengths: torch.Tensor, alpha: float = 1.0) -> torch.Tensor:
    """rewards * (length / longest length)^alpha: short completions earn less (rl_training.py:282)."""
    return rewards * (lengths.float() / lengths.max().clamp(min=1).float()) ** alpha


def calculate_pad_tokens_in_prompt(input_ids: torch.Tensor, logits_to_keep: int, pad_token_id: int) -> torch.Tensor:
    """Pad tokens in the prompt part (everything but the last `logits_to_keep` positions) of every row."""
    return (input_ids[:, :-logits_to_keep] == pad_token_id).sum(-1)


def create_completion_attention_mask(input_ids: torch.Tensor, pad_token_id: int) -> torch.Tensor:
    return (input_ids != pad_token_id).long()


def autotune_batch_and_chunks(total_rows: int, seq_len: int, hidden_dim: int, vocab_dim: int, dtype_bytes: int = 16,
                              multiplier: int | None = None, budget_bytes: int | None = None) -> tuple[int, int]:
    """(rows per pass, number of vocabulary chunks) for a chunked log-softmax over `total_rows` sequences
    (rl_training.py:198-238).  A pass holds rows x seq_len hidden states and one chunk of the logits, rows x seq_len x
    vocab / chunks in fp32; rows is the largest divisor of `total_rows` that fits the budget (default 4 GiB; on a
    180 GB part pass `budget_bytes`), chunks defaults to max(4, seq_len / 4096).  `dtype_bytes` is in BITS, as in the
    reference."""
    chunks = multiplier if multiplier is not None else max(4, seq_len // 4096)
    budget = budget_bytes if budget_bytes is not None else 4 * 2 ** 30
    per_row = seq_len * hidden_dim * dtype_bytes / 8 + seq_len * vocab_dim * 4 / chunks
    rows = int(max(1, min(total_rows, budget // max(per_row, 1))))
    while total_rows % rows:
        rows -= 1
    return rows, chunks


# ---- the three group-relative losses in the reference's POSITIONAL order (data_pipeline/trainer/rl_training.py:297-440):
# what `from data_pipeline.trainer.rl_training import grpo_loss` resolves to under `reference_paths`, so that
# `grpo_loss(policy_log_probs, ref_log_probs, advantages, mask, beta)` called by position means what it means there
def _reference_grpo_loss(policy_log_probs, ref_log_probs, advantages, mask, beta: float = 0.04):
    return grpo_loss(policy_log_probs=policy_log_probs, ref_log_probs=ref_log_probs, advantages=advantages, mask=mask,
                     beta=beta)


def _reference_drgrpo_loss(policy_log_probs, ref_log_probs, advantages, mask, beta: float = 0.04, epsilon: float = 0.1):
    return drgrpo_loss(policy_log_probs=policy_log_probs, ref_log_probs=ref_log_probs, advantages=advantages, mask=mask,
                       beta=beta, epsilon=epsilon)


def _reference_dapo_loss(policy_log_probs, ref_log_probs, rewards, mask, beta: float = 0.04, temperature: float = 1.0):
    return dapo_loss(policy_log_probs=policy_log_probs, ref_log_probs=ref_log_probs, rewards=rewards, mask=mask, beta=beta,
                     temperature=temperature)


grpo_loss.__reference_form__ = _reference_grpo_loss
drgrpo_loss.__reference_form__ = _reference_drgrpo_loss
dapo_loss.__reference_form__ = _reference_dapo_loss
