"""The operators of a post-training step that are timed, each through the entry point a user's program calls:

* ``logp``        `rl.token_log_probs`: log-probabilities of the chosen tokens, and the entropies, out of a model's logits;
* ``policy``      `rl.clipped_policy_loss`: the clipped policy loss with its KL term over token log-probabilities;
* ``preference``  `rl.preference_loss`: losses of (chosen, rejected) pairs out of token log-probabilities;
* ``clip``        `optim.clip_grad_norm_`: the global norm of a list of gradients, and their clipping.

The plain forms below compute the same with elementary tensor operations in 32 bits (where a value next to a border or a
long sum decides, in 64).
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEVICE = "cuda"
IGNORE = -100
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4, "bool": 1, "int64": 8, "float": 4}
# decoders whose gradients are clipped: hidden size, intermediate size, layers, vocabulary, width of the packed q/k/v
# projection, width of the output projection's input (presets of models/llama.py)
MODELS = {"tiny": (256, 688, 4, 32000, 768, 256), "llama3-1b": (2048, 8192, 16, 128256, 5120, 2048),
          "llama3-8b": (4096, 14336, 32, 128256, 6144, 4096)}


def listed() -> list[dict]:
    return [
        # the last positions of a few prompts, scored one by one: launches and one long vocabulary are all there is
        _logp("logp_few", 9, 1, 128256, "bf16"),
        # the old policy's log-probabilities of a rollout, kept without a gradient; the prompts' targets are ignored
        _logp("logp_rollout", 6, 700, 32000, "bf16", prompt=211),
        # a policy step on a Llama-3 vocabulary: sampling temperature, entropy bonus, logits of all but the last position
        _logp("logp_train", 4, 511, 128256, "bf16", prompt=100, temperature=0.7, entropy=True, grad=True, sliced=True),
        # capped logits of an odd vocabulary in fp32
        _logp("logp_capped", 3, 701, 32001, "fp32", cap=30.0, grad=True),
        # one prompt, eight sampled answers of a few tokens
        _policy("policy_group", 8, 61, "fp32", "bool", "sequence", beta=0.04),
        # an ordinary rollout batch normalised over its tokens, two clip bounds, no reference model
        _policy("policy_batch", 256, 1023, "fp32", "int64", "token", high=0.28),
        # long reasoning traces with a KL term
        _policy("policy_long", 512, 16384, "fp32", "float", "sequence", beta=0.01),
        # the batch of configs/llama3_8b_dpo.yaml: 8 pairs of at most 2048 tokens
        _pref("pref_dpo", 8, 2047, "fp32", "bool", "sigmoid"),
        # length-normalised, reference-free pairs of an odd length, 16-bit log-probabilities
        _pref("pref_simpo", 96, 1777, "bf16", "bool", "sigmoid", beta=2.0, gamma=0.5, normalized=True, ref=False),
        # long answers, squared loss
        _pref("pref_long", 160, 16384, "fp32", "float", "ipo"),
        # adapters of rank 8 on every projection of a small decoder: many little tensors
        _clip("clip_adapters", "llama3-1b", 16, "fp32", rank=8),
        # all gradients of a decoder a quarter as deep as llama3-1b
        _clip("clip_full", "llama3-1b", 4, "bf16"),
    ]


def _logp(name, batch, seq, vocab, dtype, prompt=0, temperature=1.0, cap=0.0, entropy=False, grad=False, sliced=False) -> dict:
    return {"name": name, "path": "logp", "batch": batch, "seq": seq, "vocab": vocab, "dtype": dtype, "prompt": prompt,
            "temperature": temperature, "cap": cap, "entropy": entropy, "grad": grad, "sliced": sliced}


def _policy(name, batch, seq, dtype, mask, reduction, beta=0.0, low=0.2, high=0.2, per_token=False) -> dict:
    return {"name": name, "path": "policy", "batch": batch, "seq": seq, "dtype": dtype, "mask": mask, "reduction": reduction,
            "beta": beta, "low": low, "high": high, "per_token": per_token}


def _pref(name, pairs, seq, dtype, mask, kind, beta=0.1, gamma=0.0, smoothing=0.0, normalized=False, nll=0.0, ref=True) -> dict:
    return {"name": name, "path": "preference", "pairs": pairs, "seq": seq, "dtype": dtype, "mask": mask, "kind": kind,
            "beta": beta, "gamma": gamma, "smoothing": smoothing, "normalized": normalized, "nll": nll, "ref": ref}


def _clip(name, model, layers, dtype, rank=0, norm="2", active=True) -> dict:
    return {"name": name, "path": "clip", "model": model, "layers": layers, "dtype": dtype, "rank": rank, "norm": norm,
            "active": active}


def _spread(rng: random.Random, low: int, high: int) -> int:
    """An integer of [low, high], evenly over its logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng: random.Random) -> dict:
    most = {}
    for c in listed():
        most[c["path"]] = max(most.get(c["path"], 0), work(c)["bytes"])
    while True:
        case = _drawn(rng)
        del case["name"]
        if work(case)["bytes"] <= most[case["path"]]:
            return case


def _drawn(rng: random.Random) -> dict:
    path = rng.choice(("logp", "policy", "preference", "clip"))
    if path == "logp":
        vocab = rng.choice((32000, 32064, 128256, 152064, _spread(rng, 500, 160000)))
        batch, seq, grad = _spread(rng, 1, 64), _spread(rng, 1, 4096), rng.random() < 0.7
        return _logp("", batch, seq, vocab, rng.choice(("bf16", "bf16", "fp16", "fp32")), rng.choice((0, seq // 3)),
                     rng.choice((1.0, 0.6, 1.3)), rng.choice((0.0, 0.0, 30.0)), rng.random() < 0.4, grad, rng.random() < 0.4)
    if path == "policy":
        return _policy("", _spread(rng, 1, 2048), _spread(rng, 1, 32768), rng.choice(("fp32", "fp32", "bf16")),
                       rng.choice(("bool", "int64", "float")), rng.choice(("sequence", "token", "constant")),
                       rng.choice((0.0, 0.04)), 0.2, rng.choice((0.2, 0.28)), rng.random() < 0.25)
    if path == "preference":
        normalized = rng.random() < 0.4
        return _pref("", _spread(rng, 1, 512), _spread(rng, 1, 32768), rng.choice(("fp32", "fp32", "bf16")),
                     rng.choice(("bool", "int64", "float")), rng.choice(("sigmoid", "robust", "hinge", "ipo")),
                     2.0 if normalized else 0.1, 0.0, rng.choice((0.0, 0.1)), normalized, rng.choice((0.0, 0.5)),
                     rng.random() < 0.7)
    model = rng.choice(("tiny", "llama3-1b", "llama3-8b"))
    rank = rng.choice((0, 4, 8, 64)) if model != "llama3-8b" else rng.choice((4, 8, 64))
    return _clip("", model, rng.randint(1, MODELS[model][2]), rng.choice(("fp32", "bf16", "mixed")), rank,
                 rng.choice(("2", "2", "2", "inf", "1")), rng.random() < 0.75)


# ------------------------------------------------------------------------------------------------ inputs
def _generator(seed: int) -> torch.Generator:
    return torch.Generator(device=DEVICE).manual_seed(seed)


def _normal(g: torch.Generator, *shape: int, std: float = 1.0) -> torch.Tensor:
    return torch.empty(shape, device=DEVICE).normal_(0.0, std, generator=g)


def _uniform(g: torch.Generator, *shape: int) -> torch.Tensor:
    return torch.rand(shape, device=DEVICE, generator=g)


def prepare(case: dict, seed: int):
    make = {"logp": _prepare_logp, "policy": _prepare_policy, "preference": _prepare_preference, "clip": _prepare_clip}
    return {"case": case, **make[case["path"]](case, seed)}


def _prepare_logp(case: dict, seed: int):
    """Logits [batch, seq (+ 1), vocab] of a model that knows most of the next tokens, and those tokens."""
    g, B, T, V = _generator(seed), case["batch"], case["seq"], case["vocab"]
    full = torch.empty(B, T + case["sliced"], V, dtype=TYPES[case["dtype"]], device=DEVICE).normal_(0.0, 2.5, generator=g)
    labels = torch.randint(0, V, (B, T), device=DEVICE, generator=g)
    logits = full[:, :T]
    known = torch.where(_uniform(g, B, T) < 0.7, 10.0, 0.0).to(full.dtype)
    logits.scatter_add_(2, labels.unsqueeze(2), known.unsqueeze(2))
    labels[:, :case["prompt"]] = IGNORE
    return {"logits": logits, "labels": labels, "g": _normal(g, B, T, std=1e-3), "h": _normal(g, B, T, std=1e-4)}


def _mask(case: dict, g: torch.Generator, rows: int) -> torch.Tensor:
    """Answers of all lengths behind prompts of all lengths; the last of many rows has no token of its own."""
    T = case["seq"]
    at = torch.arange(T, device=DEVICE)
    first = (_uniform(g, rows, 1) * 0.3 * T).long()
    last = first + 1 + (_uniform(g, rows, 1) * (T - first)).long()
    mask = (at >= first) & (at < last)
    if rows > 8:
        mask[-1] = False
    return mask.to({"bool": torch.bool, "int64": torch.int64, "float": torch.float32}[case["mask"]])


def _logprobs(g: torch.Generator, *shape: int) -> torch.Tensor:
    return -_uniform(g, *shape).clamp(min=1e-6).log() * 0.8


def _prepare_policy(case: dict, seed: int):
    g, B, T, dtype = _generator(seed), case["batch"], case["seq"], TYPES[case["dtype"]]
    logp = -_logprobs(g, B, T)
    reward = _normal(g, B, T) if case["per_token"] else _normal(g, B)
    return {"logp": logp.to(dtype).requires_grad_(), "old": (logp + _normal(g, B, T, std=0.12)).to(dtype),
            "ref": (logp + _normal(g, B, T, std=0.3)).to(dtype) if case["beta"] else None, "advantages": reward,
            "mask": _mask(case, g, B)}


def _prepare_preference(case: dict, seed: int):
    g, R, T, dtype = _generator(seed), 2 * case["pairs"], case["seq"], TYPES[case["dtype"]]
    logp = -_logprobs(g, R, T)
    ref = logp - _normal(g, R, 1, std=2.0 / T) + _normal(g, R, T, std=0.1)
    return {"logp": logp.to(dtype).requires_grad_(), "ref": ref.to(dtype) if case["ref"] else None,
            "mask": _mask(case, g, R)}


def _shapes(case: dict) -> list[tuple[int, ...]]:
    H, I, _, V, qkv, o = MODELS[case["model"]]
    layer = [(qkv, H), (H, o), (2 * I, H), (H, I)]
    if case["rank"]:
        return [s for _ in range(case["layers"]) for n, k in layer for s in ((case["rank"], k), (n, case["rank"]))]
    return [(V, H)] + [s for _ in range(case["layers"]) for s in [(H,), layer[0], layer[1], (H,), layer[2], layer[3]]] + [(H,)]


def _types(case: dict) -> list[torch.dtype]:
    """`mixed`: matrices in bf16, vectors and every third matrix in fp32."""
    if case["dtype"] != "mixed":
        return [TYPES[case["dtype"]]] * len(_shapes(case))
    return [torch.float32 if len(s) == 1 or i % 3 == 0 else torch.bfloat16 for i, s in enumerate(_shapes(case))]


def _prepare_clip(case: dict, seed: int):
    """Gradients that are views of one buffer for each type, as data-parallel training keeps them."""
    g, shapes, types = _generator(seed), _shapes(case), _types(case)
    buffers, parameters = {}, []
    for t in dict.fromkeys(types):
        buffers[t] = torch.empty(sum(math.prod(s) for s, u in zip(shapes, types) if u == t), dtype=t, device=DEVICE)
    at = dict.fromkeys(buffers, 0)
    for shape, t in zip(shapes, types):
        p = torch.nn.Parameter(torch.empty(shape, dtype=t, device=DEVICE))
        p.grad = buffers[t][at[t]:at[t] + p.numel()].view(shape).normal_(0.0, 2e-3 / math.sqrt(shape[-1]), generator=g)
        at[t] += p.numel()
        parameters.append(p)
    norm = _norm64(list(buffers.values()), case["norm"])
    return {"parameters": parameters, "buffers": list(buffers.values()), "limit": float(norm) * (0.3 if case["active"] else 2.0)}


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    make = {"logp": _run_logp, "policy": _run_policy, "preference": _run_preference, "clip": _run_clip}
    return make[state["case"]["path"]](state, state["case"])


def _run_logp(s, case):
    if own:
        from trainscale_b200.rl import token_log_probs
        x = s["logits"].detach().requires_grad_(case["grad"])
        out = token_log_probs(x, s["labels"], temperature=case["temperature"], logit_softcapping=case["cap"],
                              ignore_index=IGNORE, return_entropy=case["entropy"])
        logp, entropy = out if case["entropy"] else (out, None)
        if not case["grad"]:
            return [logp] if entropy is None else [logp, entropy]
        if entropy is None:
            return [logp.detach(), *torch.autograd.grad(logp, x, s["g"])]
        return [logp.detach(), entropy.detach(), *torch.autograd.grad((logp, entropy), x, (s["g"], s["h"]))]
    z, slope = s["logits"].float(), 1.0
    if case["cap"]:
        t = torch.tanh(z / case["cap"])
        z, slope = case["cap"] * t, 1 - t * t
    z = z / case["temperature"]
    valid = s["labels"] != IGNORE
    at = s["labels"].clamp(min=0).unsqueeze(2)
    top = z.max(-1, keepdim=True).values
    log_p = z - (top + (z - top).exp().sum(-1, keepdim=True).log())
    logp = torch.where(valid, log_p.gather(2, at).squeeze(2), 0.0)
    p = log_p.exp()
    entropy = torch.where(valid, -(p * log_p).sum(-1), 0.0) if case["entropy"] else None
    out = [logp] if entropy is None else [logp, entropy]
    if case["grad"]:
        g = torch.where(valid, s["g"], 0.0).unsqueeze(2)
        d = -p * g
        d.scatter_add_(2, at, g)
        if case["entropy"]:
            h = torch.where(valid, s["h"], 0.0).unsqueeze(2)
            d = d - p * (log_p + entropy.unsqueeze(2)) * h
        out.append((d * slope / case["temperature"]).to(s["logits"].dtype))
    return out


def _run_policy(s, case):
    if own:
        from trainscale_b200.rl import clipped_policy_loss
        loss, stats = clipped_policy_loss(s["logp"], s["old"], s["advantages"], s["mask"], s["ref"], clip=case["low"],
                                          clip_high=case["high"], beta=case["beta"], reduction=case["reduction"],
                                          return_stats=True)
        (grad,) = torch.autograd.grad(loss, s["logp"])
        return [loss.detach(), grad, stats.kl, stats.clip_fraction, stats.ratio]
    logp, old, mask = s["logp"].detach().float(), s["old"].float(), s["mask"].float()
    a = s["advantages"] if case["per_token"] else s["advantages"].unsqueeze(1)
    ratio = (logp - old).exp()
    inside = (logp.double() - old.double()).exp()                 # which side of a clip bound: decided in 64 bits
    clipped = ((a > 0) & (inside > 1 + case["high"])) | ((a < 0) & (inside < 1 - case["low"]))
    bound = torch.where(a > 0, 1 + case["high"], 1 - case["low"])
    token = -torch.where(clipped, bound, ratio) * a
    slope = torch.where(clipped, 0.0, -ratio * a)
    kl = torch.zeros_like(token)
    if s["ref"] is not None:
        d = s["ref"].double() - logp.double()                     # e^d - 1 - d of small d: 32 bits would cancel
        kl = (d.expm1() - d).float()
        token, slope = token + case["beta"] * kl, slope - case["beta"] * d.expm1().float()
    count = mask.double().sum().clamp(min=1)
    weight = _policy_weight(case, mask)
    used = mask != 0
    total = lambda x, w: torch.where(used, x * w, 0.0).double().sum().float()      # noqa: E731
    return [total(token, weight), torch.where(used, slope * weight, 0.0).to(s["logp"].dtype), total(kl, mask / count),
            total(clipped.float(), mask / count), total(ratio, mask / count)]


def _policy_weight(case, mask):
    """What a token's loss counts for in the batch's."""
    rows, length = mask.shape
    if case["reduction"] == "sequence":
        return mask / mask.sum(1, keepdim=True).clamp(min=1) / rows
    return mask / (mask.double().sum().clamp(min=1) if case["reduction"] == "token" else rows * length)


def _run_preference(s, case):
    if own:
        from trainscale_b200.rl import preference_loss
        loss, chosen, rejected = preference_loss(s["logp"], s["ref"], s["mask"], beta=case["beta"], loss_type=case["kind"],
                                                 label_smoothing=case["smoothing"], gamma=case["gamma"],
                                                 length_normalized=case["normalized"], nll_weight=case["nll"])
        (grad,) = torch.autograd.grad(loss, s["logp"])
        return [loss.detach(), chosen, rejected, grad]
    # long sums whose difference decides: 64 bits
    return _preference(s, case)


def _preference(s, case, out=torch.float32):
    """Sums over a sequence in 64 bits; results in `out`, the gradient in the type of its input where that is 32 bits."""
    logp, P = s["logp"].detach().double(), case["pairs"]
    mask = s["mask"].double()
    delta = logp if s["ref"] is None else logp - s["ref"].double()
    count = mask.sum(1).clamp(min=1)
    score = torch.where(mask != 0, delta * mask, 0.0).sum(1)
    if case["normalized"]:
        score = score / count
    x = score[:P] - score[P:]
    b, eps = case["beta"], case["smoothing"]
    m = b * x - case["gamma"]
    up, down = torch.log1p((-m.abs()).exp()) - m.clamp(max=0), torch.log1p((-m.abs()).exp()) + m.clamp(min=0)
    right, wrong = 1 / (1 + m.exp()), 1 / (1 + (-m).exp())         # sigma(-m), sigma(m): the slopes of up and down
    if case["kind"] == "sigmoid":
        loss, slope = (1 - eps) * up + eps * down, b * (eps * wrong - (1 - eps) * right)
    elif case["kind"] == "robust":
        loss, slope = ((1 - eps) * up - eps * down) / (1 - 2 * eps), b * -((1 - eps) * right + eps * wrong) / (1 - 2 * eps)
    elif case["kind"] == "hinge":
        loss, slope = (1 - m).clamp(min=0), -b * (m < 1).double()
    else:
        loss, slope = (x - 1 / (2 * b)) ** 2, 2 * (x - 1 / (2 * b))
    row = torch.cat((slope, -slope)) / P
    if case["normalized"]:
        row = row / count
    nll = torch.where(mask != 0, logp * mask, 0.0).sum(1)[:P] / count[:P]
    loss = loss - case["nll"] * nll
    row[:P] -= case["nll"] / count[:P] / P
    grad = torch.where(mask != 0, row.unsqueeze(1) * mask, 0.0)
    return [loss.mean().to(out), (b * score[:P]).to(out), (b * score[P:]).to(out),
            grad.to(s["logp"].dtype if out == torch.float32 else out)]


def _run_clip(s, case):
    # a pass clips what the last one left to a little less, so that each has the gradients to scale
    limit, s["limit"] = s["limit"], s["limit"] * (0.999 if case["active"] else 1.0)
    kind = float(case["norm"])
    if own:
        from trainscale_b200.optim import clip_grad_norm_
        norm = clip_grad_norm_(s["parameters"], limit, kind)
        return [norm.float(), *s["buffers"]]        # (the largest value of gradients of one type comes in that type)
    grads = [p.grad for p in s["parameters"]]
    if case["norm"] == "inf":
        norm = torch.stack([g.float().abs().max() for g in grads]).max()
    elif case["norm"] == "1":
        norm = torch.stack([g.float().abs().sum() for g in grads]).sum()
    else:
        norm = torch.stack([(g.float() * g.float()).sum() for g in grads]).sum().sqrt()
    coef = (limit / (norm + 1e-6)).clamp(max=1.0)
    for g in grads:
        g.copy_(g.float() * coef)
    return [norm, *s["buffers"]]


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case: dict) -> dict:
    if case["path"] == "logp":
        rows, b = case["batch"] * (case["seq"] - case["prompt"]), BYTES[case["dtype"]]
        n = rows * case["vocab"]
        # the logits of rows that count in, all rows of their gradient out; labels, results and their gradients
        out = case["batch"] * case["seq"] * case["vocab"] * b if case["grad"] else 0
        return {"bytes": n * b + out + case["batch"] * case["seq"] * (8 + 4 * (1 + case["entropy"]) * (1 + case["grad"])),
                "flops": n * (4 + 2 * case["entropy"] + 4 * case["grad"])}
    if case["path"] == "policy":
        n, b = case["batch"] * case["seq"], BYTES[case["dtype"]]
        size = n * ((4 if case["beta"] else 3) * b + BYTES[case["mask"]]) + 4 * (n if case["per_token"] else case["batch"])
        return {"bytes": size, "flops": n * (20 if case["beta"] else 12)}
    if case["path"] == "preference":
        n, b = 2 * case["pairs"] * case["seq"], BYTES[case["dtype"]]
        return {"bytes": n * ((3 if case["ref"] else 2) * b + BYTES[case["mask"]]), "flops": 6 * n}
    size = [math.prod(s) for s in _shapes(case)]
    held = sum(n * (4 if t == torch.float32 else 2) for n, t in zip(size, _types(case)))
    return {"bytes": held * (2 if case["active"] else 1), "flops": sum(size) * (3 if case["active"] else 2)}


# ------------------------------------------------------------------------------------------------ the same in 64 bits
def exact(case: dict, seed: int):
    s = prepare(case, seed)
    make = {"logp": _exact_logp, "policy": _exact_policy, "preference": _exact_preference, "clip": _exact_clip}
    return make[case["path"]](s, case)


def _exact_logp(s, case):
    """Derivatives by differentiating the definition, a few rows of the vocabulary at a time."""
    V = case["vocab"]
    logits, labels = s["logits"].reshape(-1, V), s["labels"].reshape(-1)
    logps, entropies, grads = [], [], []
    for r in torch.arange(len(labels), device=DEVICE).split(max(1, (1 << 25) // V)):
        x = logits[r].double().requires_grad_(case["grad"])
        z = case["cap"] * torch.tanh(x / case["cap"]) if case["cap"] else x
        log_p = torch.log_softmax(z / case["temperature"], -1)
        valid = (labels[r] != IGNORE).double()
        logp = log_p.gather(1, labels[r].clamp(min=0).unsqueeze(1)).squeeze(1) * valid
        entropy = -(log_p.exp() * log_p).sum(-1) * valid
        logps.append(logp.detach())
        entropies.append(entropy.detach())
        if case["grad"]:
            total = (logp * s["g"].reshape(-1)[r]).sum()
            if case["entropy"]:
                total = total + (entropy * s["h"].reshape(-1)[r]).sum()
            grads.append(torch.autograd.grad(total, x)[0])
    out = [torch.cat(logps).view(s["labels"].shape)]
    if case["entropy"]:
        out.append(torch.cat(entropies).view(s["labels"].shape))
    if case["grad"]:
        out.append(torch.cat(grads).view(s["logits"].shape))
    return out


def _exact_policy(s, case):
    logp = s["logp"].detach().double().requires_grad_()
    mask, a = s["mask"].double(), s["advantages"].double()
    a = a if case["per_token"] else a.unsqueeze(1)
    ratio = torch.exp(logp - s["old"].double())
    surrogate = torch.minimum(ratio * a, ratio.clamp(1 - case["low"], 1 + case["high"]) * a)
    kl = torch.zeros_like(logp)
    if s["ref"] is not None:
        d = s["ref"].double() - logp
        kl = torch.expm1(d) - d
    token = (case["beta"] * kl - surrogate) * mask
    if case["reduction"] == "sequence":
        loss = (token.sum(1) / mask.sum(1).clamp(min=1)).mean()
    else:
        loss = token.sum() / (mask.sum().clamp(min=1) if case["reduction"] == "token" else mask.numel())
    (grad,) = torch.autograd.grad(loss, logp)
    share = mask / mask.sum().clamp(min=1)
    clipped = (surrogate < ratio * a).double()
    return [loss.detach(), grad, *((x.detach() * share).sum() for x in (kl, clipped, ratio))]


def _exact_preference(s, case):
    logp, P = s["logp"].detach().double().requires_grad_(), case["pairs"]
    mask = s["mask"].double()
    count = mask.sum(1).clamp(min=1)
    own_score = (logp * mask).sum(1)
    score = own_score if s["ref"] is None else own_score - (s["ref"].double() * mask).sum(1)
    if case["normalized"]:
        score = score / count
    x, b, eps = score[:P] - score[P:], case["beta"], case["smoothing"]
    m = b * x - case["gamma"]
    good, bad = torch.nn.functional.logsigmoid(m), torch.nn.functional.logsigmoid(-m)
    loss = {"sigmoid": lambda: -(1 - eps) * good - eps * bad, "robust": lambda: (eps * bad - (1 - eps) * good) / (1 - 2 * eps),
            "hinge": lambda: torch.relu(1 - m), "ipo": lambda: (x - 1 / (2 * b)) ** 2}[case["kind"]]()
    loss = (loss - case["nll"] * own_score[:P] / count[:P]).mean()
    (grad,) = torch.autograd.grad(loss, logp)
    return [loss.detach(), b * score[:P].detach(), b * score[P:].detach(), grad]


def _norm64(grads, kind: str):
    if kind == "inf":
        return torch.stack([g.abs().max().double() for g in grads]).max()
    parts = [c.double() for g in grads for c in g.reshape(-1).split(1 << 26)]
    if kind == "1":
        return torch.stack([c.abs().sum() for c in parts]).sum()
    return torch.stack([(c * c).sum() for c in parts]).sum().sqrt()


def _exact_clip(s, case):
    norm = _norm64(s["buffers"], case["norm"])
    coef = (s["limit"] / (norm + 1e-6)).clamp(max=1.0)
    return [norm, *(b.double() * coef for b in s["buffers"])]
