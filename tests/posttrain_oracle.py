"""Definitions in fp64 of the operators between a model's logits and its update, written apart from the framework's code."""
import math

import torch


def token_oracle(z, y, temperature=1.0, cap=0.0, scale=0.0, ignore=-100):
    """(log-probabilities, entropies), differentiable in z; 0 log 0 is 0."""
    z = z.double()
    if cap:
        z = cap * torch.tanh(z / cap)
    z = z * (scale or 1.0) / temperature
    lp = z - torch.logsumexp(z, -1, keepdim=True)
    flat, rows = lp.reshape(-1, lp.shape[-1]), []
    ent = []
    for r, label in enumerate(y.reshape(-1).tolist()):
        if label == ignore:
            rows.append(flat.new_zeros(()))
            ent.append(flat.new_zeros(()))
            continue
        rows.append(flat[r, label])
        some = flat[r][flat[r] > -math.inf]
        ent.append(-(some.exp() * some).sum())
    return torch.stack(rows).view(y.shape), torch.stack(ent).view(y.shape)


def policy_oracle(logp, old, adv, mask, ref, low, high, beta, reduction, length):
    """(loss, gradient, (kl, share of clipped tokens, ratio)), token by token in Python's floats for small inputs, by the formula."""
    B, T = logp.shape
    m = mask.double()
    used = m != 0
    a = (adv if adv.dim() == 2 else adv.unsqueeze(1)).double().expand(B, T)
    lp, o = torch.where(used, logp.double(), 0.0), torch.where(used, old.double(), 0.0)
    r = (lp - o).exp()
    clipped = ((a > 0) & (r > 1 + high)) | ((a < 0) & (r < 1 - low))
    bound = torch.where(a > 0, torch.full_like(r, 1 + high), torch.full_like(r, 1 - low))
    token, slope = -a * torch.where(clipped, bound, r), torch.where(clipped, 0.0, -a * r)
    kl = torch.zeros_like(r)
    if ref is not None:
        d = torch.where(used, ref.double(), 0.0) - lp
        kl = torch.where(d.abs() < 1e-2, d * d / 2 * (1 + d / 3 * (1 + d / 4 * (1 + d / 5 * (1 + d / 6)))), d.exp() - 1 - d)
        token, slope = token + beta * kl, slope + beta * (1 - d.exp())
    if reduction == "sequence":
        w = (1.0 / m.sum(1).clamp(min=1) / B).unsqueeze(1)
    elif reduction == "token":
        w = 1.0 / m.sum().clamp(min=1)
    else:
        w = 1.0 / (B * length)
    n = m.sum().clamp(min=1)
    return (token * m * w).sum(), slope * m * w, ((kl * m).sum() / n, (clipped * m).sum() / n, (r * m).sum() / n)


def preference_oracle(lp, ref, mask, beta, kind, eps, gamma, normalized, nll):
    """(loss, chosen rewards, rejected rewards, gradient), pair by pair in Python's floats."""
    R, T = lp.shape
    P = R // 2
    m = mask.double().cpu()
    v = torch.where(m != 0, lp.double().cpu(), 0.0)
    b = torch.zeros_like(v) if ref is None else torch.where(m != 0, ref.double().cpu(), 0.0)
    n = m.sum(1).clamp(min=1)
    own = (v * m).sum(1)
    s = ((v - b) * m).sum(1)
    if normalized:
        s = s / n
    total, grad = 0.0, torch.zeros_like(v)
    for p in range(P):
        x = float(s[p] - s[P + p])
        q = beta * x - gamma
        sig = lambda t: 1 / (1 + math.exp(-t)) if t > -700 else 0.0                        # noqa: E731
        log_sig = lambda t: min(t, 0.0) - math.log1p(math.exp(-abs(t)))                     # noqa: E731
        if kind == "sigmoid":
            loss, slope = -(1 - eps) * log_sig(q) - eps * log_sig(-q), beta * (eps * sig(q) - (1 - eps) * sig(-q))
        elif kind == "robust":
            loss = (-(1 - eps) * log_sig(q) + eps * log_sig(-q)) / (1 - 2 * eps)
            slope = -beta * ((1 - eps) * sig(-q) + eps * sig(q)) / (1 - 2 * eps)
        elif kind == "hinge":
            loss, slope = max(0.0, 1 - q), -beta if q < 1 else 0.0
        else:
            loss, slope = (x - 1 / (2 * beta)) ** 2, 2 * (x - 1 / (2 * beta))
        total += loss - nll * float(own[p] / n[p])
        for row, sign in ((p, 1.0), (P + p, -1.0)):
            grad[row] = sign * slope * m[row] / (float(n[row]) if normalized else 1.0)
        grad[p] -= nll * m[p] / n[p]
    rewards = beta * s
    return torch.tensor(total / P, dtype=torch.float64), rewards[:P], rewards[P:], grad / P
