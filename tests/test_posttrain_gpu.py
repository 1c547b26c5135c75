"""Kernels between a model's logits and its update (csrc/logprob.cu, csrc/posttrain.cu, csrc/gradnorm.cu) against definitions in
fp64.  Tolerances count roundings: half a step of the result's type, and what fp32 exponentials and sums may be off by."""
import math

import pytest
import torch

from posttrain_oracle import policy_oracle, preference_oracle

pytestmark = pytest.mark.gpu
DEV = "cuda"
HALF = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.bfloat16, torch.float16)}
F32 = HALF[torch.float32]


def _gen(seed):
    return torch.Generator(DEV).manual_seed(seed)


def _near(got, want, tol):
    """|got - want| <= tol elementwise; equal where not finite."""
    got, want = got.double(), want.double()
    finite = want.isfinite()
    assert torch.equal(finite, got.isfinite()), "finite in other places"
    off = (got - want).abs() - tol
    worst = off.where(finite, -1.0).max() if off.numel() else torch.tensor(-1.0)
    assert float(worst) <= 0, f"off by {float(worst):.3e} more than allowed"
    assert torch.equal(got[~finite].nan_to_num(7.0), want[~finite].nan_to_num(7.0))


# ------------------------------------------------------------------------------------------------ log-probabilities
def _token64(z, y, temperature, cap, g, h):
    """Log-probabilities, entropies, gradient, and what fp32 may be off by in each: rows' largest |logit| counts in the exponent's
    rounding, the number of terms of a thread in a sum's, two units in the last place in an exponential's."""
    V = z.shape[-1]
    x = z.double()
    t = torch.tanh(x / cap) if cap else None
    v = (cap * t if cap else x) / temperature
    slope = (1 - t * t if cap else torch.ones_like(x)) / temperature
    used = y != -100
    lse = torch.logsumexp(v, -1, keepdim=True)
    lp = v - lse
    p = lp.exp()
    safe = lp.where(p > 0, 0.0)
    at = y.where(used, 0).unsqueeze(-1)
    logp = lp.gather(-1, at).squeeze(-1).where(used, 0.0)
    H = -(p * safe).sum(-1)
    big = v.where(v.isfinite(), 0.0).abs().amax(-1) + (cap / temperature if cap else 0.0)
    tol = F32 * (8 * big + V / 256 + 64)
    g, h = (torch.zeros_like(H) if d is None else d.double().where(used, 0.0) for d in (g, h))
    one = torch.zeros_like(x).scatter_(-1, at, 1.0)
    grad = slope * (one * g.unsqueeze(-1) - p * (g.unsqueeze(-1) + h.unsqueeze(-1) * (safe + H.unsqueeze(-1))))
    size = slope.abs().amax(-1) * (g.abs() + h.abs() * (H + 1 + safe.abs().amax(-1)))
    return logp, H.where(used, 0.0), grad, tol, tol * 4 * (1 + H), (size * tol * 4).unsqueeze(-1)


def _check_tokens(z, y, temperature=1.0, cap=0.0, entropy=True, seed=0):
    from trainscale_b200.rl import token_log_probs
    g, h = (torch.randn(y.shape, device=DEV, generator=_gen(seed + i)) for i in (1, 2))
    h = h if entropy else None
    logp, H, grad, tol, tol_H, tol_grad = _token64(z, y, temperature, cap, g, h)
    a = dict(temperature=temperature, logit_softcapping=cap, return_entropy=entropy)
    out = token_log_probs(z, y, **a)
    out = out if entropy else (out,)
    _near(out[0], logp, tol + F32 * logp.abs().where(logp.isfinite(), 0.0))
    if entropy:
        _near(out[1], H, tol_H)
    x = z.detach().requires_grad_()
    again = token_log_probs(x, y, **a)
    again = again if entropy else (again,)
    assert all(torch.equal(u, v) for u, v in zip(out, again))
    (d,) = torch.autograd.grad(again, x, (g, h) if entropy else (g,))
    assert d.dtype == z.dtype and d.shape == z.shape
    _near(d, grad, tol_grad + HALF[z.dtype] * grad.abs() * 1.01 + (2.0 ** -25 if z.dtype == torch.float16 else 0.0))
    assert (d[y == -100] == 0).all()


@pytest.mark.parametrize("dtype", list(HALF))
@pytest.mark.parametrize("V", [1, 2, 7, 8, 33, 1000, 1001, 4099, 32001])
def test_token_log_probs(V, dtype):
    z = (torch.randn(2, 9, V, device=DEV, generator=_gen(V)) * 3).to(dtype)
    y = torch.randint(0, V, (2, 9), device=DEV, generator=_gen(V + 1))
    y[0, :3] = -100
    _check_tokens(z, y)


@pytest.mark.parametrize("entropy", [False, True])
@pytest.mark.parametrize("cap", [0.0, 20.0])
@pytest.mark.parametrize("rows,V,dtype", [(1, 128256, torch.bfloat16), (9, 128256, torch.float32), (150, 50001, torch.float16),
                                          (700, 32000, torch.bfloat16)])
def test_token_log_probs_of_few_and_many_rows(rows, V, dtype, cap, entropy):
    z = (torch.randn(rows, V, device=DEV, generator=_gen(rows)) * 6).to(dtype)
    y = torch.randint(0, V, (rows,), device=DEV, generator=_gen(rows + 1))
    _check_tokens(z, y, 0.6, cap, entropy)


def _gradient64(z, y, temperature, cap, g, h):
    """The gradient, and what fp32 may be off by in each of its elements.  A probability p_j is off by what its logarithm is: the
    roundings of its exponent (4 of F32 times the largest |logit| and the distance between logits), of an exponential (two units in the
    last place) and of the sum it is divided by (as many additions as a thread makes, at most V / 256 + 32).  With a cap, tanh and its
    slope add 2^-21 each.  ln p + H is off by as much, against 1 + |ln p| + H; the chosen token's g by three roundings.  Exponentials
    below 2^-126 are zero."""
    V = z.shape[-1]
    x = z.double()
    t = torch.tanh(x / cap) if cap else None
    v = (cap * t if cap else x) / temperature
    slope = (1 - t * t if cap else torch.ones_like(x)) / temperature
    lp = torch.log_softmax(v, -1)
    p, used = lp.exp(), (y != -100).unsqueeze(-1)
    H = -(p * lp).sum(-1, keepdim=True)
    one = torch.zeros_like(x).scatter_(-1, y.clamp(min=0).unsqueeze(-1), 1.0)
    g, h = (torch.zeros_like(H) if d is None else d.double().unsqueeze(-1) for d in (g, h))
    grad = slope * (one * g - p * (g + h * (lp + H)))
    big = v.abs().amax(-1, keepdim=True) + (v - v.amax(-1, keepdim=True)).abs()
    rel = F32 * (4 * big + V / 256 + 40) + (2.0 ** -21 * (2 + big) if cap else 0.0)
    tol = slope * (p * rel * (g.abs() + 2 * h.abs() * (1 + lp.abs() + H)) + one * g.abs() * (3 * F32 + (2.0 ** -21 if cap else 0.0)))
    tol = tol + 2.0 ** -126 * (g.abs() + h.abs() * 200) + HALF[z.dtype] * grad.abs() * 1.01 + (2.0 ** -25 if z.dtype == torch.float16 else 2.0 ** -133)
    return grad.where(used, 0.0), tol.where(used, 0.0)


@pytest.mark.parametrize("entropy", [False, True])
@pytest.mark.parametrize("cap", [0.0, 20.0])
@pytest.mark.parametrize("dtype", list(HALF))
@pytest.mark.parametrize("rows,V,first", [(19, 4099, 0), (19, 4099, 3), (19, 4104, 8), (3, 50001, 0), (620, 9001, 5)])
def test_gradients_of_every_logit(rows, V, first, dtype, cap, entropy):
    """Each element against its own size: a vector left out, a wrong tail or a missing term would show in any column."""
    from trainscale_b200.rl import token_log_probs
    z = (torch.randn(rows, first + V, device=DEV, generator=_gen(V)) * 3).to(dtype)[:, first:]
    y = torch.randint(0, V, (rows,), device=DEV, generator=_gen(V + 1))
    y[1] = -100
    scale = 4096.0 if dtype == torch.float16 else 1.0       # (a loss scale, as training in fp16 has it)
    g, h = (torch.randn(rows, device=DEV, generator=_gen(i)) * scale for i in (1, 2))
    h = h if entropy else None
    x = z.detach().requires_grad_()
    out = token_log_probs(x, y, temperature=0.8, logit_softcapping=cap, return_entropy=entropy)
    (d,) = torch.autograd.grad(out, x, (g, h) if entropy else (g,))
    grad, tol = _gradient64(z, y, 0.8, cap, g, h)
    used = y != -100
    # the test looks at nearly every element: few are as small as what they may be off by
    assert float((grad[used].abs() > 4 * tol[used]).double().mean()) > (0.85 if dtype == torch.float16 else 0.99)
    _near(d, grad, tol)


@pytest.mark.parametrize("V", [515, 520])
def test_rows_that_lie_elsewhere(V):
    """Slices, pitched rows, unaligned starts, transposed storage, one row, four dimensions."""
    for dtype in HALF:
        full = (torch.randn(3, 8, V + 5, device=DEV, generator=_gen(5)) * 2).to(dtype)
        for z in (full[:, :-1, :V], full[:, 1:, 3:3 + V], full[::2, ::3, 5:], full[1, :, :V], full[0, 2, 1:1 + V],
                  full[:, :, :V].transpose(1, 2).contiguous().transpose(1, 2), full[:, :, :V].unsqueeze(1).expand(3, 2, 8, V)):
            y = torch.randint(0, z.shape[-1], z.shape[:-1], device=DEV, generator=_gen(6))
            _check_tokens(z, y)


@pytest.mark.parametrize("dtype", list(HALF))
def test_logits_that_are_not_finite_or_far_apart(dtype):
    from trainscale_b200.rl import token_log_probs
    V = 777
    z = torch.randn(8, V, device=DEV, generator=_gen(1)).to(dtype)
    z[0, 1:] = -math.inf                                    # one token left
    z[1, ::2] = -math.inf
    z[2, :] = torch.finfo(dtype).min                        # a mask of the lowest value over everything
    z[3, :-1] = torch.finfo(dtype).min
    z[4, 5] = 3e4                                           # one that drowns the others
    z[5] = 60000.0
    z[6] *= 1e-4
    y = torch.tensor([0, 2, 3, 776, 6, 1, 1, 0], device=DEV)
    want = torch.log_softmax(z.double(), -1).gather(1, y.unsqueeze(1)).squeeze(1)
    got, H = token_log_probs(z, y, return_entropy=True)
    _near(got, want, F32 * (8 * z.double().where(z.isfinite() & (z > -1e4), 0.0).abs().amax(1) + 128) + F32 * want.abs().where(want.isfinite(), 0.0) * 2)
    assert float(H[0]) == 0 and float(H[3]) == 0 and abs(float(H[2]) - math.log(V)) < 1e-5 and abs(float(H[5]) - math.log(V)) < 1e-5
    x = z.clone().requires_grad_()
    logp, H = token_log_probs(x, y, return_entropy=True)
    (logp.where(logp.isfinite(), 0.0).sum() + H.sum()).backward()
    assert x.grad.isfinite().all() and float(x.grad[0].abs().max()) == 0 and (x.grad[1, ::2] == 0)[1:].all()
    bad = torch.zeros(5, V, device=DEV, dtype=dtype)
    bad[0], bad[1, 700], bad[2, 3], bad[3, 3], bad[3, 4] = -math.inf, math.nan, math.inf, math.inf, math.nan
    lp, H = token_log_probs(bad, torch.tensor([0, 0, 0, 3, 0], device=DEV), return_entropy=True)
    assert lp[:2].isnan().all() and float(lp[2]) == -math.inf and lp[3].isnan() and lp[4].isfinite() and H[:4].isnan().all()
    lp = token_log_probs(bad, torch.tensor([-100, -100, V, -1, 5], device=DEV))
    assert (lp[:2] == 0).all() and lp[2:4].isnan().all()


@pytest.mark.parametrize("cap", [0.5, 5.0, 300.0, 1e6])
def test_caps_far_below_and_above_the_logits(cap):
    """A capped logit is off by 2^-21 of its own size, however large the cap."""
    from trainscale_b200.rl import token_log_probs
    z = torch.randn(400, 999, device=DEV, generator=_gen(8)) * 4
    z[0] *= 1e-3
    y = torch.randint(0, 999, (400,), device=DEV, generator=_gen(9))
    v = cap * torch.tanh(z.double() / cap)
    want = torch.log_softmax(v, -1).gather(1, y.unsqueeze(1)).squeeze(1)
    tol = F32 * (24 * v.abs().amax(1) + 64) + F32 * want.abs()
    for rows in (400, 3):                                   # a warp per part of a row, and a block per row
        _near(token_log_probs(z[:rows], y[:rows], logit_softcapping=cap), want[:rows], tol[:rows])


def _pytorch_capped(z, y, cap):
    v = cap * torch.tanh(z / cap)
    return v.gather(1, y.unsqueeze(1)).squeeze(1) - torch.logsumexp(v, -1)


def _rms(got, want):
    return float((got.double() - want).pow(2).mean().sqrt())


@pytest.mark.parametrize("cap", [5.0, 30.0])
def test_a_capped_logit_is_as_good_as_the_librarys(cap):
    """Of two logits, 0 and z < 0, z is chosen: its log-probability is c tanh(z / c), less a logarithm that is small where z is far.  It is
    off by the roundings of 1 / c, of z / c, of the product by c and of the difference (2^-24 each), by tanh (2^-23) and by the logarithm's
    few units."""
    from trainscale_b200.rl import token_log_probs
    x = torch.rand(400000, device=DEV, generator=_gen(3)) * 3 + 1e-3
    z = torch.stack((torch.zeros_like(x), -x * cap), 1)
    y = torch.ones(len(x), dtype=torch.long, device=DEV)
    v = cap * torch.tanh(z[:, 1].double() / cap)
    want = v - torch.log1p(v.exp())
    got = token_log_probs(z, y, logit_softcapping=cap)
    _near(got, want, F32 * (6 * v.abs() + 4))
    plain = _pytorch_capped(z, y, cap)
    assert _rms(got, want) <= 1.1 * _rms(plain, want)


@pytest.mark.parametrize("rows", [900, 30])
@pytest.mark.parametrize("cap", [5.0, 30.0])
def test_capped_log_probabilities_are_as_good_as_the_pytorch_form(cap, rows):
    """Many rows (a warp each) and few (blocks): errors against 64 bits, forward and backward, no larger in the mean.  A root mean square
    of n independent errors is itself uncertain by 1 / sqrt(2 n) of its value, the quotient of two by 1 / sqrt(n), and n is the number of
    rows (a gradient's errors are largest at its row's label): three times that is allowed, 10 % for 900 rows and 55 % for 30."""
    from trainscale_b200.rl import token_log_probs
    z = torch.randn(rows, 4100, device=DEV, generator=_gen(5)) * 4
    y = torch.randint(0, 4100, (rows,), device=DEV, generator=_gen(6))

    def both(f, z):
        z = z.detach().requires_grad_()
        logp = f(z, y)
        return logp.detach(), torch.autograd.grad(logp.sum(), z)[0]

    want = both(lambda z, y: _pytorch_capped(z, y, cap), z.double())
    got, plain = both(lambda z, y: token_log_probs(z, y, logit_softcapping=cap), z), both(lambda z, y: _pytorch_capped(z, y, cap), z)
    for g, p, w in zip(got, plain, want):
        assert _rms(g, w) <= (1 + 3 / math.sqrt(rows)) * _rms(p, w)


def test_offsets_that_pass_32_bits():
    from trainscale_b200.rl import token_log_probs
    rows, V = 16500, 131080                                 # 2.16e9 logits
    z = torch.zeros(rows, V, device=DEV, dtype=torch.bfloat16)
    some = torch.tensor([0, 1, 16383, 16384, rows - 1], device=DEV)
    z[some] = (torch.randn(5, V, device=DEV, generator=_gen(1)) * 2).bfloat16()
    y = torch.randint(0, V, (rows,), device=DEV, generator=_gen(2))
    x = z.requires_grad_()
    logp = token_log_probs(x, y)
    want = torch.log_softmax(z[some].detach().double(), -1)
    _near(logp[some].detach(), want.gather(1, y[some].unsqueeze(1)).squeeze(1), F32 * 1000)
    (d,) = torch.autograd.grad(logp.sum(), x)
    one = torch.zeros_like(want).scatter_(1, y[some].unsqueeze(1), 1.0)
    _near(d[some], one - want.exp(), 2e-4 * want.exp() + HALF[torch.bfloat16] * (one - want.exp()).abs() * 1.01)
    assert float(logp[777]) == pytest.approx(-math.log(V), rel=1e-6)
    del x, z, d
    stride = (1 << 31) + 8                                  # rows of losses that lie that far apart
    far = torch.empty(3 * stride + 100, device=DEV, dtype=torch.bfloat16).as_strided((4, 100), (stride, 1))
    logp, old, adv, mask, ref = _policy_case(4, 100, torch.bfloat16, torch.bool, 3)
    _check_policy(far.copy_(logp), old, adv, mask, ref)
    lp, rf, m = _pair_case(2, 100, torch.bfloat16, torch.bool, 3)
    _check_pairs(far.copy_(lp), rf, m)
    del far
    g = torch.full(((1 << 31) + 77,), 2.0, device=DEV, dtype=torch.bfloat16)
    assert float(_clip([g], 1.0)) == pytest.approx(2 * math.sqrt(g.numel()), rel=1e-6)
    want = 1.0 / math.sqrt(g.numel())
    assert float(g[0]) == pytest.approx(want, rel=4e-3) and float(g[-1]) == float(g[0]) == float(g[1 << 31])


def test_constants_made_in_inference_mode():
    from trainscale_b200.rl import clipped_policy_loss, preference_loss, token_log_probs
    logp, old, adv, mask, ref = _policy_case(6, 50, torch.float32, torch.bool, 3)
    with torch.inference_mode():
        a = [t.clone() for t in (old, adv, mask, ref)]
        y = torch.arange(6, device=DEV)
    x = logp.clone().requires_grad_()
    loss = clipped_policy_loss(x, *a, beta=0.1)
    loss.backward()
    z = logp.clone().requires_grad_()
    clipped_policy_loss(z, old, adv, mask, ref, beta=0.1).backward()
    assert torch.equal(x.grad, z.grad)
    x = logp.clone().requires_grad_()
    preference_loss(x, a[3], a[2])[0].backward()
    w = torch.randn(6, 9, device=DEV, requires_grad=True)
    token_log_probs(w, y).sum().backward()
    with torch.inference_mode():
        clipped_policy_loss(logp, *a, beta=0.1)
        token_log_probs(w, y, return_entropy=True)


def test_broadcast_inputs():
    """A row that several sequences share gets the sum of their gradients."""
    from trainscale_b200.rl import clipped_policy_loss, preference_loss, token_log_probs
    logp, old, adv, mask, ref = _policy_case(6, 52, torch.float32, torch.bool, 3, spoil=False)
    one = logp[:1].clone().requires_grad_()
    clipped_policy_loss(one.expand(6, 52), old, adv, mask, ref, beta=0.1).backward()
    _, grad, _ = policy_oracle(logp[:1].expand(6, 52), old, adv, mask, ref, 0.2, 0.2, 0.1, "sequence", 52)
    torch.testing.assert_close(one.grad.double(), grad.sum(0, keepdim=True), rtol=1e-5, atol=1e-8)
    one = logp[:1].clone().requires_grad_()
    preference_loss(one.expand(6, 52), ref, mask, loss_type="ipo")[0].backward()
    *_, grad = preference_oracle(logp[:1].expand(6, 52), ref, mask, 0.1, "ipo", 0.0, 0.0, False, 0.0)
    torch.testing.assert_close(one.grad.double().cpu(), grad.sum(0, keepdim=True), rtol=1e-5, atol=1e-8)
    z = torch.randn(1, 1, 99, device=DEV, requires_grad=True)
    y = torch.arange(12, device=DEV).view(3, 4)
    token_log_probs(z.expand(3, 4, 99), y).sum().backward()
    p = torch.softmax(z.detach().double(), -1)
    torch.testing.assert_close(z.grad.double(), (torch.arange(99, device=DEV) < 12).double() - 12 * p, rtol=1e-4, atol=1e-5)


def test_transforms_take_the_pytorch_form():
    """torch.func and forward-mode derivatives, which cannot see into a kernel."""
    from trainscale_b200.rl import clipped_policy_loss, preference_loss, token_log_probs
    logp, old, adv, mask, ref = _policy_case(6, 20, torch.float32, torch.bool, 3, spoil=False)
    for f in (lambda p: clipped_policy_loss(p, old, adv, mask, ref, beta=0.1), lambda p: preference_loss(p, ref, mask)[0]):
        x = logp.clone().requires_grad_()
        f(x).backward()
        torch.testing.assert_close(torch.func.grad(f)(logp), x.grad, rtol=1e-4, atol=1e-7)
        _, tangent = torch.func.jvp(f, (logp,), (torch.ones_like(logp),))
        torch.testing.assert_close(tangent, x.grad.sum(), rtol=1e-4, atol=1e-6)
    z, y = torch.randn(5, 3, 33, device=DEV), torch.randint(0, 33, (5, 3), device=DEV)
    torch.testing.assert_close(torch.func.vmap(token_log_probs)(z, y), token_log_probs(z, y), rtol=1e-5, atol=1e-5)


def _recorded_calls():
    """(name, function of one tensor, its argument) of everything that has PyTorch operations to record."""
    from trainscale_b200 import rl
    from trainscale_b200.optim import clip_grad_norm_
    from trainscale_b200.parallel.dist_utils import fused_clip_grad_norm_
    logp, old, adv, mask, ref = _policy_case(6, 52, torch.float32, torch.float32, 3, spoil=False)
    y = torch.randint(0, 33, (5,), device=DEV, generator=_gen(1))
    z = torch.randn(5, 33, device=DEV, generator=_gen(2))

    def clipped(clip):
        def f(g):
            p = torch.nn.Parameter(torch.zeros_like(g))
            p.grad = g.clone()
            return clip([p], 0.5), p.grad
        return f

    return [("selective_log_softmax", lambda z: rl.selective_log_softmax(z, y), z), ("token_log_probs", lambda z: rl.token_log_probs(z, y), z),
            ("grpo", lambda x: rl.grpo_loss(x, old, ref, adv, mask), logp), ("drgrpo", lambda x: rl.drgrpo_loss(x, old, adv, mask), logp),
            ("dapo", lambda x: rl.dapo_loss(x, old, adv, mask), logp), ("pairs", lambda x: rl.preference_loss(x, ref, mask)[0], logp),
            ("clip", clipped(clip_grad_norm_), logp), ("fused clip", clipped(fused_clip_grad_norm_), logp)]


@pytest.mark.parametrize("how", ["jit.trace", "make_fx", "compile"])
def test_recorded_calls_replay(how):
    """A recording holds the operations, not the memory that a kernel once filled."""
    from torch.fx.experimental.proxy_tensor import make_fx
    for name, f, x in _recorded_calls():
        if how == "compile" and "clip" in name:
            continue                                        # (a parameter made inside: not for fullgraph)
        recorded = {"jit.trace": lambda: torch.jit.trace(f, x, check_trace=False), "make_fx": lambda: make_fx(f)(x),
                    "compile": lambda: torch.compile(f, backend="eager", fullgraph=True)}[how]()
        other = x * 0.5 + 0.1
        for a, b in zip(*[(t if isinstance(t, tuple) else (t,)) for t in (recorded(other), f(other))]):
            torch.testing.assert_close(a, b, rtol=1e-4, atol=1e-6, msg=lambda m: f"{name}: {m}")


def test_recorded_gradients_replay():
    """The gradient of a loss that a kernel has computed, recorded as a function of what flows into it."""
    from torch.fx.experimental.proxy_tensor import make_fx
    for name, f, x in _recorded_calls()[:6]:
        x = x.clone().requires_grad_()
        out = f(x)
        assert type(out.grad_fn).__name__ in ("_LossBackward", "_TokenLogProbsBackward"), name
        grad = lambda g: torch.autograd.grad(out, x, g, retain_graph=True)[0]       # noqa: E731, B023
        recorded = make_fx(grad)(torch.ones_like(out))
        g = torch.rand_like(out)
        torch.testing.assert_close(recorded(g), grad(g), rtol=1e-4, atol=1e-7, msg=lambda m: f"{name}: {m}")


def test_batched_gradients():
    """Several upstream gradients in one backward pass, and Jacobians made of them."""
    from trainscale_b200 import rl
    for name, f, x in _recorded_calls()[:6]:
        x = x.clone().requires_grad_()
        out = f(x)
        many = torch.randn(4, *out.shape, device=DEV, generator=_gen(9))
        (got,) = torch.autograd.grad(out, x, many, is_grads_batched=True, retain_graph=True)
        want = torch.stack([torch.autograd.grad(out, x, g, retain_graph=True)[0] for g in many])
        torch.testing.assert_close(got, want, rtol=1e-4, atol=1e-7, msg=lambda m: f"{name}: {m}")
        torch.testing.assert_close(torch.autograd.functional.jacobian(f, x, vectorize=True), torch.autograd.functional.jacobian(f, x),
                                   rtol=1e-4, atol=1e-7, msg=lambda m: f"{name}: {m}")
    z, y = torch.randn(4, 9, device=DEV, requires_grad=True), torch.arange(4, device=DEV)
    _, H = rl.token_log_probs(z, y, return_entropy=True)
    many = torch.randn(3, 4, device=DEV)
    (got,) = torch.autograd.grad(H, z, many, is_grads_batched=True, retain_graph=True)
    for g, d in zip(many, got):
        torch.testing.assert_close(d, torch.autograd.grad(H, z, g, retain_graph=True)[0], rtol=1e-4, atol=1e-6)


def test_two_streams_at_once():
    """Calls that run side by side have workspaces of their own."""
    from trainscale_b200.rl import clipped_policy_loss, preference_loss, token_log_probs
    cases = [(_policy_case(500, 700, torch.float32, torch.bool, i), _pair_case(200, 3000, torch.float32, torch.bool, i),
              torch.randn(700, 9000, device=DEV, generator=_gen(i))) for i in range(2)]
    y = torch.randint(0, 9000, (700,), device=DEV)

    def run(case):
        (logp, old, adv, mask, ref), (lp, rf, m), z = case
        grads = [z.clone(), lp.nan_to_num(neginf=0.0)]
        return [*clipped_policy_loss(logp, old, adv, mask, ref, beta=0.1, return_stats=True)[1], *preference_loss(lp, rf, m),
                *token_log_probs(z, y, return_entropy=True), _clip(grads, 1.0), *grads]

    want = [run(c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(5):
        got = []
        for s, c in zip(streams, cases):
            with torch.cuda.stream(s):
                got.append(run(c))
        torch.cuda.synchronize()
        for a, b in zip(want, got):
            assert all(torch.equal(u, v) for u, v in zip(a, b))


def test_inputs_changed_before_their_gradient():
    from trainscale_b200.rl import clipped_policy_loss
    logp, old, adv, mask, ref = _policy_case(6, 50, torch.float32, torch.bool, 3, spoil=False)
    x = logp.clone().requires_grad_()
    loss = clipped_policy_loss(x, old, adv, mask, ref, beta=0.1)
    (a,) = torch.autograd.grad(loss, x, retain_graph=True)
    old.zero_()                                             # a second pass would need it
    with pytest.raises(RuntimeError, match="changed in place"):
        torch.autograd.grad(loss, x)
    loss = clipped_policy_loss(x, old, adv, mask, ref, beta=0.1)
    loss.backward()
    with pytest.raises(RuntimeError, match="second time"):
        loss.backward()


def test_log_probabilities_changed_after_their_loss():
    """Their gradient is known by then; a loss that has to compute it again refuses."""
    from trainscale_b200 import rl
    logp, old, adv, mask, ref = _policy_case(6, 50, torch.float32, torch.float32, 3, spoil=False)
    for f in (lambda x: rl.grpo_loss(x, old, ref, adv, mask), lambda x: rl.drgrpo_loss(x, old, adv, mask),
              lambda x: rl.dapo_loss(x, old, adv, mask), lambda x: rl.preference_loss(x, ref, mask)[0]):
        leaf = logp.clone().requires_grad_()
        (want,) = torch.autograd.grad(f(leaf * 1), leaf)
        x = leaf * 1
        loss = f(x)
        x.zero_()
        (got,) = torch.autograd.grad(loss, leaf, retain_graph=True)
        assert torch.equal(got, want)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(loss, leaf)


def test_rows_without_an_upstream_gradient_and_unused_results():
    from trainscale_b200.rl import token_log_probs
    z = torch.randn(6, 300, device=DEV, requires_grad=True)
    y = torch.arange(6, device=DEV)
    logp, H = token_log_probs(z, y, return_entropy=True)
    w = torch.tensor([0.0, 1, 0, 2, 0, 3], device=DEV)
    (a,) = torch.autograd.grad((logp * w).sum(), z, retain_graph=True)
    assert (a[::2] == 0).all()
    torch.testing.assert_close(a, torch.autograd.grad((torch.log_softmax(z, -1)[y, y] * w).sum(), z)[0], rtol=1e-5, atol=1e-6)
    (b,) = torch.autograd.grad(H.sum(), z)
    lp = torch.log_softmax(z, -1)
    torch.testing.assert_close(b, torch.autograd.grad(-(lp.exp() * lp).sum(), z)[0], rtol=1e-4, atol=1e-6)
    logp, H = token_log_probs(z, y, return_entropy=True)
    logp *= 2                                               # results may be changed in place
    H += 1
    (logp.sum() + H.sum()).backward()


@pytest.mark.parametrize("T,V,chunk", [(37, 1000, 16), (700, 4003, 4096), (1, 129, 4)])
def test_log_probs_of_the_fused_head(T, V, chunk):
    """The chunked head on the same kernels, the gradient written over the logits; labels outside the vocabulary are ignored there."""
    from trainscale_b200.ops.cross_entropy import fused_linear_token_logprobs
    h = (torch.randn(T, 128, device=DEV, generator=_gen(1))).bfloat16().requires_grad_()
    w = (torch.randn(V, 128, device=DEV, generator=_gen(2)) * 0.3).bfloat16().requires_grad_()
    y = torch.randint(0, V, (T,), device=DEV, generator=_gen(3))
    if T > 3:
        y[0], y[1], y[2] = -100, V, -1
    g = torch.randn(T, device=DEV, generator=_gen(4))
    logp = fused_linear_token_logprobs(h, w, y, chunk_tokens=chunk)
    dh, dw = torch.autograd.grad(logp, (h, w), g)
    a, b = h.detach().double().requires_grad_(), w.detach().double().requires_grad_()
    z = a @ b.t()
    z = z + (z.bfloat16().double() - z).detach()            # logits are held in bf16
    used = (y >= 0) & (y < V)
    want = torch.log_softmax(z, -1).gather(1, y.where(used, 0).unsqueeze(1)).squeeze(1).where(used, 0.0)
    # (a logit that lies on a border of bf16 may fall to either side: 2^-8 of its size)
    _near(logp, want, 2.0 ** -8 * z.detach().abs().amax(1) * 2)
    ea, eb = torch.autograd.grad(want, (a, b), g.double())
    for d, e in ((dh, ea), (dw, eb)):
        assert float((d.double() - e).norm()) <= 2.0 ** -6 * float(e.norm())
    assert torch.equal(logp[~used], torch.zeros_like(logp[~used])) and (dh[~used] == 0).all()
    with torch.no_grad():
        assert torch.equal(logp, fused_linear_token_logprobs(h, w, y, chunk_tokens=chunk))


@pytest.mark.parametrize("case", ["every other", "column", "int32 column"])
def test_fused_head_reads_labels_that_lie_apart(case):
    """Labels of a tensor that can be viewed as one dimension and keeps a stride: log-probabilities, losses and their gradients."""
    from trainscale_b200.ops import cross_entropy as ce
    h = torch.randn(6, 128, device=DEV, generator=_gen(1)).bfloat16()
    w = (torch.randn(40, 128, device=DEV, generator=_gen(2)) * 0.3).bfloat16()
    ids = torch.randint(0, 40, (6, 2), device=DEV, generator=_gen(3))
    y = {"every other": ids.view(-1)[::2], "column": ids[:, 1:], "int32 column": ids.int()[:, 1:]}[case]
    assert not y.reshape(-1).is_contiguous()
    z = torch.randn(6, 40, device=DEV, generator=_gen(4)).bfloat16()
    calls = (lambda h, y: ce.fused_linear_token_logprobs(h, w, y).sum(), lambda h, y: ce.fused_linear_cross_entropy(h, w, y)[0],
             lambda h, y: ce.cross_entropy_rows(z + 0 * h[:, :40], y).sum(),
             lambda h, y: ce.focal_loss_rows(z + 0 * h[:, :40], y.reshape(-1)).sum(), lambda h, y: ce.cross_entropy_logits(z, y)[0].sum() + 0 * h.sum())
    for call in calls:
        out = []
        for labels in (y, y.long().clone(memory_format=torch.contiguous_format)):
            x = h.clone().requires_grad_()
            loss = call(x, labels)
            out.append((loss.detach(), *torch.autograd.grad(loss, x)))
        assert all(torch.equal(u, v) for u, v in zip(*out))


def test_selective_log_softmax_keeps_its_results():
    from trainscale_b200.rl import selective_log_softmax
    y = torch.randint(0, 999, (4, 5), device=DEV)
    for dtype, kw in ((torch.float32, dict(temperature=0.7, logit_softcapping=9.0, logit_scale=1.2)), (torch.float32, {}),
                      (torch.bfloat16, {}), (torch.bfloat16, dict(temperature=0.7, logit_softcapping=9.0))):
        z = (torch.randn(4, 5, 999, device=DEV, generator=_gen(3)) * 4).to(dtype)
        v = z
        if kw:
            v = kw["logit_softcapping"] * torch.tanh(z / kw["logit_softcapping"])
            v = v * kw.get("logit_scale", 1.0) / kw["temperature"] if "logit_scale" in kw else v / kw["temperature"]
        want = v.gather(-1, y.unsqueeze(-1)).squeeze(-1).float() - torch.logsumexp(v.float(), -1)
        torch.testing.assert_close(selective_log_softmax(z, y, **kw), want, rtol=2e-6, atol=2e-5)
    z = torch.randn(3, 7, device=DEV, requires_grad=True)   # a gradient that is differentiated itself
    (d,) = torch.autograd.grad(selective_log_softmax(z, torch.tensor([0, 3, 6], device=DEV)).sum(), z, create_graph=True)
    (dd,) = torch.autograd.grad(d.pow(2).sum(), z)
    x = z.detach().double().requires_grad_()
    (e,) = torch.autograd.grad(torch.log_softmax(x, -1)[[0, 1, 2], [0, 3, 6]].sum(), x, create_graph=True)
    (ee,) = torch.autograd.grad(e.pow(2).sum(), x)
    torch.testing.assert_close(dd.double(), ee, rtol=1e-4, atol=1e-5)


def test_an_index_outside_the_vocabulary():
    from trainscale_b200.rl import selective_log_softmax
    z = torch.randn(4, 9, device=DEV)
    for dtype in HALF:
        got = selective_log_softmax(z.to(dtype), torch.tensor([0, 9, -1, 8], device=DEV))
        assert got.isnan().tolist() == [False, True, True, False]
    with pytest.raises(RuntimeError):
        selective_log_softmax(z.cpu(), torch.tensor([0, 9, -1, 8]))


# ------------------------------------------------------------------------------------------------ policy loss
MASKS = [torch.bool, torch.uint8, torch.int32, torch.int64, torch.float32, torch.bfloat16, torch.float16, torch.float64]


def _policy_case(B, T, dtype, mask_type, seed, per_token=False, spoil=True):
    g = _gen(seed)
    logp = -torch.rand(B, T, device=DEV, generator=g) * 3
    old = (logp + 0.15 * torch.randn(B, T, device=DEV, generator=g)).to(dtype)
    ref = (logp + 0.4 * torch.randn(B, T, device=DEV, generator=g)).to(dtype)
    logp = logp.to(dtype)
    mask = torch.rand(B, T, device=DEV, generator=g) < 0.7
    if B > 1:
        mask[B // 2] = False
    if spoil:
        logp[~mask], old[~mask], ref[~mask] = math.nan, math.inf, -math.inf
    adv = torch.randn(B, T, device=DEV, generator=g) if per_token else torch.randn(B, device=DEV, generator=g)
    if not per_token and B > 2:
        adv[0] = 0
    mask = mask.to(mask_type)
    if mask.is_floating_point():
        mask = mask * 0.5                                   # weights count
    return logp, old, adv, mask, ref


def _check_policy(logp, old, adv, mask, ref, low=0.2, high=0.28, beta=0.1, reduction="sequence", length=None):
    from trainscale_b200.rl import clipped_policy_loss
    want, grad, stats = policy_oracle(logp, old, adv, mask, ref, low, high, beta, reduction, length or logp.shape[1])
    # an exponential is off by 2^-22, its argument (a rounded difference of a few units) by as much: 2^-21 of every term
    size = policy_oracle(logp, old, adv.abs(), mask, ref, -1e30, 1e30, 0.0, reduction, length or logp.shape[1])
    kl_size = beta * 2 * float(policy_oracle(logp, old, adv * 0, mask, ref, low, high, 1.0, reduction, length or logp.shape[1])[0]) if ref is not None else 0
    x = logp.clone().requires_grad_() if logp.is_contiguous() else logp.detach().requires_grad_()
    loss, got = clipped_policy_loss(x, old, adv, mask, ref, clip=low, clip_high=high, beta=beta, reduction=reduction, max_len=length,
                                    return_stats=True)
    assert loss.dtype == torch.float32 and loss.dim() == 0
    _near(loss, want, 2.0 ** -21 * (size[0].abs() + kl_size + want.abs()) + 1e-12)
    for u, v in zip(got, stats):
        _near(u, v, 2.0 ** -20 * v.abs() + 1e-9)
    (d,) = torch.autograd.grad(loss, x, retain_graph=True)
    assert d.dtype == logp.dtype and d.shape == logp.shape
    m = mask.double()
    d_ref = torch.where(m != 0, (ref.double() - logp.double()), 0.0).expm1().abs() if ref is not None else 0.0
    w = (size[1].abs() + beta * d_ref * m)
    tol = 2.0 ** -20 * w * 2 + HALF[logp.dtype] * grad.abs() * 1.01 + (2.0 ** -25 if logp.dtype == torch.float16 else 1e-30)
    _near(d, grad, tol)
    assert (d[mask == 0] == 0).all()
    (again,) = torch.autograd.grad(loss, x, retain_graph=True)
    assert torch.equal(d, again) and d.data_ptr() != again.data_ptr()
    # another upstream gradient: one rounding of the scaled gradient, not two
    s = torch.tensor(0.3, device=DEV)
    (scaled,) = torch.autograd.grad(loss, x, s)
    f = float(s)
    _near(scaled, grad * f, tol * f + F32 * 2 * grad.abs() * f + (2.0 ** -25 if logp.dtype == torch.float16 else 0.0))
    assert torch.equal(loss.detach(), clipped_policy_loss(x.detach(), old, adv, mask, ref, clip=low, clip_high=high, beta=beta,
                                                          reduction=reduction, max_len=length))


@pytest.mark.parametrize("reduction", ["sequence", "token", "constant"])
@pytest.mark.parametrize("B,T", [(1, 1), (2, 1), (1, 7), (3, 33), (8, 61), (1025, 5), (257, 130), (5, 4099), (2, 70001), (3000, 17)])
def test_policy_loss(B, T, reduction):
    _check_policy(*_policy_case(B, T, torch.float32, torch.bool, B + T), reduction=reduction, length=None if T % 2 else T + 3)


@pytest.mark.parametrize("mask_type", MASKS)
@pytest.mark.parametrize("dtype", list(HALF))
def test_policy_loss_types(dtype, mask_type):
    for reduction, per_token in (("sequence", True), ("token", False)):
        _check_policy(*_policy_case(9, 203, dtype, mask_type, 3, per_token), reduction=reduction)
        logp, old, adv, mask, _ = _policy_case(130, 202, dtype, mask_type, 4, per_token)
        _check_policy(logp, old, adv, mask, None, beta=0.0, reduction=reduction)


def test_policy_loss_of_inputs_that_lie_elsewhere():
    logp, old, adv, mask, ref = _policy_case(40, 70, torch.float32, torch.int64, 9, True)
    _check_policy(logp[:, 1:], old[:, :-1].clone(), adv[:, 1:], mask[:, 1:], ref[:, 1:])
    _check_policy(logp[::3, 5:50], old[::3, 5:50], adv[::3, 5:50], mask[::3, 5:50], ref[::3, 5:50])
    one = mask[1:2].expand(40, 70)
    logp, old, _, _, ref = _policy_case(40, 70, torch.float32, torch.bool, 9, spoil=False)
    _check_policy(logp, old[:1].expand(40, 70), adv[:, 0], one, ref.t().contiguous().t())
    _check_policy(logp.t(), old.t(), torch.randn(70, device=DEV, generator=_gen(1)), one.t(), ref.t(), reduction="token")
    _check_policy(logp.bfloat16(), old, adv[:, 0], one, ref.half())                # three types: computed in fp32


def test_policy_bounds_and_extremes():
    from trainscale_b200.rl import clipped_policy_loss
    up, down = math.log(1.2), math.log(0.8)
    old = torch.zeros(1, 8, device=DEV)
    f = lambda v, to: torch.nextafter(torch.tensor(v, dtype=torch.float32), torch.tensor(to, dtype=torch.float32)).item()      # noqa: E731
    logp = torch.tensor([[f(up, 9.0), f(up, -9.0), f(down, 9.0), f(down, -9.0), 100.0, 100.0, -200.0, 0.0]], device=DEV)
    for sign in (1.0, -1.0):
        adv = torch.full((1,), sign, device=DEV)
        x = logp.clone().requires_grad_()
        clipped_policy_loss(x, old, adv, torch.tensor([[1, 1, 1, 1, 0, 0, 1, 1]], device=DEV)).backward()
        _, want, _ = policy_oracle(logp, old, adv, torch.tensor([[1, 1, 1, 1, 0, 0, 1, 1]], device=DEV), None, 0.2, 0.2, 0.0, "sequence", 8)
        _near(x.grad, want, 2.0 ** -20 * want.abs() + 2.0 ** -126)      # (e^-200 is below fp32)
    zero = clipped_policy_loss(logp, old, torch.zeros(1, device=DEV), torch.ones(1, 8, device=DEV))
    assert float(zero) == 0                                 # ratios that overflow have no say without an advantage
    assert float(clipped_policy_loss(logp, old, torch.ones(1, device=DEV), torch.zeros(1, 8, device=DEV))) == 0
    for device in (DEV, "cpu"):                             # a reference that is only looked at, however far away
        x = torch.zeros(1, 4, device=device, requires_grad=True)
        far = torch.full((1, 4), 200.0, device=device)
        loss, stats = clipped_policy_loss(x, torch.zeros(1, 4, device=device), torch.ones(1, device=device), torch.ones(1, 4, device=device),
                                          far, return_stats=True)
        loss.backward()
        assert float(loss) == -1 and (x.grad == -0.25).all() and float(stats.kl) == math.inf
    bad = logp.clone()
    bad[0, 2] = math.nan
    assert clipped_policy_loss(bad, old, torch.zeros(1, device=DEV), torch.ones(1, 8, device=DEV)).isnan()


def test_group_relative_losses_keep_their_results():
    from trainscale_b200 import rl
    logp, old, adv, mask, ref = _policy_case(16, 300, torch.float32, torch.float32, 5, spoil=False)

    def pytorch(kind, x, clip_high=0.2):
        ratio = torch.exp(x - old)
        obj = torch.minimum(ratio * adv[:, None], ratio.clamp(0.8, 1 + clip_high) * adv[:, None])
        if kind == "dapo":
            return -(obj * mask).sum() / mask.sum().clamp(min=1)
        if kind == "drgrpo":
            return -((obj * mask).sum(-1) / 512).mean()
        d = ref - x
        return ((-obj + 0.01 * (torch.exp(d) - d - 1)) * mask).sum(-1).div(mask.sum(-1).clamp(min=1)).mean()

    calls = {"grpo": lambda x: rl.grpo_loss(x, old, ref, adv, mask), "drgrpo": lambda x: rl.drgrpo_loss(x, old, adv, mask, max_len=512),
             "dapo": lambda x: rl.dapo_loss(x, old, adv, mask)}
    for kind, call in calls.items():
        x, y = logp.clone().requires_grad_(), logp.clone().requires_grad_()
        a, b = call(x), pytorch(kind, y, 0.28 if kind == "dapo" else 0.2)
        assert type(a.grad_fn).__name__ == "_LossBackward"
        torch.testing.assert_close(a, b, rtol=1e-4, atol=1e-6)
        a.backward()
        b.backward()
        torch.testing.assert_close(x.grad, y.grad, rtol=1e-4, atol=1e-8)
    # gradients of other inputs, and of a gradient, as before
    o = old.clone().requires_grad_()
    rl.grpo_loss(logp.clone().requires_grad_(), o, ref, adv, mask).backward()
    assert o.grad.abs().sum() > 0
    x = logp.clone().requires_grad_()
    (d,) = torch.autograd.grad(rl.grpo_loss(x, old, ref, adv, mask), x, create_graph=True)
    (dd,) = torch.autograd.grad(d.sum(), x)
    y = logp.clone().requires_grad_()
    (e,) = torch.autograd.grad(pytorch("grpo", y), y, create_graph=True)
    torch.testing.assert_close(dd, torch.autograd.grad(e.sum(), y)[0], rtol=1e-4, atol=1e-8)
    rewards = torch.randn(16, device=DEV, generator=_gen(8))
    d = ref - logp
    kl = float(((torch.exp(d) - d - 1) * mask).sum() / mask.sum())
    for variant in ("grpo", "drgrpo", "dapo"):
        g = rl.GRPOCompute(group_size=4, beta=0.01, variant=variant)
        x = logp.clone().requires_grad_()
        loss, stats = g.compute_grpo_loss(x, ref, rewards, mask, old)
        assert set(stats) == {"reward_mean", "reward_std", "advantage_abs_mean", "kl"} and type(loss.grad_fn).__name__ == "_LossBackward"
        assert stats["kl"] == pytest.approx(kl, rel=1e-4)
        torch.testing.assert_close(loss, g(x, old, ref, rewards, mask), rtol=1e-6, atol=1e-8)
        assert "kl" not in g.compute_grpo_loss(x, None, rewards, mask, old)[1]


def test_policies_without_a_bound():
    """Infinite clip ranges and temperatures, which the kernels' own entries refuse, as on the CPU."""
    from trainscale_b200 import rl
    logp, old, adv, mask, ref = _policy_case(8, 20, torch.float32, torch.float32, 5, spoil=False)
    z, y = torch.randn(8, 50, device=DEV, generator=_gen(2)), torch.arange(8, device=DEV)
    for f, args, kw in ((rl.grpo_loss, (logp, old, ref, adv, mask), dict(clip=math.inf)), (rl.drgrpo_loss, (logp, old, adv, mask), dict(clip=math.inf)),
                        (rl.dapo_loss, (logp, old, adv, mask), dict(clip_high=math.inf)), (rl.selective_log_softmax, (z, y), dict(temperature=math.inf))):
        torch.testing.assert_close(f(*args, **kw).cpu(), f(*[t.cpu() for t in args], **kw), rtol=1e-5, atol=1e-6)


def test_masks_in_fp64_give_losses_in_fp64():
    from trainscale_b200 import rl
    logp, old, adv, mask, ref = _policy_case(8, 20, torch.float32, torch.float64, 5, spoil=False)
    for f, args in ((rl.grpo_loss, (logp, old, ref, adv, mask)), (rl.drgrpo_loss, (logp, old, adv, mask)), (rl.dapo_loss, (logp, old, adv, mask))):
        got, want = f(*args), f(*[t.cpu() for t in args])
        assert got.dtype == want.dtype == torch.float64
        torch.testing.assert_close(got.cpu(), want, rtol=1e-6, atol=1e-8)


def test_overflowing_ratios_whose_gradient_is_differentiated():
    """The PyTorch form behind a kernel's gradient keeps the kernel's zeros."""
    from trainscale_b200.rl import clipped_policy_loss
    old, mask = torch.zeros(2, 3, device=DEV), torch.ones(2, 3, device=DEV)
    x = torch.tensor([[100.0, 0.0, -0.5], [100.0, 0.0, -0.5]], device=DEV, requires_grad=True)
    adv = torch.tensor([1.0, 0.0], device=DEV)
    loss = clipped_policy_loss(x, old, adv, mask)
    (d,) = torch.autograd.grad(loss, x, retain_graph=True)
    (e,) = torch.autograd.grad(loss, x, create_graph=True)
    torch.testing.assert_close(d, e.detach(), rtol=1e-6, atol=1e-9)
    assert d.isfinite().all() and (d[1] == 0).all() and float(d[0, 0]) == 0
    (dd,) = torch.autograd.grad(e.sum(), x)
    torch.testing.assert_close(dd, e.detach(), rtol=1e-6, atol=1e-9)        # (the derivative of -a r / n is itself)


def test_an_overridden_policy_loss_is_called():
    from trainscale_b200.rl import GRPOCompute
    logp, old, _, mask, ref = _policy_case(8, 20, torch.float32, torch.float32, 5, spoil=False)

    class Own(GRPOCompute):
        def __call__(self, *args):
            return 3 * super().__call__(*args)

    rewards = torch.randn(8, device=DEV, generator=_gen(1))
    for variant in ("grpo", "drgrpo", "dapo"):
        loss, stats = GRPOCompute(4, variant=variant).compute_grpo_loss(logp, ref, rewards, mask, old)
        own, same = Own(4, variant=variant).compute_grpo_loss(logp, ref, rewards, mask, old)
        assert float(own) == pytest.approx(3 * float(loss), rel=1e-5)
        assert {k: pytest.approx(v, rel=1e-4) for k, v in stats.items()} == same


# ------------------------------------------------------------------------------------------------ pairs
def _pair_case(P, T, dtype, mask_type, seed, spoil=True):
    g = _gen(seed)
    lp = -torch.rand(2 * P, T, device=DEV, generator=g) * 3
    ref = (lp + torch.randn(2 * P, T, device=DEV, generator=g) * (2 / math.sqrt(T))).to(dtype)
    lp = lp.to(dtype)
    mask = torch.rand(2 * P, T, device=DEV, generator=g) < 0.8
    if P > 1:
        mask[1] = False
        mask[2 * P - 1] = False
    if spoil:
        lp[~mask], ref[~mask] = -math.inf, math.nan
    mask = mask.to(mask_type)
    return lp, ref, mask * 0.5 if mask.is_floating_point() else mask


def _check_pairs(lp, ref, mask, kind="sigmoid", beta=0.1, eps=0.0, gamma=0.0, normalized=False, nll=0.0):
    from trainscale_b200.rl import preference_loss
    want = preference_oracle(lp, ref, mask, beta, kind, eps, gamma, normalized, nll)
    # fp64 throughout: one rounding to fp32, and what a difference of long fp64 sums leaves
    scale = 1e-13 * float((lp.double().where(mask != 0, 0.0).abs().sum(1).max() + 1) * (1 + beta)) * (1 + float(want[0].abs().sqrt()))
    x = lp.clone().requires_grad_() if lp.is_contiguous() else lp.detach().requires_grad_()
    kw = dict(beta=beta, loss_type=kind, label_smoothing=eps, gamma=gamma, length_normalized=normalized, nll_weight=nll)
    got = preference_loss(x, ref, mask, **kw)
    for u, v in zip(got, want[:3]):
        assert u.dtype == torch.float32
        _near(u.cpu(), v, F32 * 1.01 * v.abs() + scale)
    (d,) = torch.autograd.grad(got[0], x, retain_graph=True)
    grad = want[3].to(DEV)
    tiny = scale + (2.0 ** -25 if lp.dtype == torch.float16 else 1e-30)
    _near(d, grad, HALF[lp.dtype] * 1.01 * grad.abs() + tiny)
    (again,) = torch.autograd.grad(got[0], x, torch.tensor(0.7, device=DEV))
    f = float(torch.tensor(0.7))
    _near(again, grad * f, (HALF[lp.dtype] * 1.01 + F32 * 2) * grad.abs() * f + tiny)
    assert all(torch.equal(u.detach(), v) for u, v in zip(got, preference_loss(x.detach(), ref, mask, **kw)))


@pytest.mark.parametrize("kind", ["sigmoid", "robust", "hinge", "ipo"])
@pytest.mark.parametrize("P,T", [(1, 1), (1, 2), (3, 31), (8, 2047), (300, 5), (2, 40001), (70, 1000), (1, 100003)])
def test_preference_loss(P, T, kind):
    lp, ref, mask = _pair_case(P, T, torch.float32, torch.bool, P + T)
    _check_pairs(lp, ref, mask, kind, eps=0.1)
    _check_pairs(lp, None, mask, kind, 2.0, 0.1, 0.0 if kind == "ipo" else 0.5, True, 0.3)


@pytest.mark.parametrize("mask_type", MASKS)
@pytest.mark.parametrize("dtype", list(HALF))
def test_preference_loss_types(dtype, mask_type):
    for P, T in ((5, 77), (40, 3001)):
        _check_pairs(*_pair_case(P, T, dtype, mask_type, 1), eps=0.1, nll=0.2)


def test_preference_loss_of_inputs_that_lie_elsewhere():
    lp, ref, mask = _pair_case(6, 90, torch.float32, torch.int64, 2)
    _check_pairs(lp[:, 1:], ref[:, 1:], mask[:, 1:])
    _check_pairs(lp[::2, 3:80:2], ref[::2, 3:80:2], mask[::2, 3:80:2])
    lp, ref, _ = _pair_case(6, 90, torch.float32, torch.bool, 2, spoil=False)
    _check_pairs(lp.t().contiguous().t(), ref[:1].expand(12, 90), mask[:1].expand(12, 90))
    _check_pairs(lp.half(), ref, mask)


def test_far_pairs_do_not_overflow():
    from trainscale_b200.rl import preference_loss
    for device in (DEV, "cpu"):                             # a rejected token of no probability: nothing is left to learn
        lp = torch.tensor([[-1.0, -2.0], [-math.inf, -1.0]], device=device, requires_grad=True)
        for kind in ("sigmoid", "robust", "hinge"):
            loss, chosen, rejected = preference_loss(lp, None, torch.ones(2, 2, device=device), loss_type=kind)
            (d,) = torch.autograd.grad(loss, lp)
            assert float(loss) == 0 and (d == 0).all() and float(rejected) == -math.inf
    lp = torch.tensor([[-3e4, -3e4], [0.0, 0.0]], device=DEV, requires_grad=True)
    for kind in ("sigmoid", "robust", "hinge", "ipo"):
        for order in (lp, lp.flip(0)):
            loss, _, _ = preference_loss(order, None, torch.ones(2, 2, device=DEV), beta=1.0, loss_type=kind)
            (d,) = torch.autograd.grad(loss, lp)
            assert loss.isfinite() and d.isfinite().all()


@pytest.mark.parametrize("kind,kw", [("dpo", {}), ("dpo", dict(loss_type="ipo")), ("dpo", dict(loss_type="robust", label_smoothing=0.1)),
                                     ("dpo", dict(loss_type="hinge")), ("dpo", dict(reference_free=True)), ("simpo", dict(gamma=0.4)),
                                     ("cpo", dict(alpha=0.5)), ("dpo", dict(loss_type="kto_pair")), ("orpo", {}), ("kto", {})])
def test_preference_trainer_goes_through_the_kernel(kind, kw, monkeypatch):
    """The trainer's loss, metrics and weight gradients, with the pair kernel and without it."""
    from trainscale_b200.data.synthetic import synthetic_preference_dataloader
    from trainscale_b200.models.llama import build_model
    from trainscale_b200.ops import policy
    from trainscale_b200.rl import PreferenceTrainer
    torch.manual_seed(0)
    model = build_model("tiny", dtype=torch.bfloat16, device=DEV)
    ref = PreferenceTrainer.make_reference(model)
    with torch.no_grad():
        for p in model.parameters():
            p.add_(torch.randn_like(p) * 0.01)
    batch = next(iter(synthetic_preference_dataloader(32000, 20, 40, 4)))
    batch = {k: v.to(DEV) for k, v in batch.items()}

    def run():
        t = PreferenceTrainer(model, None, ref, kind, **({} if kind == "orpo" else dict(beta=0.3)), **kw)
        model.zero_grad()
        loss, metrics = t.compute_loss(batch)
        loss.backward()
        return loss.detach(), metrics, [p.grad.float() for p in model.parameters()]

    seen = []
    one = policy.preference_loss
    monkeypatch.setattr(policy, "preference_loss", lambda *a, **k: seen.append(1) or one(*a, **k))
    a = run()
    assert bool(seen) == (kind in ("dpo", "simpo", "cpo") and kw.get("loss_type") != "kto_pair")
    monkeypatch.setattr(PreferenceTrainer, "_pair_kernel", lambda self: None)
    b = run()
    torch.testing.assert_close(a[0], b[0], rtol=1e-4, atol=1e-4)
    assert set(a[1]) == set(b[1])
    for k in a[1]:
        torch.testing.assert_close(a[1][k], b[1][k], rtol=1e-3, atol=1e-4)
    for u, v in zip(a[2], b[2]):
        assert float((u - v).norm()) <= 2e-2 * float(v.norm()) + 1e-6       # bf16 weight gradients of two fp32 roundings apart


def test_preference_trainer_calls_a_loss_of_its_users_own():
    from trainscale_b200.data.synthetic import synthetic_preference_dataloader
    from trainscale_b200.losses import DPOLoss
    from trainscale_b200.models.llama import build_model
    from trainscale_b200.rl import PreferenceTrainer
    torch.manual_seed(0)
    model = build_model("tiny", dtype=torch.bfloat16, device=DEV)
    t = PreferenceTrainer(model, None, PreferenceTrainer.make_reference(model), "dpo", 0.3)
    batch = {k: v.to(DEV) for k, v in next(iter(synthetic_preference_dataloader(32000, 20, 40, 4))).items()}
    plain = float(t.compute_loss(batch)[0].detach())

    class Twice(DPOLoss):
        def forward(self, *args):
            loss, *rest = super().forward(*args)
            return 2 * loss, *rest

    t.loss_fn = Twice(0.3)
    assert float(t.compute_loss(batch)[0].detach()) == pytest.approx(2 * plain, rel=1e-4)
    t.loss_fn, seen = DPOLoss(0.3), []
    t.loss_fn.register_forward_hook(lambda *a: seen.append(1))
    t.compute_loss(batch)
    assert seen == [1]


# ------------------------------------------------------------------------------------------------ gradient clipping
def _clip(grads, limit, kind=2.0, **kw):
    from trainscale_b200.optim import clip_grad_norm_
    ps = []
    for g in grads:
        p = torch.nn.Parameter(torch.empty(0, device=g.device, dtype=g.dtype).expand(0).new_zeros(g.shape))
        p.grad = g
        ps.append(p)
    return clip_grad_norm_(ps, limit, kind, **kw)


def _norm64(grads, kind):
    v = torch.cat([g.double().reshape(-1) for g in grads])
    return torch.linalg.vector_norm(v, kind)


@pytest.mark.parametrize("kind", [2.0, 1.0, math.inf])
@pytest.mark.parametrize("sizes,types", [([(1,)], 0), ([(3,), (5, 7), (1000, 33), (1 << 20,), (0,), (70000, 3)], 1),
                                         ([(17,)] * 1500, 1), ([(9, 11)] * 40 + [(2048, 2049)], 2)])
def test_clip_grad_norm(sizes, types, kind):
    each = {0: [torch.float32], 1: [torch.float32, torch.bfloat16, torch.float16], 2: [torch.bfloat16]}[types]
    for factor in (0.3, 2.0):
        grads = [(torch.randn(s, device=DEV, generator=_gen(i)) * 0.1).to(each[i % len(each)]) for i, s in enumerate(sizes)]
        before = [g.clone() for g in grads]
        norm = _norm64(grads, kind)
        limit = float(norm) * factor
        got = _clip(grads, limit, kind)
        _near(got, norm, F32 * 2 * norm)
        c = min(1.0, limit / (float(norm) + 1e-6))
        for g, b in zip(grads, before):
            if factor > 1:
                assert torch.equal(g, b)
            else:
                want = b.double() * c
                _near(g, want, (HALF[g.dtype] * 1.01 + 6 * F32) * want.abs() + (2.0 ** -25 if g.dtype == torch.float16 else 1e-38))


def test_clip_of_views_and_neighbours():
    """Views of one buffer at odd offsets: what lies between them stays as it is."""
    for dtype in HALF:
        flat = torch.randn(5000, device=DEV, generator=_gen(1)).to(dtype)
        before = flat.clone()
        grads = [flat[1:18], flat[19:19 + 33 * 7].view(33, 7), flat[300:300], flat[401:4000], flat[4003:4003 + 35 * 7].view(35, 7).t()]
        norm = _norm64(grads, 2.0)
        got = _clip(grads, float(norm) / 4)
        _near(got, norm, F32 * 2 * norm)
        mine = torch.zeros(5000, dtype=torch.bool, device=DEV)
        for a, b in ((1, 18), (19, 19 + 33 * 7), (401, 4000), (4003, 4003 + 35 * 7)):
            mine[a:b] = True
        assert torch.equal(flat[~mine], before[~mine])
        want = before.double()[mine] * (float(norm) / 4) / (float(norm) + 1e-6)
        _near(flat[mine], want, (HALF[dtype] * 1.01 + 6 * F32) * want.abs() + (2.0 ** -25 if dtype == torch.float16 else 0.0))


def test_clip_lists_that_go_tensor_by_tensor():
    """The same gradient twice, gradients that overlap, strided and fp64 ones, another norm: as before."""
    from trainscale_b200.optim import clip_grad_norm_
    p = torch.nn.Parameter(torch.zeros(100, device=DEV))
    p.grad = torch.ones(100, device=DEV)
    assert float(clip_grad_norm_([p, p], 1.0)) == pytest.approx(math.sqrt(200))
    assert float(p.grad[0]) == pytest.approx(1 / 200, rel=1e-4)             # scaled twice, one after the other
    flat = torch.ones(64, device=DEV)
    assert float(_clip([flat[:40], flat[24:]], 1.0)) == pytest.approx(math.sqrt(80))
    assert float(flat[30]) == pytest.approx(1 / 80, rel=1e-4) and float(flat[0]) == pytest.approx(1 / math.sqrt(80), rel=1e-4)
    g = torch.ones(10, 10, device=DEV)
    assert float(_clip([g[:, ::2]], 1.0)) == pytest.approx(math.sqrt(50)) and float(g[0, 1]) == 1
    assert float(_clip([torch.ones(4, device=DEV, dtype=torch.float64)], 1.0)) == pytest.approx(2.0)
    assert float(_clip([torch.ones(8, device=DEV)], 1.0, 3.0)) == pytest.approx(2.0, rel=1e-6)
    assert _clip([torch.ones(8, device=DEV, dtype=torch.bfloat16)], 1.0, math.inf).dtype == torch.bfloat16
    from trainscale_b200.ops.optim import GradList
    assert GradList.of([torch.ones(4, 4, device=DEV).to_sparse()], 2.0) is None
    assert GradList.of([torch.ones(4, 4, device=DEV).to_sparse_csr()], 2.0) is None
    assert GradList.of([torch.ones(4), torch.ones(4, device=DEV)], 2.0) is None
    assert GradList.of([torch.ones(4, device=DEV), torch.ones(4)], 2.0) is None
    assert GradList.of([torch.zeros(0, device=DEV)], 2.0) is None


def test_clip_of_extreme_gradients():
    one = lambda v, dtype=torch.float32: [torch.full((3000,), v, device=DEV, dtype=dtype)]          # noqa: E731
    for v in (1e30, 1e-30, 3e-42, 1e-20, 0.0):              # squares that leave the range of fp32
        g = one(v)
        norm = _norm64(g, 2.0)
        _near(_clip(g, math.inf), norm, F32 * 2 * norm + 2.0 ** -150)
    g = one(1e30)
    _clip(g, 1.0)
    assert float(g[0][0]) == pytest.approx(1 / math.sqrt(3000), rel=1e-5)
    mixed = one(1e-25) + one(1.0)
    norm = _norm64(mixed, 2.0)
    _near(_clip(mixed, math.inf), norm, F32 * 2 * norm)
    for bad in (math.nan, math.inf, -math.inf):
        for kind in (2.0, 1.0, math.inf):
            g = one(1.0)
            g[0][1234] = bad
            got = _clip(g, 1.0, kind)
            assert got.isnan() if math.isnan(bad) else float(got) == math.inf
            if math.isnan(bad):
                assert g[0].isnan().all()
            with pytest.raises(RuntimeError):
                _clip(one(1.0) + g, 1.0, kind, error_if_nonfinite=True)


def test_fused_clip_grad_norm():
    from trainscale_b200.parallel.dist_utils import fused_clip_grad_norm_
    m = torch.nn.Sequential(torch.nn.Linear(64, 65), torch.nn.Linear(65, 3)).to(DEV)
    for kind in (2.0, 1.0, math.inf):
        for p in m.parameters():
            p.grad = torch.randn(p.shape, device=DEV, generator=_gen(2))
        norm = _norm64([p.grad for p in m.parameters()], kind)
        got = fused_clip_grad_norm_(m, float(norm) / 3, norm_type=kind)
        _near(got, norm, F32 * 2 * norm)
        after = _norm64([p.grad for p in m.parameters()], kind)
        assert float(after) == pytest.approx(float(norm) / 3, rel=1e-5)


@pytest.mark.parametrize("scale", [1.0, 1e25, 1e-25])
def test_fused_clip_grad_norm_over_a_group(scale, monkeypatch):
    """The kernels' norm between two ranks that hold the same (the collective is a stand-in): powers of it stay in range."""
    import torch.distributed as dist
    from trainscale_b200.parallel.dist_utils import fused_clip_grad_norm_
    group, seen = object(), []

    def all_reduce(t, op=dist.ReduceOp.SUM, group=None):
        seen.append((t.dtype, group))
        if op == dist.ReduceOp.SUM:
            t.mul_(2)

    monkeypatch.setattr(dist, "is_initialized", lambda: True)
    monkeypatch.setattr(dist, "get_world_size", lambda group=None: 2)
    monkeypatch.setattr(dist, "all_reduce", all_reduce)
    for kind in (2.0, 1.0, math.inf):
        p = torch.nn.Parameter(torch.zeros(1000, device=DEV))
        p.grad = torch.randn(1000, device=DEV, generator=_gen(2)) * scale
        before = p.grad.double()
        norm = torch.linalg.vector_norm(torch.cat((before, before)), kind)
        got = fused_clip_grad_norm_([p], float(norm) / 3, group=group, norm_type=kind)
        _near(got, norm, F32 * 4 * norm)
        want = before * min(1.0, float(norm) / 3 / (float(norm) + 1e-6))
        _near(p.grad, want, 8 * F32 * want.abs() + 1e-38)
    assert seen == [(torch.float64, group)] * 3


def test_clip_marks_gradients_as_changed():
    x = torch.randn(50, device=DEV, requires_grad=True)
    p = torch.nn.Parameter(torch.zeros(50, device=DEV))
    g = (x * x).detach()
    p.grad = g
    y = x * g                                               # keeps g for its backward pass
    from trainscale_b200.optim import clip_grad_norm_
    clip_grad_norm_([p], 1e-3)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


# ------------------------------------------------------------------------------------------------ together
def _step(logits, labels, old, ref, adv, mask, weight, native=True):
    """Logits -> log-probabilities and entropies -> policy loss -> gradient of the head's weight -> clipping."""
    from trainscale_b200.optim import clip_grad_norm_
    from trainscale_b200.rl import clipped_policy_loss, token_log_probs
    head = torch.nn.Parameter(weight.clone())
    z = (logits @ head)[:, :-1]
    if native:
        logp, H = token_log_probs(z, labels, temperature=0.8, return_entropy=True)
        loss = clipped_policy_loss(logp, old, adv, mask, ref, beta=0.05) - 0.01 * (H * mask).sum() / mask.sum()
        loss.backward()
        norm = clip_grad_norm_([head], 0.01)
    else:
        lp = torch.log_softmax(z / 0.8, -1)
        logp, H = lp.gather(-1, labels.unsqueeze(-1)).squeeze(-1), -(lp.exp() * lp).sum(-1)
        r, d = (logp - old).exp(), ref - logp
        token = -torch.minimum(r * adv[:, None], r.clamp(0.8, 1.2) * adv[:, None]) + 0.05 * (d.exp() - 1 - d)
        loss = ((token * mask).sum(1) / mask.sum(1).clamp(min=1)).mean() - 0.01 * (H * mask).sum() / mask.sum()
        loss.backward()
        norm = head.grad.norm()
        head.grad.mul_((0.01 / (norm + 1e-6)).clamp(max=1.0))
    return loss.detach(), norm, head.grad


def _step_inputs(dtype=torch.float32):
    g = _gen(0)
    B, T, H, V = 6, 17, 32, 1003
    x = torch.randn(B, T + 1, H, device=DEV, generator=g)
    weight = torch.randn(H, V, device=DEV, generator=g) * 0.2
    labels = torch.randint(0, V, (B, T), device=DEV, generator=g)
    lp = torch.log_softmax((x @ weight)[:, :-1] / 0.8, -1).gather(-1, labels.unsqueeze(-1)).squeeze(-1)
    old = lp + 0.1 * torch.randn(B, T, device=DEV, generator=g)
    ref = lp + 0.3 * torch.randn(B, T, device=DEV, generator=g)
    mask = (torch.rand(B, T, device=DEV, generator=g) < 0.8).float()
    mask[2] = 0
    return [t.to(dtype) if t.is_floating_point() else t for t in (x, labels, old, ref, torch.randn(B, device=DEV, generator=g), mask, weight)]


def test_a_policy_step():
    a = _step_inputs()
    got = _step(*a)
    want = _step(*[t.double() if t.is_floating_point() else t for t in a], native=False)
    torch.testing.assert_close(got[0].double(), want[0], rtol=1e-5, atol=1e-6)
    torch.testing.assert_close(got[1].double(), want[1], rtol=1e-5, atol=1e-7)
    torch.testing.assert_close(got[2].double(), want[2], rtol=1e-4, atol=1e-7)


def test_a_captured_policy_step_and_another_stream():
    from trainscale_b200.ops.optim import GradList
    from trainscale_b200.rl import clipped_policy_loss, preference_loss, token_log_probs
    x, labels, old, ref, adv, mask, weight = _step_inputs()
    logits = (x @ weight)[:, :-1].contiguous()
    pairs = old.clone()

    def step(z, p):
        z, p = z.detach().requires_grad_(), p.detach().requires_grad_()
        logp, H = token_log_probs(z, labels, return_entropy=True)
        loss = clipped_policy_loss(logp, old, adv, mask, ref, beta=0.05, reduction="token") + 0.01 * H.mean()
        second, chosen, rejected = preference_loss(p, ref, mask)
        dz, dp = torch.autograd.grad((loss, second), (z, p), (torch.full((), 0.5, device=DEV), torch.ones((), device=DEV)))
        listed = GradList.of([dz, dp], 2.0)
        norm = listed.norm(2.0)
        listed.clip_(norm, 0.05)
        return loss.detach(), second.detach(), chosen, rejected, dz, dp, norm

    want = [t.clone() for t in step(logits, pairs)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            other = step(logits, pairs)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(u, v) for u, v in zip(want, other))
    z, p = torch.zeros_like(logits), torch.zeros_like(pairs)
    graphs = []
    for _ in range(2):                                      # two graphs, each with its own workspaces
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(z, p)
        graphs.append((g, out))
    z.copy_(logits)
    p.copy_(pairs)
    for _ in range(3):
        for g, _ in graphs:
            g.replay()
    torch.cuda.synchronize()
    for _, out in graphs:
        assert all(torch.equal(u, v) for u, v in zip(want, out))


def test_runs_are_the_same_bits():
    from trainscale_b200.rl import clipped_policy_loss, preference_loss, token_log_probs
    z = torch.randn(33, 50257, device=DEV, generator=_gen(1)).bfloat16()
    y = torch.randint(0, 50257, (33,), device=DEV, generator=_gen(2))
    logp, old, adv, mask, ref = _policy_case(300, 900, torch.float32, torch.bool, 5)
    lp, rf, m = _pair_case(20, 9001, torch.float32, torch.bool, 6)
    grads = [torch.randn(100000 + i, device=DEV, generator=_gen(i)) for i in range(20)]

    def run():
        x, p, q = z.clone().requires_grad_(), logp.clone().requires_grad_(), lp.clone().requires_grad_()
        a, H = token_log_probs(x, y, return_entropy=True)
        b, s = clipped_policy_loss(p, old, adv, mask, ref, beta=0.1, return_stats=True)
        c = preference_loss(q, rf, m)
        return [a, H, b, *s, *c, *torch.autograd.grad((a.sum(), H.sum(), b, c[0]), (x, p, q)), _clip([g.clone() for g in grads], 1.0)]

    first = run()
    for _ in range(3):
        assert all(torch.equal(u, v) for u, v in zip(first, run()))
