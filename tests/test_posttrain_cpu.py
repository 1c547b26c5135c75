"""Log-probabilities out of logits, policy and preference losses, gradient clipping: refusals, and the PyTorch forms that run where
the kernels do not, against definitions written apart from them in fp64."""
import math

import pytest
import torch

from posttrain_oracle import policy_oracle, preference_oracle, token_oracle
from trainscale_b200.optim import clip_grad_norm_
from trainscale_b200.rl import clipped_policy_loss, preference_loss, token_log_probs


def _gen(seed):
    return torch.Generator().manual_seed(seed)


@pytest.mark.parametrize("cap", [0.0, 5.0])
@pytest.mark.parametrize("shape", [(), (4,), (2, 3), (2, 3, 2)])
def test_token_log_probs(shape, cap):
    g = _gen(1)
    z = torch.randn(*shape, 11, generator=g, dtype=torch.float64).mul_(3)
    z.view(-1)[3] = -math.inf
    y = torch.randint(0, 11, shape, generator=g)
    if shape:
        y.view(-1)[-1] = -100
    z.requires_grad_()
    a = dict(temperature=0.7, logit_softcapping=cap, logit_scale=1.5, return_entropy=True)
    got, want = token_log_probs(z, y, **a), token_oracle(z, y, 0.7, cap, 1.5)
    for x, w in zip(got, want):
        torch.testing.assert_close(x, w, rtol=1e-12, atol=1e-12)
    up = [torch.randn(shape, generator=g, dtype=torch.float64) for _ in range(2)]
    ga, = torch.autograd.grad(got, z, up)
    gb, = torch.autograd.grad(want, z, up)
    torch.testing.assert_close(ga, gb, rtol=1e-10, atol=1e-12)


def test_a_label_outside_the_vocabulary_gives_nan():
    lp = token_log_probs(torch.zeros(3, 4), torch.tensor([4, -1, 3]))
    assert lp.isnan().tolist() == [True, True, False]
    assert float(token_log_probs(torch.zeros(1, 4), torch.tensor([-100]))) == 0
    assert float(token_log_probs(torch.zeros(1, 4), torch.tensor([-100]), ignore_index=None)) != 0


@pytest.mark.parametrize("per_token", [False, True])
@pytest.mark.parametrize("reduction", ["sequence", "token", "constant"])
def test_policy_loss(reduction, per_token):
    g = _gen(2)
    B, T = 4, 9
    logp = torch.randn(B, T, generator=g, dtype=torch.float64)
    old, ref = logp + 0.3 * torch.randn(B, T, generator=g), logp + torch.randn(B, T, generator=g)
    adv = torch.randn(B, T, generator=g) if per_token else torch.randn(B, generator=g)
    mask = (torch.rand(B, T, generator=g) < 0.6).long()
    mask[2] = 0
    logp[mask == 0], ref[mask == 0], old[mask == 0] = math.nan, math.inf, -math.inf       # what masked places hold is of no interest
    x = logp.clone().requires_grad_()
    loss, stats = clipped_policy_loss(x, old, adv, mask, ref, clip=0.2, clip_high=0.28, beta=0.1, reduction=reduction, max_len=12,
                                      return_stats=True)
    want, grad, want_stats = policy_oracle(logp, old, adv, mask, ref, 0.2, 0.28, 0.1, reduction, 12)
    torch.testing.assert_close(loss, want, rtol=1e-10, atol=1e-12)
    for a, b in zip(stats, want_stats):
        torch.testing.assert_close(a, b, rtol=1e-10, atol=1e-12)
    loss.backward()
    torch.testing.assert_close(x.grad, grad, rtol=1e-10, atol=1e-12)
    assert (x.grad[mask == 0] == 0).all()


@pytest.mark.parametrize("normalized", [False, True])
@pytest.mark.parametrize("kind", ["sigmoid", "robust", "hinge", "ipo"])
def test_preference_loss(kind, normalized):
    g = _gen(3)
    P, T = 5, 8
    lp = torch.randn(2 * P, T, generator=g, dtype=torch.float64)
    ref = lp + torch.randn(2 * P, T, generator=g)
    mask = torch.rand(2 * P, T, generator=g) < 0.7
    mask[P + 1] = False
    lp[~mask], ref[~mask] = math.nan, math.inf
    a = (0.8, kind, 0.1, 0.0 if kind == "ipo" else 0.3, normalized, 0.2)
    x = lp.clone().requires_grad_()
    got = preference_loss(x, ref, mask, beta=a[0], loss_type=kind, label_smoothing=a[2], gamma=a[3], length_normalized=normalized,
                          nll_weight=a[5])
    want = preference_oracle(lp, ref, mask, *a)
    for u, v in zip(got, want[:3]):
        torch.testing.assert_close(u, v, rtol=1e-10, atol=1e-12)
    got[0].backward()
    torch.testing.assert_close(x.grad, want[3], rtol=1e-10, atol=1e-12)


def test_label_smoothing_counts_where_there_is_a_smoothed_form():
    lp, mask = torch.randn(6, 4, generator=_gen(7)), torch.ones(6, 4)
    for kind, counts in (("sigmoid", True), ("robust", True), ("hinge", False), ("ipo", False)):
        a, b = (preference_loss(lp, None, mask, beta=0.5, loss_type=kind, label_smoothing=e)[0] for e in (0.0, 0.2))
        assert bool(a != b) == counts


def test_gradients_against_differences():
    g = _gen(4)
    z, y = torch.randn(3, 5, generator=g, dtype=torch.float64, requires_grad=True), torch.tensor([0, 4, -100])
    f = lambda z: token_log_probs(z, y, temperature=0.5, logit_softcapping=3.0, return_entropy=True)       # noqa: E731
    assert torch.autograd.gradcheck(f, (z,)) and torch.autograd.gradgradcheck(f, (z,))
    lp = torch.randn(4, 5, generator=g, dtype=torch.float64, requires_grad=True)
    old, adv, mask = lp.detach() + 0.05, torch.randn(4, generator=g), torch.ones(4, 5)
    assert torch.autograd.gradcheck(lambda p: clipped_policy_loss(p, old, adv, mask, old - 0.3, beta=0.3), (lp,))
    assert torch.autograd.gradcheck(lambda p: preference_loss(p, old, mask, loss_type="ipo")[0], (lp,))


def test_nothing_to_learn_from():
    empty = torch.zeros(0, 4, requires_grad=True)
    loss = clipped_policy_loss(empty, empty.detach(), torch.zeros(0), empty.detach())
    loss.backward()
    assert float(loss) == 0 and empty.grad.shape == (0, 4)
    assert float(clipped_policy_loss(torch.zeros(3, 0), torch.zeros(3, 0), torch.zeros(3), torch.zeros(3, 0))) == 0
    assert float(preference_loss(torch.zeros(0, 4), None, torch.zeros(0, 4))[0]) == 0
    assert float(preference_loss(torch.zeros(2, 0), None, torch.zeros(2, 0))[0]) == pytest.approx(math.log(2))
    assert token_log_probs(torch.zeros(0, 4), torch.zeros(0, dtype=torch.long)).shape == (0,)


def test_refusals():
    z, y = torch.zeros(2, 3, 5), torch.zeros(2, 3, dtype=torch.long)
    for kw in (dict(temperature=0.0), dict(temperature=math.inf), dict(temperature=-1.0), dict(logit_softcapping=-1.0),
               dict(logit_scale=-2.0), dict(logit_softcapping=math.nan), dict(temperature=1e-35), dict(logit_scale=1e20, logit_softcapping=1e15)):
        with pytest.raises(ValueError):
            token_log_probs(z, y, **kw)
    with pytest.raises(ValueError):
        token_log_probs(z, y[:, :2])
    with pytest.raises(ValueError):
        token_log_probs(torch.zeros(2, 0), torch.zeros(2, dtype=torch.long))
    with pytest.raises(TypeError):
        token_log_probs(z, y.float())
    with pytest.raises(TypeError):
        token_log_probs(z.long(), y)
    p, a, m = torch.zeros(2, 3), torch.zeros(2), torch.ones(2, 3)
    for args, kw in (((p, p, a, m), dict(reduction="mean")), ((p, p, a, m), dict(beta=0.1)), ((p, p, a, m), dict(clip=-0.1)),
                     ((p, p, a, m), dict(clip_high=math.nan)), ((p, p, a, m), dict(max_len=0)), ((p, p, a, m), dict(beta=math.inf)),
                     ((p[0], p[0], a, m[0]), {}), ((p, p[:, :2], a, m), {}), ((p, p, torch.zeros(3), m), {}), ((p, p, a, m[:1]), {}),
                     ((p, p, a, m, p[:1]), {})):
        with pytest.raises(ValueError):
            clipped_policy_loss(*args, **kw)
    for args, kw in (((p, None, m), dict(loss_type="dpo")), ((p, None, m), dict(beta=0.0)), ((p, None, m), dict(beta=math.nan)),
                     ((p, None, m), dict(label_smoothing=1.5)), ((p, None, m), dict(loss_type="robust", label_smoothing=0.5)),
                     ((p, None, m), dict(loss_type="ipo", gamma=0.1)), ((p, None, m), dict(nll_weight=math.inf)),
                     ((torch.zeros(3, 2), None, torch.zeros(3, 2)), {}), ((p, p[:1], m), {}), ((p, None, m[:, :1]), {}),
                     ((p[0], None, m[0]), {})):
        with pytest.raises(ValueError):
            preference_loss(*args, **kw)


def test_clipping_on_the_cpu_is_as_before():
    ps = [torch.nn.Parameter(torch.zeros(3)), torch.nn.Parameter(torch.zeros(2, 2))]
    for p in ps:
        p.grad = torch.full_like(p, 2.0)
    assert float(clip_grad_norm_(ps, 1.0)) == pytest.approx(math.sqrt(28))
    assert float(ps[0].grad[0]) == pytest.approx(2 / math.sqrt(28), rel=1e-5)
    assert float(clip_grad_norm_([torch.nn.Parameter(torch.zeros(1))], 1.0)) == 0


def test_labels_of_the_fused_head():
    """What the row kernels read: dense int64 labels, one for every row at least, where the rows are."""
    from trainscale_b200.ops.cross_entropy import _dense_labels
    ids = torch.arange(8).view(4, 2)
    cpu = torch.device("cpu")
    for labels in (ids[:, 1:], ids[:, 1], ids[:, 1].int(), ids[:, 1:].unsqueeze(0)):
        got = _dense_labels(labels, 4, cpu)
        assert got.is_contiguous() and got.dtype == torch.int64 and got.tolist() == [1, 3, 5, 7]
    same = torch.arange(4)
    assert _dense_labels(same, 4, cpu).data_ptr() == same.data_ptr()
    for labels, device in ((torch.arange(3), cpu), (torch.arange(4, device="meta"), cpu)):
        with pytest.raises(ValueError, match="labels"):
            _dense_labels(labels, 4, device)


def test_operations_that_are_recorded_or_transformed():
    """Where a kernel called by address would leave nothing behind: traces, modes, transforms, compiled functions."""
    from torch.fx.experimental.proxy_tensor import make_fx
    from torch.utils.flop_counter import FlopCounterMode
    from trainscale_b200.ops import _lib
    seen, x = [], torch.ones(3)

    def f(x):
        seen.append(_lib.eager())
        return x + 1

    assert f(x) is not None and seen.pop()
    torch.jit.trace(f, x, check_trace=False)
    make_fx(f)(x)
    make_fx(f, tracing_mode="fake")(x)
    torch.func.vmap(f)(x)
    torch.func.grad(lambda x: f(x).sum())(x)
    torch.func.jvp(f, (x,), (x,))
    with FlopCounterMode(display=False):
        f(x)
    assert seen == [False] * 7
    g = torch.compile(lambda x: x + (1 if _lib.eager() else 2), backend="eager", fullgraph=True)
    assert torch.equal(g(x), x + 2) and _lib.eager()


def test_preference_trainer_asks_the_loss_that_it_holds():
    """The pair kernel stands for the losses that the trainer makes itself, and for nothing that a user put in their place."""
    from trainscale_b200 import rl
    from trainscale_b200.losses import CPOLoss, DPOLoss, SimPOLoss

    def trainer(kind, **kw):
        return rl.PreferenceTrainer(None, None, None, kind, **kw)

    assert trainer("dpo")._pair_kernel() == dict(loss_type="sigmoid", label_smoothing=0.0, beta=0.1)
    assert trainer("simpo", gamma=0.4)._pair_kernel() == dict(label_smoothing=0.0, gamma=0.4, length_normalized=True, beta=0.1)
    assert trainer("cpo", alpha=0.5)._pair_kernel() == dict(label_smoothing=0.0, nll_weight=0.5, beta=0.1)
    for kind, base in (("dpo", DPOLoss), ("simpo", SimPOLoss), ("cpo", CPOLoss)):
        class Own(base):
            def forward(self, *args):
                return super().forward(*args)

        for change in (lambda t: setattr(t, "loss_fn", Own()), lambda t: setattr(t, "loss_fn", torch.nn.MSELoss()),
                       lambda t: t.loss_fn.register_forward_hook(lambda *a: None),
                       lambda t: t.loss_fn.register_forward_pre_hook(lambda *a: None),
                       lambda t: t.loss_fn.register_full_backward_hook(lambda *a: None),
                       lambda t: setattr(t.loss_fn, "forward", lambda *a: None),
                       lambda t: setattr(t.loss_fn, "beta", torch.nn.Parameter(torch.tensor(0.1))),
                       lambda t: setattr(t.loss_fn, "beta", math.inf)):
            t = trainer(kind)
            assert t._pair_kernel() is not None
            change(t)
            assert t._pair_kernel() is None
        t = trainer(kind)
        handle = torch.nn.modules.module.register_module_forward_hook(lambda *a: None)
        try:
            assert t._pair_kernel() is None
        finally:
            handle.remove()
    t = trainer("dpo")
    t.loss_fn = lambda *a: None                             # no module at all
    assert t._pair_kernel() is None


def test_preference_trainer_keeps_an_overridden_sum():
    """A trainer that makes its sequences' log-probabilities in its own way is asked for them, of the policy too."""
    from trainscale_b200 import rl
    asked = []

    class Own(rl.PreferenceTrainer):
        def _seq_logps(self, model, ids, mask, labels, grad):
            asked.append(model)
            return torch.full((4,), -1.0, requires_grad=grad), torch.full((4,), 3)

    batch = {f"{side}_{k}": torch.ones(2, 3, dtype=torch.long) for side in ("chosen", "rejected")
             for k in ("input_ids", "attention_mask", "labels")}
    for kind in ("dpo", "simpo", "cpo", "orpo"):
        t = Own(torch.nn.Linear(1, 1), None, None, kind)
        assert not t._sums_plainly() and t.compute_loss(batch)[0].isfinite()
        assert asked.pop() is t.policy and not asked
    t = rl.PreferenceTrainer(None, None, None, "dpo")
    assert t._sums_plainly()


def test_calls_that_the_kernels_entries_would_refuse_keep_the_pytorch_form(monkeypatch):
    """No bound on a ratio, an infinite temperature, numbers that are tensors: the dispatch leaves them where they were."""
    from trainscale_b200 import rl
    g = _gen(6)
    logp = torch.randn(4, 5, generator=g)
    old, ref, adv, mask = logp + 0.5 * torch.randn(4, 5, generator=g), logp + 0.1, torch.randn(4, generator=g), torch.ones(4, 5)
    z, y = torch.randn(4, 9, generator=g), torch.arange(4)
    inf, nan, one = math.inf, math.nan, torch.tensor(0.2)
    rewards = torch.randn(4, generator=g)

    def group(**kw):
        return rl.GRPOCompute(2, **kw).compute_grpo_loss(logp, ref, rewards, mask, old)[0]

    calls = [lambda: rl.grpo_loss(logp, old, ref, adv, mask, clip=inf), lambda: rl.grpo_loss(logp, old, ref, adv, mask, beta=inf),
             lambda: rl.grpo_loss(logp, old, ref, adv, mask, clip=one), lambda: rl.drgrpo_loss(logp, old, adv, mask, clip=inf),
             lambda: rl.drgrpo_loss(logp, old, adv, mask, max_len=torch.tensor(7.0)), lambda: rl.dapo_loss(logp, old, adv, mask, clip_high=inf),
             lambda: rl.dapo_loss(logp, old, adv, mask, clip_low=inf), lambda: group(clip=inf), lambda: group(clip=nan),
             lambda: group(clip=inf, variant="dapo"), lambda: rl.selective_log_softmax(z, y, inf),
             lambda: rl.selective_log_softmax(z, y, 1e-35), lambda: rl.selective_log_softmax(z, y, 1.0, inf),
             lambda: rl.selective_log_softmax(z, y, 1.0, 30.0, 1e35), lambda: rl.selective_log_softmax(z, y, torch.tensor(0.7)),
             lambda: rl.selective_log_softmax(z, y, 1.0, torch.tensor(5.0))]
    want = [call() for call in calls]
    asked = []
    monkeypatch.setattr(rl.policy_ops, "native", lambda *t: True)
    monkeypatch.setattr(rl.lp_ops, "native", lambda *t: True)
    monkeypatch.setattr(rl, "clipped_policy_loss", lambda *a, **k: asked.append(1))
    monkeypatch.setattr(rl, "token_log_probs", lambda *a, **k: asked.append(1))
    for call, w in zip(calls, want):
        torch.testing.assert_close(call(), w, rtol=0, atol=0, equal_nan=True)
    assert not asked
    rl.grpo_loss(logp, old, ref, adv, mask)
    rl.drgrpo_loss(logp, old, adv, mask, max_len=7)
    rl.dapo_loss(logp, old, adv, mask)
    rl.selective_log_softmax(z, y, 0.7, None, 1.5)
    assert len(asked) == 4


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
def test_ratios_that_overflow(dtype):
    """A clipped ratio, and one without an advantage, have no say: neither in the loss nor in its derivatives, however large."""
    far = 100.0 if dtype == torch.float32 else 800.0
    old, mask = torch.zeros(1, 3, dtype=dtype), torch.ones(1, 3)
    for adv, want, slope in ((1.0, -(1.2 + 1.0 + 0.5) / 3, [0.0, -1 / 3, -0.5 / 3]), (0.0, 0.0, [0.0, 0.0, 0.0])):
        x = torch.tensor([[far, 0.0, math.log(0.5)]], dtype=dtype, requires_grad=True)
        loss, stats = clipped_policy_loss(x, old, torch.tensor([adv]), mask, return_stats=True)
        (d,) = torch.autograd.grad(loss, x, create_graph=True)
        (dd,) = torch.autograd.grad(d.sum(), x)
        assert float(loss) == pytest.approx(want, rel=1e-6) and d[0].tolist() == pytest.approx(slope, rel=1e-6) and dd.isfinite().all()
        assert float(stats.ratio) == math.inf and float(stats.clip_fraction) == pytest.approx(1 / 3 if adv else 0.0)
    x = torch.tensor([[-far, 0.0, 0.0]], dtype=dtype, requires_grad=True)
    loss = clipped_policy_loss(x, old, torch.tensor([-1.0]), mask)
    assert float(loss) == pytest.approx((0.8 + 2) / 3, rel=1e-6)
    assert torch.autograd.grad(loss, x)[0][0].tolist() == pytest.approx([0.0, 1 / 3, 1 / 3], rel=1e-6)
    x = torch.tensor([[far, 0.0, 0.0]], dtype=dtype, requires_grad=True)      # one that counts does overflow
    loss = clipped_policy_loss(x, old, torch.tensor([-1.0]), mask)
    assert float(loss) == math.inf and float(torch.autograd.grad(loss, x)[0][0, 0]) == math.inf
    assert clipped_policy_loss(torch.full((1, 3), math.nan, dtype=dtype), old, torch.zeros(1), mask).isnan()


def test_tokens_at_a_clip_bound():
    """A difference that fp32 rounds onto the bound, or past it, is on the side where it lies."""
    from fractions import Fraction
    x = torch.tensor([[-1.0, -1.0, -1.0, -1.0]])
    up, down = math.log1p(0.2), math.log1p(-0.2)
    f32 = lambda v: torch.tensor(v, dtype=torch.float32)                               # noqa: E731
    old = torch.stack([f32(-1.0 - up), torch.nextafter(f32(-1.0 - up), f32(0.0)), f32(-1.0 - down), torch.nextafter(f32(-1.0 - down), f32(-2.0))])
    moved = [Fraction(-1) - Fraction(float(o)) for o in old]
    above, below = [v > Fraction(up) for v in moved], [v < Fraction(down) for v in moved]
    for sign, want in ((1.0, above), (-1.0, below)):
        p = x.clone().requires_grad_()
        clipped_policy_loss(p, old.unsqueeze(0), torch.tensor([sign]), torch.ones(1, 4)).backward()
        assert [float(d) == 0 for d in p.grad[0]] == want


@pytest.mark.parametrize("listed,port", [("", 29781), ("0,1", 29782), ("1", 29783)])
def test_a_norm_over_ranks(listed, port):
    """Two ranks, tensor by tensor, through the kernels' list (a stand-in), and one of each."""
    import subprocess
    import sys
    from pathlib import Path
    case = Path(__file__).parent / "dist_cases" / "clip_norm.py"
    r = subprocess.run([sys.executable, "-m", "torch.distributed.run", "--nnodes=1", "--nproc-per-node=2", "--master-addr", "127.0.0.1",
                        "--master-port", str(port), str(case), f"--listed={listed}"], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-2000:]
    assert r.stdout.count("ok=True") == 2


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64, torch.bfloat16])
def test_rows_without_a_distribution(dtype):
    """What a logit of +inf, a row of -inf and a NaN leave, as the kernel has it."""
    z = torch.zeros(5, 7, dtype=dtype)
    z[0], z[1, 6], z[2, 3], z[3, 3] = -math.inf, math.nan, math.inf, math.inf
    lp, H = token_log_probs(z, torch.tensor([0, 0, 0, 3, 0]), return_entropy=True)
    assert lp[:2].isnan().all() and float(lp[2]) == -math.inf and lp[3].isnan() and lp[4].isfinite() and H[:4].isnan().all()
    lp = token_log_probs(z, torch.tensor([-100, -100, 7, -1, 5]))
    assert (lp[:2] == 0).all() and lp[2:4].isnan().all()
