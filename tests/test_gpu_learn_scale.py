"""The policy loss at any temperature, on every kernel that it has: rows shorter than 16 bytes, held rows, streamed ones and rows cut
into parts. log2 e times the scale is taken in two floats, and -infinity (an illegal column, a place past the row's end) has to
come out as 0 whatever those are: scales whose nearest float lies below the product, above it and on it.

Bounds are those of test_gpu_learn_losses.py (K U relative for a probability, K U absolute for logp) but for the gradient's. Its factor
is c = -ratio adv + kl_coef (1 - e^d), d = ref_logp - logp: logp's error K U is a relative one of ratio and of e^d, so c is off by
K U (ratio |adv| + |kl_coef| (1 + e^d)), the terms as they are before they cancel (in one row of 362 columns here they leave a
125th), and the gradient by that times w s (onehot + p). The hardware's exponential gives 0 for what lies below 2^-126 (at a scale of 10
a row's least probabilities do): gradient j = w s (c (onehot - p_j) + kl_coef p_j (d_j - kl)) is off by up to 2^-126 times the
factor of its p_j."""

import ctypes
import importlib
import math

import numpy as np
import pytest
import torch

import learn_abi as abi
import learn_ref as ref
from test_gpu_learn_losses import _close, _inputs, _k

LOG2E = 1.44269504088896340736
BELOW, ABOVE, ON = [0.7, 1.9, 2.0, 1 / 64], [0.8, 0.9, 1 / 0.7, 1 / 3, 10.0], [1.4000163254418458, 0.284626006026787]


@pytest.fixture(scope="module")
def learn():
    return importlib.import_module("katago-rs_amd.learn")


def _case(learn, n, v, dtype, kl, legal, seed, scale, edit=None, kl_coef=0.3, clip=(0.2, 0.3), ld=None):
    g, full = _inputs(n, v, dtype, seed, ld)
    z = full[:, :v]
    actions = torch.randint(0, v, (n,), generator=g, dtype=torch.int32)
    mask = None
    if legal:
        mask = torch.rand(n, v, generator=g) < 0.6
        mask.scatter_(1, actions[:, None].long(), True)
    refl = (z.float() + 0.4 * torch.randn(n, v, generator=g)).to(dtype) if kl == "full" else None
    adv, weight = torch.randn(n, generator=g), torch.rand(n, generator=g)
    rows = torch.arange(n)
    lp = ref.log_softmax(z.double() * scale, mask)[rows, actions.long()]
    old = (lp + 0.25 * torch.randn(n, generator=g)).float()
    rlp = (lp + 0.5 * torch.randn(n, generator=g)).float() if kl == "estimate" else None
    if edit:
        edit(z, actions, mask, refl)
    lsm = ref.log_softmax(z.double() * scale, mask)
    lp = lsm[rows, actions.long().clamp(0, v - 1)]
    for border in (math.log(1 - clip[0]), math.log(1 + clip[1])):
        assert not ((lp - old.double() - border).abs() < 1e-5).any()
    loss, logp, klw, gw, size = ref.policy(z, actions, old, adv, mask, weight, scale, clip, kl_coef, refl, rlp)
    dev = lambda t: None if t is None else t.cuda()  # noqa: E731
    got = learn.policy_loss(full.cuda()[:, :v], dev(actions), dev(old), dev(adv), legal=dev(mask), weight=dev(weight),
                            logit_scale=scale, clip=clip, kl_coef=kl_coef, ref_logits=dev(refl), ref_logp=dev(rlp))
    k = _k(z, scale, v, mask) + (_k(refl, scale, v, mask) if kl == "full" else 0)
    factor = lambda d: torch.exp(d.clamp(-50, 50)).nan_to_num(0, 0, 0)  # noqa: E731
    ratio, ed = factor(logp - old.double()), torch.zeros(n, dtype=torch.float64) if rlp is None else factor(rlp.double() - logp)
    _close(got.logp, logp, torch.ones(n), k, "logp")
    ksize = (klw.abs() + 2) * 2 if kl != "estimate" else ed + 10
    _close(got.kl, klw, ksize, k, "kl")
    _close(got.loss, loss, weight * (ratio * adv.abs() + kl_coef * ksize), k, "loss")
    if rlp is not None:
        hot = torch.zeros(n, v, dtype=torch.float64)
        hot[rows, actions.long().clamp(0, v - 1)] = 1
        size = (scale * weight * (ratio * adv.abs() + kl_coef * (1 + ed)))[:, None] * (hot + torch.exp(lsm).nan_to_num(0, 0, 0))
    c = ratio * adv.abs() + (kl_coef * (1 + ed) if rlp is not None else 0)
    gap = torch.zeros(n, v, dtype=torch.float64) if refl is None else \
        kl_coef * ((lsm - ref.log_softmax(refl.double() * scale, mask)).abs().nan_to_num(0, 0, 0) + klw.abs()[:, None])
    lost = 2.0 ** -126 * (scale * weight)[:, None] * (c[:, None] + gap)
    _close(got.grad, gw, size + lost / (k * ref.U), k, "grad")
    return got


def _side(scale):
    """Of the nearest float to scale log2 e: 1 below it, -1 above, 0 on it."""
    return (scale * LOG2E > float(np.float32(scale * LOG2E))) - (scale * LOG2E < float(np.float32(scale * LOG2E)))


def test_the_scales_lie_on_all_sides():
    for sign, scales in ((1, BELOW), (-1, ABOVE), (0, ON)):
        assert [_side(s) for s in scales] == [sign] * len(scales)


@pytest.mark.parametrize("scale,refused", [(2.0 ** -64, False), (2.0 ** 64, False), (2.0 ** -64.1, True), (2.0 ** 64.1, True),
                                           (1e-320, True), (1e300, True), (math.inf, True), (-1.0, True)])
def test_scales_outside_the_range_are_refused(kgx, scale, refused):
    args = abi.PolicyArgs(rows=0, columns=9, logit_scale=scale)
    assert kgx.lib().kg_policy_loss(0, None, ctypes.byref(args)) == refused
    assert not refused or "logit_scale" in kgx.lib().kg_last_error().decode()


@pytest.mark.gpu
@pytest.mark.parametrize("scale", BELOW + ABOVE + ON)
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_policy_loss_at_any_scale(learn, scale, dtype):
    for v, rows in ((1, 3), (3, 5), (7, 5), (362, 5), (2500, 4), (16300, 2), (20001, 2), (70001, 2)):
        for kl in ("none", "estimate", "full"):
            for legal in (False, True):
                _case(learn, rows, v, dtype, kl, legal, 11 * v + rows, scale, ld=v + 1)


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [0.7, 0.8, 1 / 0.7, ON[0]])
def test_policy_loss_of_many_long_rows_at_any_scale(learn, scale):
    for v, dtype, kl, legal in ((20001, torch.float32, "full", True), (41001, torch.float32, "none", False),
                                (33001, torch.bfloat16, "estimate", True)):
        _case(learn, 385, v, dtype, kl, legal, v, scale)


@pytest.mark.gpu
def test_policy_loss_masked_values_at_any_scale(learn):
    """Columns of -infinity and of the lowest value, rows without a legal column, padding; NaN stays in its row."""
    for scale in (0.7, 0.8, ON[0]):
        for v in (7, 362, 20001):
            def edit(z, actions, legal, refl):
                actions[0] = -1
                legal[1] = False
                z[2, torch.arange(v) != actions[2]] = -torch.inf
                refl[2] = 0
                z[3, torch.arange(v) != actions[3]] = torch.finfo(torch.float32).min
                refl[3] = 0
                z[4, ~legal[4]] = torch.nan
                refl[4, ~legal[4]] = -torch.inf
            got = _case(learn, 6, v, torch.float32, "full", True, v + 1, scale, edit)
            assert float(got.logp[0]) == 0 and float(got.logp[1]) == -math.inf and abs(float(got.logp[2])) == 0
        z = torch.randn(2, 362, device="cuda")
        z[1, 40] = torch.nan
        f = torch.full((2,), -6.0, device="cuda")
        r = learn.policy_loss(z, torch.zeros(2, dtype=torch.int32, device="cuda"), f, f, logit_scale=scale)
        assert torch.isfinite(r.grad[0]).all() and torch.isnan(r.grad[1]).all() and torch.isnan(r.logp).tolist() == [False, True]


@pytest.mark.gpu
def test_policy_loss_at_the_least_scale(learn):
    """All legal columns are as likely."""
    for v in (3, 362, 20001):
        got = _case(learn, 4, v, torch.float32, "full", True, v + 2, 2.0 ** -64)
        assert torch.all(got.kl.abs() <= 1e-6)
