"""Values at the edge of the learning operators' definitions: what has to stay finite, and what must not become finite."""

import importlib
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def learn():
    return importlib.import_module("katago-rs_amd.learn")


@pytest.mark.parametrize("v", [3, 362, 20001])
def test_no_advantage_no_part(learn, v):
    """An advantage of 0 takes no part, also where the ratio passes float's range (e^90 and more): only the KL term is left."""
    n = 5
    g = torch.Generator().manual_seed(v)
    z, refl = torch.randn(n, v, generator=g).cuda(), torch.randn(n, v, generator=g).cuda()
    act = torch.arange(n, dtype=torch.int32, device="cuda") % v
    old = torch.tensor([-1e2, -2e2, -1e4, -1e30, -math.inf], device="cuda")
    zero, near = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
    got = learn.policy_loss(z, act, old, zero, kl_coef=0.5, ref_logits=refl)
    want = learn.policy_loss(z, act, near, zero, kl_coef=0.5, ref_logits=refl)
    assert torch.equal(got.loss, want.loss) and torch.equal(got.grad, want.grad) and torch.isfinite(got.grad).all()
    # With one: clipped from above, and never where it is negative.
    up = learn.policy_loss(z, act, old, near + 2.0, clip=(0.2, 0.25))
    assert torch.equal(up.loss, torch.full_like(up.loss, -2.5)) and not up.grad.any()
    assert torch.all(learn.policy_loss(z, act, old, near - 2.0).loss == math.inf)
    # NaN is not hidden by it.
    z[:, 0] = torch.nan
    r = learn.policy_loss(z, act, old, zero)
    assert torch.isnan(r.loss).all() and torch.isnan(r.grad).all()
    assert torch.isnan(learn.policy_loss(refl, act, old, zero * torch.nan).grad).all()


@pytest.mark.parametrize("shape", [(2, 37, 24, 3), (2, 5000, 96, 4), (2, 9, 2056, 8), (1, 901, 3, 3)])
@pytest.mark.parametrize("act", ["identity", "relu", "mish", "silu"])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_no_number_is_seen(learn, shape, act, bad):
    """A value that is no finite number at a point that counts makes its group's results NaN, in y and dx too, and no other's."""
    b, p, c, groups = shape
    g = torch.Generator().manual_seed(p)
    x, dy = torch.randn(b, p, c, generator=g).cuda(), torch.randn(b, p, c, generator=g).cuda()
    x[0, p // 2, c - 1] = bad
    y, mean, rstd = learn.group_norm(x, groups, act=act)
    dx, dgamma, _ = learn.group_norm_backward(dy, x, mean, rstd, groups, act=act)
    w = c // groups
    for t in (y, dx):
        assert torch.isnan(t[0, :, c - w:]).all() and torch.isfinite(t[0, :, :c - w]).all() and torch.isfinite(t[1:]).all()
    assert torch.isnan(rstd[0, -1]) and torch.isfinite(rstd[0, :-1]).all() and torch.isfinite(rstd[1:]).all()
    assert torch.isnan(dgamma[c - w:]).all() and torch.isfinite(dgamma[:c - w]).all()
