"""Group norm's statistics where the first value that a thread meets lies far from the rest, on rows that go through the simple
kernels (channels fewer than a 16-byte column's, groups wider than a share's workgroup joins), in which a thread takes hundreds of points.

Bounds. One value of a group lies P = 10^4 above the others (standard normal), so it makes nearly all of the squared deviations M2, P^2. Its
thread takes 16 points at a time relative to its mean so far, s1 and s2 their sum and sum of squares, and adds s2 - s1^2 / n. In the
first such piece 15 values lie P below the first: s2 = 15 P^2 within 18 U, s1^2 / 16 = 14.1 P^2 within 35 U, together 770 U P^2. In the q-th
the mean is P / 16 q, so s2 = P^2 / 16 q^2 and all of them together add 6 U P^2. M2's own additions are a rounding each 16 points,
50 U here, and the joins 100 U: 1000 U of M2, and half of that of rstd. The mean of that thread takes 16 (16 + 2) U P from the first
piece's sum and less than as much from all others, divided by its points; with the other threads' (a few U of means below 1, and the joins' 100 U
of the sum of all sizes) the group's mean is off by at most 1000 U P / N + 100 U."""

import importlib

import pytest
import torch

import learn_ref as ref

pytestmark = pytest.mark.gpu
U, P = ref.U, 1e4


@pytest.fixture(scope="module")
def learn():
    return importlib.import_module("katago-rs_amd.learn")


@pytest.mark.parametrize("batch,points,channels", [(2048, 200000, 1), (300, 3500, 1100)])
@pytest.mark.parametrize("masked", [False, True])
def test_a_far_first_value(learn, batch, points, channels, masked):
    g = torch.Generator(device="cuda").manual_seed(points)
    x = torch.randn(batch, points, channels, generator=g, device="cuda")
    mask, first = None, 0
    if masked:
        mask = (torch.rand(batch, points, generator=g, device="cuda") < 0.7).float()
        mask[:, :3] = torch.tensor([0.0, 1.0, 1.0], device="cuda")
        x[:, 0] = torch.nan
        first = 1
    x[:, first, channels // 2] += P
    y, mean, rstd = learn.group_norm(x, 1, mask=mask)
    rows = [0, 1, batch // 2, batch - 1]
    _, wm, wr = ref.group_norm(x[rows].cpu(), 1, mask=None if mask is None else mask[rows].cpu())
    count = points * channels if mask is None else mask[rows].sum(1).cpu().double()[:, None] * channels
    assert ((rstd[rows].cpu().double() - wr).abs() <= 520 * U * wr).all()
    assert ((mean[rows].cpu().double() - wm).abs() <= 1000 * U * P / count + 100 * U).all()
    assert torch.isfinite(y[rows]).all()
