"""Layer norm and RMS norm on the GPU against their definitions in float64 (tests/student_ref.py).

Bounds. A row's sums are float over a thread's share (at most C / 64 + 8 values one after another) and a tree: G U = (C / 64 + 24)
U of the sum of the terms' sizes. The mean is corrected by the deviations' own mean, so it is off by its rounding and G U of the
mean deviation; the variance by (G + 4) U relative, rstd by half of that and its rounding. h = (x - mean) rstd takes both.
Backward, for the given statistics: h is off by 3 U, d by U, the row's two means by (G + 4) U of their terms' sizes. Sums over
N rows: N / 64 + 40 additions in float at most, then double. A result's rounding to its type comes on top."""

import importlib
import math

import pytest
import torch

import learn_ref
import student_ref as ref
from test_gpu_distill import close

pytestmark = pytest.mark.gpu
U = learn_ref.U
TYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.fixture(scope="module")
def learn():
    return importlib.import_module("katago-rs_amd.learn")


def make(n, c, dtype, seed, shift=1.0, params=True, ld=0):
    g = torch.Generator().manual_seed(seed)
    full = ((torch.randn(n, c + ld, generator=g) * (0.5 + torch.rand(c + ld, generator=g)) + shift) * (0.5 + torch.rand(n, 1, generator=g))).to(dtype)
    dy = torch.randn(n, c + ld, generator=g).to(dtype)
    gamma, beta = (1 + 0.3 * torch.randn(c, generator=g), torch.randn(c, generator=g)) if params else (None, None)
    return full, dy, gamma, beta


def forward(learn, full, gamma, beta, at, c, rms, eps=1e-5, **more):
    x = full.cuda()[:, at:at + c]
    dev = lambda t: None if t is None else t.cuda()  # noqa: E731
    y, mean, rstd = learn.layer_norm(x, dev(gamma), dev(beta), eps=eps, rms=rms, **more)
    x = full[:, at:at + c]
    want, wmean, wrstd, h = ref.layer_norm(x, gamma, beta, eps, rms)
    g = c / 64 + 24
    spread = (x.double() - wmean[:, None]).abs().mean(1)
    if rms:
        assert mean is None
    else:
        close(mean, wmean, spread, g, "mean")
    close(rstd, wrstd, wrstd, g + 6, "rstd")
    gm = torch.ones(c) if gamma is None else gamma
    size = (h.abs() + (wrstd * spread)[:, None]) * gm.double().abs() + want.abs() + (0.0 if beta is None else beta.double().abs())
    close(y, want, size, 2 * g + 8, "y")
    return y, mean, rstd


def backward(learn, full, dy, mean, rstd, gamma, at, c, **more):
    """With the statistics on the host as given to the call."""
    dev = lambda t: None if t is None else t.cuda()  # noqa: E731
    n = full.shape[0]
    got = learn.layer_norm_backward(dy.cuda()[:, at:at + c], full.cuda()[:, at:at + c], dev(mean), dev(rstd), dev(gamma), **more)
    want, sizes = ref.layer_norm_backward(dy[:, at:at + c], full[:, at:at + c], mean, rstd, gamma)
    g = c / 64 + 24
    for t, w, s, k, name in zip(got, want, sizes, (2 * g + 12, n / 64 + 48, n / 64 + 40), ("dx", "dgamma", "dbeta")):
        close(t, w, s, k, name)
    return got


def both(learn, n, c, dtype, seed, rms=False, params=True, ld=0, shift=1.0):
    full, dy, gamma, beta = make(n, c, dtype, seed, shift, params, ld)
    y, mean, rstd = forward(learn, full, gamma, beta, ld // 2, c, rms)
    return y, *backward(learn, full, dy, None if rms else mean.cpu(), rstd.cpu(), gamma, ld // 2, c)


CHANNELS = [1, 2, 3, 4, 5, 7, 8, 9, 15, 16, 17, 31, 33, 63, 64, 65, 96, 127, 128, 129, 255, 257, 384, 511, 512, 513, 768, 1000, 1024, 1025,
            2047, 2049, 4095, 4096, 4097, 8191, 8193, 16383, 16385, 33000]


@pytest.mark.parametrize("c", CHANNELS)
@pytest.mark.parametrize("dtype", TYPES)
def test_channels(learn, c, dtype):
    for i, (rms, params) in enumerate([(False, True), (True, True), (True, False), (False, False)]):
        both(learn, 37 if c < 3000 else 5, c, dtype, 4 * c + i, rms, params, ld=(0, 3, 8, 2)[i])


@pytest.mark.parametrize("n", [1, 2, 3, 63, 64, 65, 361, 1000, 4097, 20001])
@pytest.mark.parametrize("c,dtype", [(24, torch.float32), (130, torch.bfloat16), (384, torch.float16)])
def test_rows(learn, n, c, dtype):
    both(learn, n, c, dtype, n, rms=n % 2 == 0)


def test_many_narrow_rows(learn):
    both(learn, 300001, 16, torch.bfloat16, 5)
    both(learn, 300001, 5, torch.float32, 6, rms=True)


def test_few_wide_rows(learn):
    for dtype in TYPES:
        both(learn, 2, 70001, dtype, 7)
        both(learn, 1, 131072, dtype, 8, rms=True)


def test_far_from_zero(learn):
    """A mean ten thousand deviations off: it is rounded to float, and its rounding is not the result's."""
    for c in (40, 384, 3000, 40000):
        full, _, gamma, beta = make(9, c, torch.float32, c, shift=1e4)
        forward(learn, full, gamma, beta, 0, c, False)


def test_rows_without_spread(learn):
    """Equal values: variance 0, y = beta; and a row of zeros."""
    for c in (1, 16, 384, 5000, 40000):
        x = torch.full((4, c), 3.0)
        x[1], x[3] = 0.0, -0.5
        beta = torch.randn(c)
        y, mean, rstd = learn.layer_norm(x.cuda(), torch.ones(c, device="cuda"), beta.cuda())
        assert torch.equal(y.cpu(), beta.expand(4, c)) and torch.equal(mean.cpu(), x[:, 0])
        assert ((rstd.cpu().double() - 1e-5 ** -0.5).abs() <= 2 * U * 1e-5 ** -0.5).all()
        y, _, rstd = learn.layer_norm(torch.zeros(2, c, device="cuda"), rms=True)
        assert not y.any() and ((rstd.cpu().double() - 1e-5 ** -0.5).abs() <= 2 * U * 1e-5 ** -0.5).all()


def test_not_numbers(learn):
    for c in (16, 384, 5000, 40000):
        for rms in (False, True):
            x, dy = torch.randn(5, c), torch.randn(5, c)
            x[2, c // 2] = math.nan
            x[4, c - 1] = math.inf
            y, mean, rstd = learn.layer_norm(x.cuda(), rms=rms)
            assert torch.isnan(y[2]).all() and torch.isnan(y[4, c - 1]) and torch.isfinite(y[[0, 1, 3]]).all()
            dx, dgamma, dbeta = learn.layer_norm_backward(dy.cuda(), x.cuda(), mean, rstd)
            assert torch.isnan(dx[2]).all() and torch.isfinite(dx[[0, 1, 3]]).all()
            assert torch.isnan(dgamma[c // 2]) and torch.isfinite(dbeta).all()


def test_shapes_and_given_outputs(learn):
    g = torch.Generator().manual_seed(3)
    x, dy = torch.randn(3, 5, 7, 48, generator=g).cuda(), torch.randn(3, 5, 7, 48, generator=g).cuda()
    gamma, beta = torch.randn(48, generator=g).cuda(), torch.randn(48, generator=g).cuda()
    y, mean, rstd = learn.layer_norm(x, gamma, beta)
    flat = learn.layer_norm(x.reshape(-1, 48), gamma, beta)
    assert y.shape == x.shape and mean.shape == rstd.shape == (3, 5, 7)
    assert torch.equal(y.reshape(-1, 48), flat[0]) and torch.equal(mean.reshape(-1), flat[1])
    room = torch.full((3, 5, 7, 64), 2.0, device="cuda")
    out = learn.layer_norm(x, gamma, beta, y=room[..., 8:56])[0]
    assert torch.equal(out, y) and (room[..., :8] == 2).all() and (room[..., 56:] == 2).all()
    dx, dgamma, dbeta = learn.layer_norm_backward(dy, x, mean, rstd, gamma)
    room.fill_(2.0)
    again = learn.layer_norm_backward(dy, x, mean, rstd, gamma, dx=room[..., 8:56])
    assert torch.equal(again[0], dx) and torch.equal(again[1], dgamma) and torch.equal(again[2], dbeta)
    assert (room[..., :8] == 2).all() and (room[..., 56:] == 2).all()


def test_no_rows(learn):
    x = torch.zeros(0, 24, device="cuda")
    y, mean, rstd = learn.layer_norm(x)
    assert y.shape == (0, 24) and mean.shape == (0,)
    dx, dgamma, dbeta = learn.layer_norm_backward(x, x, mean, rstd)
    assert dx.shape == (0, 24) and not dgamma.any() and not dbeta.any() and dgamma.shape == (24,)


def test_same_bits_each_time(learn):
    full, dy, gamma, beta = make(5000, 384, torch.bfloat16, 3)
    y, mean, rstd = learn.layer_norm(full.cuda(), gamma.cuda(), beta.cuda())
    first = learn.layer_norm_backward(dy.cuda(), full.cuda(), mean, rstd, gamma.cuda())
    for _ in range(3):
        for a, b in zip(first, learn.layer_norm_backward(dy.cuda(), full.cuda(), mean, rstd, gamma.cuda())):
            assert torch.equal(a, b)


@pytest.mark.parametrize("rms", [False, True])
def test_differences(learn, rms):
    """The gradients against differences of the definition, 1e-5 either way in float64."""
    full, dy, gamma, beta = make(6, 40, torch.float32, 5)
    _, mean, rstd = learn.layer_norm(full.cuda(), gamma.cuda(), beta.cuda(), rms=rms)
    got = learn.layer_norm_backward(dy.cuda(), full.cuda(), mean, rstd, gamma.cuda())
    g = torch.Generator().manual_seed(1)
    for which, t in enumerate((full, gamma, beta)):
        d = torch.randn(t.shape, generator=g, dtype=torch.float64)
        value = []
        for s in (1e-5, -1e-5):
            args = [full.double(), gamma.double(), beta.double()]
            args[which] = args[which] + s * d
            value.append((ref.layer_norm(*args, rms=rms)[0] * dy.double()).sum())
        along = float((got[which].cpu().double() * d).sum())
        assert abs(float((value[0] - value[1]) / 2e-5) - along) <= 1e-4
