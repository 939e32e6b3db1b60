"""The AdamW step with 8-bit moments where other tests do not go: tiny gradients, 16-bit parameters with and without masters, and more
tensors than a launch takes. Codes and exponents are held to the float32 restatement of tests/learn_ref.py."""

import importlib

import numpy as np
import pytest
import torch

import learn_ref as ref

pytestmark = pytest.mark.gpu
U = ref.U
F = np.float32


@pytest.fixture(scope="module")
def learn():
    return importlib.import_module("katago-rs_amd.learn")


def _state(opt):
    return [t.cpu().numpy() for t in (opt.m, opt.v, opt.m_exp, opt.v_exp)]


def _restated(opt, state, i, grad, seed, b1=0.9, b2=0.999):
    """(m, root, the noise of both) of tensor i's blocks after a step with `grad`, from the state before it."""
    mc, vc, me, ve = state
    b0, b1_ = int(opt.first_block[i]), int(opt.first_block[i + 1])
    g = np.zeros((b1_ - b0) * 256, F)
    g[:grad.numel()] = grad.float().cpu().numpy().reshape(-1)
    g = g.reshape(-1, 256)
    m0 = ref.decode_m(mc.reshape(-1, 256)[b0:b1_], me[b0:b1_])
    r0 = ref.decode_v(vc.reshape(-1, 256)[b0:b1_], ve[b0:b1_])
    m = m0 * F(b1) + g * F(1 - b1)
    v = (r0 * r0) * F(b2) + (g * g) * F(1 - b2)
    return m, v, ref.noise(np.arange(b0 * 256, b1_ * 256).reshape(-1, 256), seed), slice(b0, b1_)


def test_tiny_gradients(learn):
    """Second moments down to the subnormal: every code and exponent is the restatement's, whose roots are correctly rounded."""
    n = 256 * 40
    g = torch.Generator().manual_seed(1)
    size = 10.0 ** -(12 + 8 * torch.arange(40) / 39).repeat_interleave(256)
    grad = (torch.randn(n, generator=g) * size).cuda()
    p = torch.zeros(n, device="cuda")
    opt = learn.AdamW([p], lr=1e-3, state_bits=8)
    before = _state(opt)
    opt.step([grad], seed=77)
    mc, vc, me, ve = _state(opt)
    m, v, (um, ur), _ = _restated(opt, before, 0, grad, 77)
    assert (v >= 2.0 ** -96).any() and ((v > 0) & (v < 2.0 ** -126)).any()
    cm, em = ref.encode(m, um, True)
    cv, ev = ref.encode(np.sqrt(v), ur, False)
    assert np.array_equal(em, me) and np.array_equal(cm, mc.reshape(-1, 256))
    assert np.array_equal(ev, ve) and np.array_equal(cv, vc.reshape(-1, 256))


@pytest.mark.parametrize("bits", [32, 8])
def test_tiny_gradients_with_a_tiny_eps(learn, bits):
    """A first step of any gradient moves its parameter by lr |g| / (|g| + eps), whatever the gradient's size. Bound: m's and v's factors
    and products, a root, a quotient: 16 U, and where v is subnormal its own rounding, 2^-150 of it, half of that of its root."""
    grad = torch.tensor([1e-3, 1e-12, 1e-14, 1e-16, 1e-17, 3e-18, 1e-18, 1e-19], dtype=torch.float32).repeat_interleave(256)
    p = torch.zeros(grad.numel(), device="cuda")
    opt = learn.AdamW([p], lr=1.0, eps=1e-30, weight_decay=0.0, state_bits=bits)
    opt.step([grad.cuda()])
    v = 1e-3 * grad.double() ** 2
    bound = 16 * U + 0.5 * 2.0 ** -150 / v
    assert (bound < 0.01).all() and ((p.cpu().double() + 1).abs() <= bound + 1e-30 / grad.double()).all()


def test_step_values_off_their_alignment(learn):
    p = torch.zeros(8, device="cuda")
    opt = learn.AdamW([p], lr=1e-2)
    room = torch.zeros(64, dtype=torch.uint8, device="cuda")
    with pytest.raises(importlib.import_module("katago-rs_amd").KgError, match="values"):
        opt.step([torch.ones_like(p)], values=room[1:41])
    assert opt.step_count == 0 and not p.any()
