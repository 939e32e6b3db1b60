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


def _like_64(p0, m, v, grad_n, step, lr, wd, b1=0.9, b2=0.999, eps=1e-8):
    """(parameter, update) in float64 from the moments before their rounding."""
    upd = lr / (1 - b1 ** step) * m.astype(np.float64) / (np.sqrt(v.astype(np.float64)) / np.sqrt(1 - b2 ** step) + eps)
    upd = upd.reshape(-1)[:grad_n]
    return p0 * (1 - lr * wd) - upd, upd


SIZES = [1, 3, 255, 256, 257, 1000, 4097, 20001]


@pytest.mark.parametrize("ptype,gtype,master", [("bfloat16", "bfloat16", True), ("float16", "float16", True), ("bfloat16", "float32", True),
                                                ("bfloat16", "bfloat16", False), ("float16", "float32", False),
                                                ("float32", "float16", True)])
def test_8_bit_moments_of_16_bit_parameters(learn, ptype, gtype, master):
    """Three steps: codes and exponents bit for bit; the weights (the masters, or the parameters themselves) within the float bound of
    test_gpu_learn_adamw.py and their type's rounding; a parameter with a master is that one's rounding."""
    pt, gt = getattr(torch, ptype), getattr(torch, gtype)
    g = torch.Generator().manual_seed(3)
    params = [torch.randn(n + 1, generator=g).to(pt).cuda()[i % 2:][:n] for i, n in enumerate(SIZES)]
    masters = [p.float() + 1e-4 for p in params] if master else None
    weights = masters or params
    opt = learn.AdamW(params, lr=1e-2, weight_decay=0.02, state_bits=8, masters=masters)
    eps, least = ref.half_step(weights[0].dtype)
    for step in range(1, 4):
        grads = [(torch.randn(n + 1, generator=g) * 2.0 ** (3 * (i % 4) - 6)).to(gt).cuda()[1:] for i, n in enumerate(SIZES)]
        start, before = [w.double().cpu().numpy() for w in weights], _state(opt)
        opt.step(grads, seed=1000 * step)
        mc, vc, me, ve = _state(opt)
        for i, n in enumerate(SIZES):
            m, v, (um, ur), at = _restated(opt, before, i, grads[i], 1000 * step)
            cm, em = ref.encode(m, um, True)
            cv, ev = ref.encode(np.sqrt(v), ur, False)
            assert np.array_equal(em, me[at]) and np.array_equal(ev, ve[at]), (i, step)
            assert np.array_equal(cm, mc.reshape(-1, 256)[at]) and np.array_equal(cv, vc.reshape(-1, 256)[at]), (i, step)
            want, upd = _like_64(start[i], m, v, n, step, 1e-2, 0.02)
            err = np.abs(weights[i].double().cpu().numpy() - want)
            assert np.all(err <= eps * np.abs(want) + least + 4 * U * np.abs(start[i]) + 16 * U * np.abs(upd)), (i, step)
            if master:
                assert torch.equal(params[i], masters[i].to(pt)), (i, step)


def test_8_bit_moments_of_many_tensors(learn):
    """More tensors than a launch takes, some without a gradient, over two steps: parameters, codes and exponents of each at its own
    place in the state."""
    sizes = [1 + (97 * i) % 1500 for i in range(300)]
    g = torch.Generator().manual_seed(4)
    params = [torch.randn(n, generator=g).cuda() for n in sizes]
    without = (0, 77, 110, 111, 222, 299)
    opt = learn.AdamW(params, lr=1e-2, weight_decay=0.02, state_bits=8)
    for step in (1, 2):
        grads = [None if i in without else torch.randn(n, generator=g).cuda() for i, n in enumerate(sizes)]
        start, before = [p.double().cpu().numpy() for p in params], _state(opt)
        opt.step(grads, seed=9 + step)
        mc, vc, me, ve = _state(opt)
        for i, n in enumerate(sizes):
            if i in without:
                at = slice(int(opt.first_block[i]), int(opt.first_block[i + 1]))
                assert np.array_equal(params[i].double().cpu().numpy(), start[i]), i
                assert not mc.reshape(-1, 256)[at].any() and not vc.reshape(-1, 256)[at].any() and not me[at].any() and not ve[at].any(), i
                continue
            m, v, (um, ur), at = _restated(opt, before, i, grads[i], 9 + step)
            cm, em = ref.encode(m, um, True)
            cv, ev = ref.encode(np.sqrt(v), ur, False)
            assert np.array_equal(em, me[at]) and np.array_equal(ev, ve[at]), (i, step)
            assert np.array_equal(cm, mc.reshape(-1, 256)[at]) and np.array_equal(cv, vc.reshape(-1, 256)[at]), (i, step)
            want, upd = _like_64(start[i], m, v, n, step, 1e-2, 0.02)
            err = np.abs(params[i].double().cpu().numpy() - want)
            assert np.all(err <= 5 * U * np.abs(start[i]) + 17 * U * np.abs(upd)), (i, step)
