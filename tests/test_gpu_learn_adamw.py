"""The AdamW step on the GPU: moments in 32 bits against float64 (each of m, v and the update is a handful of float operations, so
they are off by a few U of their terms), moments in 8 bits bit for bit against the float32 restatement of tests/learn_ref.py."""

import importlib

import numpy as np
import pytest
import torch

import learn_ref as ref

pytestmark = pytest.mark.gpu
U = ref.U
SIZES = [1, 2, 3, 255, 256, 257, 1000, 4095, 4096, 4097, 16384, 70001]


@pytest.fixture(scope="module")
def learn():
    return importlib.import_module("katago-rs_amd.learn")


def _params(sizes, dtype, seed, shift=0):
    """Parameters at odd places of larger buffers, so that they start anywhere."""
    g = torch.Generator().manual_seed(seed)
    out = []
    for i, n in enumerate(sizes):
        room = torch.randn(n + shift + 3, generator=g).to(dtype).cuda()
        out.append(room[shift:shift + n] if i % 2 else room[:n].clone())
    return out


@pytest.mark.parametrize("ptype,gtype,master", [("float32", "float32", False), ("float32", "bfloat16", False), ("bfloat16", "bfloat16", True),
                                                ("float16", "float32", True), ("bfloat16", "float32", False), ("float16", "float16", False)])
def test_adamw_32_against_float64(learn, ptype, gtype, master):
    pt, gt = getattr(torch, ptype), getattr(torch, gtype)
    params = _params(SIZES, pt, 1, 1)
    masters = [p.float() + 1e-4 for p in params] if master else None
    wds = [0.1 * (i % 3) for i in range(len(SIZES))]
    opt = learn.AdamW(params, lr=3e-3, betas=(0.8, 0.99), eps=1e-6, weight_decay=wds, masters=masters)
    start = [(w if master else p).clone().cpu() for p, w in zip(params, masters or params)]
    state = [(torch.zeros(n), torch.zeros(n)) for n in SIZES]
    for step in range(1, 4):
        grads = _params(SIZES, gt, 10 + step, 2)
        opt.step(grads, grad_scale=0.5)
        for i, n in enumerate(SIZES):
            at = int(opt.first_block[i]) * 256
            p0, (m0, v0) = start[i], state[i]
            p, m, v = ref.adamw(p0.float(), grads[i].cpu(), m0, v0, step, 3e-3, 0.8, 0.99, 1e-6, wds[i], 0.5)
            gd = grads[i].cpu().double().abs() * 0.5
            gm, gv = opt.m[at:at + n].cpu(), opt.v[at:at + n].cpu()
            # m and v: two products and a sum, and the factors' own rounding to float: 4 U of the terms.
            assert ((gm.double() - m).abs() <= 4 * U * (0.8 * m0.double().abs() + 0.2 * gd) + 1e-45).all()
            assert ((gv.double() - v).abs() <= 6 * U * (v.abs()) + 1e-45).all()
            got = (masters[i] if master else params[i]).cpu()
            # The update: m's error against sqrt(v) (m's terms may cancel), and eight more roundings.
            root = torch.sqrt(v / (1 - 0.99 ** step)) + 1e-6
            terms = 3e-3 / (1 - 0.8 ** step) * (0.8 * m0.double().abs() + 0.2 * gd) / root
            eps, least = ref.half_step(got.dtype)
            assert ((got.double() - p).abs() <= eps * p.abs() + least + 3 * U * p0.double().abs() + 16 * U * terms).all(), (i, step)
            if master:  # the parameter is its master's rounding
                assert torch.equal(params[i].cpu(), got.to(pt))
            start[i], state[i] = got.clone(), (gm, gv)
            assert not opt.m[at + n:int(opt.first_block[i + 1]) * 256].any()
    assert opt.step_count == 3


def _state8(opt):
    return [t.cpu().numpy() for t in (opt.m, opt.v, opt.m_exp, opt.v_exp)]


@pytest.mark.parametrize("gtype", [torch.float32, torch.bfloat16])
def test_adamw_8_bit_codes_are_the_restatements(learn, gtype):
    """Three steps, every code and exponent equal, and the parameters within the float bound from the same moments."""
    f = np.float32
    params = _params(SIZES, torch.float32, 2, 1)
    opt = learn.AdamW(params, lr=1e-2, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.02, state_bits=8)
    b1, b1r, b2, b2r = f(0.9), f(1 - 0.9), f(0.999), f(1 - 0.999)
    for step, seed in ((1, 5), (2, 123456789), (3, 2 ** 32 - 1)):
        before = [p.cpu().numpy().astype(np.float64) for p in params]
        mc, vc, me, ve = _state8(opt)
        m0, r0 = ref.decode_m(mc.reshape(-1, 256), me), ref.decode_v(vc.reshape(-1, 256), ve)
        grads = [(g * 2.0 ** (3 * (i % 5) - 9)).to(gtype) for i, g in enumerate(_params(SIZES, torch.float32, 20 + step, 2))]
        grads[5][100:140] = 0
        opt.step(grads, seed=seed)
        mc, vc, me, ve = _state8(opt)
        for i, n in enumerate(SIZES):
            b0, b1_ = int(opt.first_block[i]), int(opt.first_block[i + 1])
            g = np.zeros((b1_ - b0) * 256, f)
            g[:n] = grads[i].float().cpu().numpy()
            g = g.reshape(-1, 256)
            m = m0[b0:b1_] * b1 + g * b1r
            v = (r0[b0:b1_] * r0[b0:b1_]) * b2 + (g * g) * b2r
            root = np.sqrt(v)
            um, ur = ref.noise(np.arange(b0 * 256, b1_ * 256).reshape(-1, 256), seed)
            cm, em = ref.encode(m, um, True)
            cv, ev = ref.encode(root, ur, False)
            assert np.array_equal(em, me[b0:b1_]) and np.array_equal(ev, ve[b0:b1_]), (i, step)
            assert np.array_equal(cm, mc.reshape(-1, 256)[b0:b1_]), (i, step)
            assert np.array_equal(cv, vc.reshape(-1, 256)[b0:b1_]), (i, step)
            s = 1e-2 / (1 - 0.9 ** step)
            upd = s * m.astype(np.float64) / (root.astype(np.float64) / np.sqrt(1 - 0.999 ** step) + 1e-8)
            want = before[i] * (1 - 1e-2 * 0.02) - upd.reshape(-1)[:n]
            err = np.abs(params[i].cpu().numpy() - want)
            assert np.all(err <= 4 * U * np.abs(before[i]) + 16 * U * np.abs(upd.reshape(-1)[:n])), (i, step)
    m, root = opt.moments()
    assert m.dtype == torch.bfloat16
    assert np.array_equal(m.float().cpu().numpy().reshape(-1, 256), ref.decode_m(mc.reshape(-1, 256), me))
    assert np.array_equal(root.float().cpu().numpy().reshape(-1, 256), ref.decode_v(vc.reshape(-1, 256), ve))


def test_adamw_8_bit_moments_hold_their_values(learn):
    """No gradients, many steps: v decays by its factor on average, though a step's change is far below a code's spacing. With
    4096 elements and 200 steps the mean of the second moments keeps to its formula within 4 % (each step's rounding of a
    root is off by at most 1/32 of it, evenly, which adds at most (1/32)^2 / 6 = 0.016 % a step to its square, 3.3 % in all, and
    scatters the mean by far less)."""
    p = torch.zeros(4096, device="cuda")
    opt = learn.AdamW([p], lr=1e-3, betas=(0.9, 0.999), state_bits=8)
    g = torch.randn(4096, device="cuda")
    opt.step([g])
    start = float((opt.moments(torch.float32)[1].double() ** 2).sum())
    z = torch.zeros_like(g)
    opt.bind([z])
    for _ in range(200):
        opt.step()
    end = float((opt.moments(torch.float32)[1].double() ** 2).sum())
    assert abs(end / start / 0.999 ** 200 - 1) <= 0.04


def test_adamw_many_tensors_and_missing_gradients(learn):
    """More tensors than a launch takes, some without a gradient: the same as one at a time, bit for bit."""
    sizes = [1 + (97 * i) % 1500 for i in range(300)]
    params = _params(sizes, torch.float32, 3)
    single = [p.clone() for p in params]
    grads = _params(sizes, torch.float32, 4)
    grads[0] = grads[77] = grads[299] = None
    for bits in (32, 8):
        opt = learn.AdamW(params, lr=1e-2, state_bits=bits)
        opt.step(grads, seed=9)
        for i, p in enumerate(single):
            one = learn.AdamW([p], lr=1e-2, state_bits=bits)
            if bits == 8:  # (its rounding goes by the place in the state)
                continue
            if grads[i] is not None:
                one.step([grads[i]])
                at = int(opt.first_block[i]) * 256
                assert torch.equal(opt.m[at:at + sizes[i]], one.m[:sizes[i]]) and torch.equal(opt.v[at:at + sizes[i]], one.v[:sizes[i]])
            assert torch.equal(p, params[i]), i
        assert not opt.m[:256].any() and not opt.v[:256].any()


def test_adamw_not_a_number_is_seen(learn):
    for bits in (32, 8):
        p = torch.ones(1024, device="cuda")
        opt = learn.AdamW([p], lr=1e-2, state_bits=bits)
        g = torch.ones(1024, device="cuda")
        g[300] = torch.nan
        opt.step([g])
        opt.step([torch.ones_like(g)])
        m, root = opt.moments(torch.float32)
        bad = torch.isnan(m).nonzero().flatten().tolist()
        assert bad == ([300] if bits == 32 else list(range(256, 512))) and torch.isnan(p[300])
        assert torch.isfinite(p[:256]).all() and torch.isfinite(p[512:]).all()
    p = torch.ones(256, device="cuda")
    opt = learn.AdamW([p], lr=1e-2, state_bits=8)
    opt.step([torch.full_like(p, torch.inf)])
    assert torch.isnan(opt.moments(torch.float32)[0]).all()


def test_adamw_tiny_and_mixed_gradients_stay_bounded(learn):
    """Elements far below their block's largest: a step moves a parameter by no more than a few lr, in 8 bits too."""
    g = torch.full((512,), 1e-7, device="cuda")
    g[::256] = 1e3
    p = torch.zeros(512, device="cuda")
    opt = learn.AdamW([p], lr=1.0, weight_decay=0.0, state_bits=8)
    for s in range(20):
        before = p.clone()
        opt.step([g])
        assert (p - before).abs().max() <= 8.0, s


def test_adamw_captured_steps_read_their_values(learn):
    """A captured step replayed with new scalars and gradients equals eager steps, bit for bit, in both kinds of state."""
    for bits in (32, 8):
        g = torch.Generator().manual_seed(8)
        start = torch.randn(5000, generator=g)
        grads = [torch.randn(5000, generator=g).cuda() for _ in range(4)]
        a, b = start.clone().cuda(), start.clone().cuda()
        eager, graphed = (learn.AdamW([t], lr=1e-2, state_bits=bits) for t in (a, b))
        buf = torch.zeros(5000, device="cuda")
        vals = torch.zeros(len(graphed.values()), dtype=torch.uint8, device="cuda")
        graphed.bind([buf])
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            graphed.step(values=vals, step=1)
        for k in range(4):
            eager.step([grads[k]], lr=1e-2 / (k + 1), seed=1000 + k)
            buf.copy_(grads[k])
            vals.copy_(graphed.values(lr=1e-2 / (k + 1), step=k + 1, seed=1000 + k))
            gr.replay()
            torch.cuda.synchronize()
            assert torch.equal(a, b) and torch.equal(eager.m, graphed.m) and torch.equal(eager.v, graphed.v), (bits, k)


def test_adamw_state_round_trip(learn):
    for bits in (32, 8):
        g = torch.Generator().manual_seed(6)
        p = torch.randn(700, generator=g).cuda()
        grads = [torch.randn(700, generator=g).cuda() for _ in range(3)]
        one = learn.AdamW([p], lr=1e-2, state_bits=bits)
        one.step([grads[0]])
        tensors, count = one.state()
        q = p.clone()
        two = learn.AdamW([q], lr=1e-2, state_bits=bits)
        two.load_state({k: t.cpu() for k, t in tensors.items()}, count)
        for k in (1, 2):
            one.step([grads[k]])
            two.step([grads[k]])
        assert torch.equal(p, q) and torch.equal(one.m, two.m) and one.step_count == two.step_count == 3


def test_adamw_refuses_on_the_gpu(learn):
    p = torch.zeros(8, device="cuda")
    opt = learn.AdamW([p], lr=1e-2)
    KgError = importlib.import_module("katago-rs_amd").KgError
    with pytest.raises(ValueError, match="needs gradients"):
        opt.step()
    with pytest.raises(ValueError, match="1 gradients"):
        opt.step([p, p])
    with pytest.raises(ValueError, match="each gradient"):
        opt.step([torch.zeros(9, device="cuda")])
    with pytest.raises(ValueError, match="values"):
        opt.step([p.clone()], values=torch.zeros(3, device="cuda"))
    with pytest.raises(KgError, match="step counts"):
        opt.step([p.clone()], step=0)
    with pytest.raises(ValueError, match="parameter 0"):
        learn.AdamW([torch.zeros(4, 4, device="cuda").t()[1:]], lr=1e-2)
    with pytest.raises(ValueError, match="master 0"):
        learn.AdamW([p.half()], lr=1e-2, masters=[p.half()])
    with pytest.raises(ValueError, match="state's v"):
        opt.load_state({"m": opt.m}, 1)
    with pytest.raises(ValueError, match="state_bits"):
        learn.AdamW([p], lr=1e-2, state_bits=16)
    with pytest.raises(ValueError, match="weight decays"):
        learn.AdamW([p], lr=1e-2, weight_decay=[0.1, 0.2])
