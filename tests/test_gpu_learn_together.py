"""The learning operators as a program uses them: a network's raw policy rows judged where they lie; and training steps of a small
head (group norm with mish under a board mask, a product, the policy loss, their gradients, AdamW) against float64 autograd,
against differences, and captured into a graph."""

import contextlib
import importlib

import numpy as np
import pytest
import torch

import learn_ref as ref

pytestmark = pytest.mark.gpu
U = ref.U


@pytest.fixture(scope="module")
def learn():
    return importlib.import_module("katago-rs_amd.learn")


def _upload(pointer, rows):
    """Copies rows into device memory that a handle owns."""
    kgx = importlib.import_module("katago-rs_amd")
    at = torch.as_tensor(kgx.DeviceArray(None, pointer, (rows.size,), (1,)), device="cuda")
    at.copy_(torch.from_numpy(rows.reshape(-1)))


@pytest.mark.parametrize("prec,channel", [("f32", 0), ("bf16", 1)])
def test_a_networks_policy_rows_are_judged_in_place(kgx, learn, synth, prec, channel):
    net = kgx.Net(synth.write_model(synth.tiny_nets()["t_res"], 5))
    channel = min(channel, net.P - 1)
    n = 6
    sp, gl, _ = synth.make_inputs(n, 11, board_sizes=[19, 13, 9, 19])
    with contextlib.closing(kgx.Handle(net, 8, prec)) as h:
        d_bin, d_glob, _, _ = h.device_buffers()
        _upload(d_bin, sp)
        _upload(d_glob, gl)
        torch.cuda.synchronize()
        out = np.empty((n, net.row_len), np.float32)
        h.run(n, out)
        h.run(n)
        h.sync()
        rows = torch.as_tensor(h.policy_rows(n, channel), device="cuda")
        want = torch.from_numpy(out)[:, channel * 362:(channel + 1) * 362]
        assert rows.shape == (n, 362) and rows.stride(0) == net.row_len and torch.equal(rows.cpu(), want)
        g = torch.Generator().manual_seed(2)
        legal = torch.rand(n, 362, generator=g) < 0.6
        legal[:, 361] = True
        actions = torch.tensor([int(torch.nonzero(row)[k]) for k, row in enumerate(legal)], dtype=torch.int32)
        zero = torch.zeros(n, device="cuda")
        first = learn.policy_loss(rows, actions.cuda(), zero, zero, legal=legal.cuda(), want_grad=False)
        old = first.logp - 0.05
        adv = torch.randn(n, generator=g)
        got = learn.policy_loss(rows, actions.cuda(), old, adv.cuda(), legal=legal.cuda())
        loss, logp, _, grad, size = ref.policy(want, actions, old.cpu(), adv, legal)
        # X: the largest exponent, in octaves; the sums have 362 terms.
        span = torch.where(legal, want, -torch.inf).max(1).values - torch.where(legal, want, torch.inf).min(1).values
        k = 3 * float(span.max() * 1.4427) + 362 / 64 + 20
        assert ((got.logp.cpu() - logp).abs() <= U * (logp.abs() + k)).all()
        assert ((got.loss.cpu() - loss).abs() <= U * loss.abs() * 2 + k * U * adv.abs() * 1.1).all()
        assert ((got.grad.cpu() - grad).abs() <= U * grad.abs() + k * U * size).all()
        assert torch.equal(rows.cpu(), want)


def test_policy_rows_refuses(kgx, synth):
    net = kgx.Net(synth.write_model(synth.tiny_nets()["t_res"], 5))
    with contextlib.closing(kgx.Handle(net, 4, "f16")) as h:
        for n, channel in ((0, 0), (5, 0), (1, -1), (1, net.P)):
            with pytest.raises(ValueError, match="policy_rows"):
                h.policy_rows(n, channel)


B, P, C, GROUPS, V = 3, 361, 96, 8, 75


def _data(seed):
    g = torch.Generator().manual_seed(seed)
    t = B * P
    mask = (torch.rand(B, P, generator=g) < 0.8).float()
    return {"x": torch.randn(B, P, C, generator=g), "mask": mask, "actions": torch.randint(0, V, (t,), generator=g, dtype=torch.int32),
            "old": -4.5 + 0.3 * torch.randn(t, generator=g), "adv": torch.randn(t, generator=g), "weight": mask.reshape(-1) / t,
            "ref": torch.randn(t, V, generator=g)}


def _parameters(seed):
    g = torch.Generator().manual_seed(seed)
    return [0.1 * torch.randn(C, V, generator=g), 1 + 0.1 * torch.randn(C, generator=g), 0.1 * torch.randn(C, generator=g)]


def _gradients(learn, d, w, gamma, beta, dw=None):
    """(sum of the losses, [dw, dgamma, dbeta], dx) of a step."""
    y, mean, rstd = learn.group_norm(d["x"], GROUPS, gamma, beta, mask=d["mask"], act="mish")
    flat = y.reshape(-1, C)
    out = learn.policy_loss(flat @ w, d["actions"], d["old"], d["adv"], weight=d["weight"], kl_coef=0.2, ref_logits=d["ref"])
    dw = torch.mm(flat.t(), out.grad, out=dw)
    dy = (out.grad @ w.t()).reshape(y.shape)
    dx, dgamma, dbeta = learn.group_norm_backward(dy, d["x"], mean, rstd, GROUPS, gamma, beta, mask=d["mask"], act="mish")
    return out.loss, [dw, dgamma, dbeta], dx


def _reference(d, x, w, gamma, beta):
    """The sum of the losses in float64, differentiable."""
    on = d["mask"].double()[:, :, None, None]
    xg = x.reshape(B, P, GROUPS, -1)
    n = on.sum((1, 2, 3), keepdim=True) * (C // GROUPS)
    mean = (xg * on).sum((1, 3), keepdim=True) / n
    var = (((xg - mean) * on) ** 2).sum((1, 3), keepdim=True) / n
    a = ((xg - mean) / torch.sqrt(var + 1e-5)).reshape(B, P, C) * gamma + beta
    y = torch.nn.functional.mish(a) * on[..., 0]
    lsm = torch.log_softmax(y.reshape(-1, C) @ w, 1)
    rsm = torch.log_softmax(d["ref"].double(), 1)
    lp = lsm.gather(1, d["actions"].long()[:, None])[:, 0]
    ratio, adv = torch.exp(lp - d["old"].double()), d["adv"].double()
    kl = (torch.exp(lsm) * (lsm - rsm)).sum(1)
    return (d["weight"].double() * (0.2 * kl - torch.minimum(ratio * adv, ratio.clamp(0.8, 1.2) * adv))).sum()


def test_a_steps_gradients(learn):
    d, par = _data(1), _parameters(2)
    dev = {k: t.cuda() for k, t in d.items()}
    loss, got, dx = _gradients(learn, dev, *[p.cuda() for p in par])
    leaves = [t.double().requires_grad_() for t in (d["x"], *par)]
    want = _reference(d, *leaves)
    grads = torch.autograd.grad(want, leaves)
    # No ratio at its border, or float's and double's sides may differ.
    with torch.no_grad():
        x, w, gamma, beta = leaves
        xg = x.reshape(B, P, GROUPS, -1)
        on = d["mask"].double()[:, :, None, None]
        n = on.sum((1, 2, 3), keepdim=True) * (C // GROUPS)
        mean = (xg * on).sum((1, 3), keepdim=True) / n
        var = (((xg - mean) * on) ** 2).sum((1, 3), keepdim=True) / n
        y = torch.nn.functional.mish(((xg - mean) / torch.sqrt(var + 1e-5)).reshape(B, P, C) * gamma + beta) * on[..., 0]
        z = y.reshape(-1, C) @ w
        ratio = torch.exp(torch.log_softmax(z, 1).gather(1, d["actions"].long()[:, None])[:, 0] - d["old"].double())
        assert min(float((ratio - 0.8).abs().min()), float((ratio - 1.2).abs().min())) > 1e-5
        # Each stage alone is held to its own bound elsewhere; together: a float sum of at most 1083 terms in any order is off by
        # 1083 U of its terms' sizes, and a logit's error Z (|y| |w| summed, times (C + 200) U for the product and the norm's
        # statistics) is a relative one of every probability and ratio. The terms' sizes: |w| (p + onehot) (ratio |adv| + 0.2
        # (|log p/r| + KL)) a logit, and what the products and the norm make of it.
        zsize = float((y.reshape(-1, C).abs() @ w.abs()).max()) + 1
        lsm, rsm = torch.log_softmax(z, 1), torch.log_softmax(d["ref"].double(), 1)
        p = torch.exp(lsm)
        hot = torch.zeros_like(p).scatter_(1, d["actions"].long()[:, None], 1.0)
        gap = (lsm - rsm).abs()
        gs = d["weight"].double()[:, None] * ((ratio * d["adv"].double().abs())[:, None] * (p + hot)
                                              + 0.2 * p * (gap + (p * gap).sum(1, keepdim=True) + 1))
        rel = U * (1083 + 2 * (C + 200) * zsize)
        flat = y.reshape(-1, C).abs()
        dw_size = flat.t() @ gs + gs.sum(0)  # (y's own error is relative to 1 + |y|)
        da = (gs @ w.abs().t()).reshape(B, P, C) * 1.1
        xh = ((xg - mean) / torch.sqrt(var + 1e-5)).reshape(B, P, C).abs()
        dg_size, db_size = (da * (xh + 1)).sum((0, 1)), da.sum((0, 1))
        d4, x4 = (da * gamma.abs()).reshape(B, P, GROUPS, -1) * on, xh.reshape(B, P, GROUPS, -1)
        m1, m2 = d4.sum((1, 3), keepdim=True) / n, (d4 * x4).sum((1, 3), keepdim=True) / n
        dx_size = ((d4 + m1 + (x4 + 1) * (m2 + m1)) / torch.sqrt(var + 1e-5)).reshape(B, P, C)
    assert abs(float(loss.double().sum()) - float(want.detach())) <= rel * float(gs.sum())
    for g, t, size in zip((dx, *got), grads, (dx_size, dw_size, dg_size, db_size)):
        assert ((g.cpu().double() - t).abs() <= 2 * rel * size).all(), float(((g.cpu().double() - t).abs() / (rel * size + 1e-30)).max())
    # And differences of the reference along random directions, half a step's square off: with steps of 1e-5 in float64.
    g = torch.Generator().manual_seed(3)
    for leaf, t in zip(leaves, (dx, *got)):
        v = torch.randn(leaf.shape, generator=g, dtype=torch.float64)
        v *= 1e-5 / v.norm()
        moved = [[q + s * v if q is leaf else q for q in leaves] for s in (1, -1)]
        slope = float((_reference(d, *moved[0]) - _reference(d, *moved[1])).detach()) / 2
        along = float((t.cpu().double() * v).sum())
        assert abs(slope - along) <= 1e-3 * float((t.cpu().double().norm() * v.norm())) + 1e-12


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_steps_are_the_eager_ones(learn, bits):
    """Three steps, eager and by one graph that is replayed: the same parameters and moments, bit for bit."""
    batches = [{k: t.cuda() for k, t in _data(10 + k).items()} for k in range(3)]
    runs = []
    for captured in (False, True):
        par = [p.cuda() for p in _parameters(2)]
        opt = learn.AdamW(par, lr=0.01, weight_decay=[0.1, 0.0, 0.0], state_bits=bits)
        losses = []
        if captured:
            buf = {k: t.clone() for k, t in batches[0].items()}
            dw = torch.empty_like(par[0])
            values = opt.values(lr=0.0).cuda()
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):  # the libraries' own first calls
                _gradients(learn, buf, *par, dw=dw)
            torch.cuda.current_stream().wait_stream(side)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                loss, grads, _ = _gradients(learn, buf, *par, dw=dw)
                opt.step(grads, values=values, step=1)
            opt.step_count = 0
        for k, d in enumerate(batches):
            lr = 0.01 / (1 + k)
            if captured:
                for name, t in d.items():
                    buf[name].copy_(t)
                values.copy_(opt.values(lr=lr, step=k + 1))
                graph.replay()
                torch.cuda.synchronize()
            else:
                loss, grads, _ = _gradients(learn, d, *par)
                opt.step(grads, lr=lr)
            losses.append(loss.clone())
        runs.append([*losses, *par, *opt.moments()])
    for a, b in zip(*runs):
        assert torch.equal(a, b)
    assert not torch.equal(runs[0][3].cpu(), _parameters(2)[0])


def test_two_programs_at_once(learn):
    """Two streams with steps of their own, interleaved: each as alone."""
    batches = [{k: t.cuda() for k, t in _data(20 + k).items()} for k in range(2)]

    def start(k):
        par = [p.cuda() for p in _parameters(30 + k)]
        return par, learn.AdamW(par, lr=0.01, state_bits=8)

    def step(k, par, opt):
        _, grads, dx = _gradients(learn, batches[k], *par)
        opt.step(grads)
        return dx

    want = []
    for k in range(2):
        par, opt = start(k)
        for _ in range(3):
            dx = step(k, par, opt)
        want.append([*par, dx, *opt.moments()])
    both, streams = [start(k) for k in range(2)], [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    dxs = [None, None]
    for _ in range(3):
        for k in range(2):
            with torch.cuda.stream(streams[k]):
                dxs[k] = step(k, *both[k])
    torch.cuda.synchronize()
    for k, (par, opt) in enumerate(both):
        for a, b in zip([*par, dxs[k], *opt.moments()], want[k]):
            assert torch.equal(a, b)
