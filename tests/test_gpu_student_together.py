"""A student as a program trains it: tokens, their embedding, layer or RMS norm, a product with the same table, the distillation loss
against a teacher's top logits, all gradients, AdamW. Against float64 autograd, captured into a graph, and on streams of their own.

Bounds of the gradients: each stage alone is held to its own bound elsewhere; together, a float sum of at most N = V + T + C terms in
any order is off by N U of its terms' sizes, and a logit's error Z (its terms' sizes |h| |w| summed, times (C + 200) U for the product and
the norm's statistics) is a relative one of every probability. The sizes are the formulas' with every term's magnitude."""

import importlib

import pytest
import torch

import learn_ref

pytestmark = pytest.mark.gpu
U = learn_ref.U
T, V, C, K, SCALE, TEMPERATURE = 61, 75, 96, 9, 3.0, 0.5


@pytest.fixture(scope="module")
def learn():
    return importlib.import_module("katago-rs_amd.learn")


def data(seed):
    g = torch.Generator().manual_seed(seed)
    teacher = 2 * torch.randn(T, V, generator=g)
    top, index = teacher.topk(K, 1)
    index = index.int()
    index[5] = -1        # padding
    index[7, 4:] = -1    # fewer entries
    tokens = torch.randint(0, V, (T,), generator=g, dtype=torch.int32)
    tokens[3], tokens[20:30] = -1, 11
    return {"tokens": tokens, "index": index, "top": top, "lse": torch.logsumexp(teacher * TEMPERATURE, 1),
            "weight": (torch.rand(T, generator=g) + 0.1) / T}


def parameters(seed):
    g = torch.Generator().manual_seed(seed)
    return [0.1 * torch.randn(V, C, generator=g), 1 + 0.1 * torch.randn(C, generator=g), 0.1 * torch.randn(C, generator=g)]


def gradients(learn, d, table, gamma, beta, rms=False, room=None):
    """(losses, [dtable, dgamma, dbeta]) of a step."""
    e = learn.embedding(d["tokens"], table, scale=SCALE)
    h, mean, rstd = learn.layer_norm(e, gamma, beta, rms=rms)
    out = learn.distill_loss(h @ table.t(), d["index"], d["top"], weight=d["weight"], logit_scale=TEMPERATURE, teacher_lse=d["lse"])
    dtable = torch.mm(out.grad.t(), h, out=room)
    de, dgamma, dbeta = learn.layer_norm_backward(out.grad @ table, e, mean, rstd, gamma)
    learn.embedding_backward(de, d["tokens"], V, scale=SCALE, grad=dtable, accumulate=True)
    return out.loss, [dtable, dgamma, dbeta]


def reference(d, table, gamma, beta, rms):
    """The sum of the losses in float64, differentiable, with what the bounds' sizes come from."""
    tokens, index = d["tokens"].long(), d["index"].long()
    e = SCALE * table[tokens.clamp(min=0)] * (tokens >= 0)[:, None]
    mean = torch.zeros(T, 1, dtype=torch.float64) if rms else e.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt(((e - mean) ** 2).mean(1, keepdim=True) + 1e-5)
    xh = (e - mean) * rstd
    h = xh * gamma + beta
    lsm = torch.log_softmax(TEMPERATURE * (h @ table.t()), 1)
    there = index >= 0
    part = there.any(1)
    q = torch.where(there, torch.exp(TEMPERATURE * d["top"].double() - d["lse"].double()[:, None]), 0.0)
    rest = 1 - q.sum(1)
    free = torch.ones(T, V, dtype=torch.bool).scatter(1, index.clamp(min=0), ~there)
    left = torch.logsumexp(torch.where(free, lsm, -torch.inf), 1)
    loss = torch.special.xlogy(q, q).sum(1) - (q * lsm.gather(1, index.clamp(min=0))).sum(1) + rest * (torch.log(rest) - left)
    qs = torch.zeros(T, V, dtype=torch.float64).scatter_add(1, index.clamp(min=0), q)
    weight = torch.where(part, d["weight"].double(), 0.0)
    p = torch.exp(lsm)
    size = weight[:, None] * TEMPERATURE * (p + qs + torch.where(free, p * (rest / torch.exp(left))[:, None], 0.0))
    return (weight * torch.where(part, loss, 0.0)).sum(), (weight * loss.abs()).sum(), size.detach(), xh.detach(), rstd.detach(), h.detach()


@pytest.mark.parametrize("rms", [False, True])
def test_a_steps_gradients(learn, rms):
    d, par = data(1), parameters(2)
    loss, got = gradients(learn, {k: t.cuda() for k, t in d.items()}, *[p.cuda() for p in par], rms=rms)
    leaves = [p.double().requires_grad_() for p in par]
    want, lsize, gs, xh, rstd, h = reference(d, *leaves, rms)
    grads = torch.autograd.grad(want, leaves)
    with torch.no_grad():
        table, gamma, _ = leaves
        n, zsize = V + T + C, TEMPERATURE * float((h.abs() @ table.abs().t()).max()) + 1
        rel = U * (n + 2 * (C + 200) * zsize)
        dh = gs @ table.abs()
        d1 = dh * gamma.abs()
        de = rstd * (d1 + d1.mean(1, keepdim=True) + (xh.abs() + 1) * (d1 * (xh.abs() + 1)).mean(1, keepdim=True))
        tokens = d["tokens"].long()
        on = tokens >= 0
        dt = gs.t() @ (h.abs() + 1) + SCALE * torch.zeros(V, C, dtype=torch.float64).index_add(0, tokens[on], de[on])
        sizes = (dt, (dh * (xh.abs() + 1)).sum(0), dh.sum(0))
    assert abs(float(loss.double().sum()) - float(want.detach())) <= rel * (float(lsize.detach()) + float(gs.sum()))
    for g, t, size in zip(got, grads, sizes):
        assert ((g.cpu().double() - t).abs() <= 2 * rel * size).all(), float(((g.cpu().double() - t).abs() / (rel * size + 1e-30)).max())
    # And differences along random directions in float64.
    r = torch.Generator().manual_seed(3)
    for i, t in enumerate(got):
        v = torch.randn(t.shape, generator=r, dtype=torch.float64)
        v *= 1e-5 / v.norm()
        value = [reference(d, *[(q + s * v if k == i else q).detach() for k, q in enumerate(leaves)], rms)[0] for s in (1, -1)]
        along = float((t.cpu().double() * v).sum())
        assert abs(float(value[0] - value[1]) / 2 - along) <= 1e-3 * float(t.cpu().double().norm() * v.norm()) + 1e-12


def test_captured_steps_are_the_eager_ones(learn):
    """Six steps, eager and by one graph that is replayed with eager work between: the same losses, parameters and moments, bit for bit."""
    batches = [{k: t.cuda() for k, t in data(10 + k).items()} for k in range(6)]
    runs = []
    for captured in (False, True):
        par = [p.cuda() for p in parameters(2)]
        opt = learn.AdamW(par, lr=0.01, weight_decay=[0.1, 0.0, 0.0])
        losses = []
        if captured:
            buf = {k: t.clone() for k, t in batches[0].items()}
            room, values = torch.empty_like(par[0]), opt.values(lr=0.0).cuda()
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):  # the libraries' own first calls
                gradients(learn, buf, *par, room=room)
            torch.cuda.current_stream().wait_stream(side)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                loss, grads = gradients(learn, buf, *par, room=room)
                opt.step(grads, values=values, step=1)
            opt.step_count = 0
        for k, d in enumerate(batches):
            lr = 0.01 / (1 + k)
            if captured:
                for name, t in d.items():
                    buf[name].copy_(t)
                values.copy_(opt.values(lr=lr, step=k + 1))
                graph.replay()
                gradients(learn, d, *[p.clone() for p in par])  # the program's own eager work
                torch.cuda.synchronize()
            else:
                loss, grads = gradients(learn, d, *par)
                opt.step(grads, lr=lr)
            losses.append(loss.clone())
        runs.append([*losses, *par, *opt.moments()])
    for a, b in zip(*runs):
        assert torch.equal(a, b)
    assert not torch.equal(runs[0][6].cpu(), parameters(2)[0])


def test_large_calls_replayed(learn):
    """The variants of more than one launch (sorted tokens, rows by slabs, losses in parts and apart) in a graph, against the eager calls."""
    g = torch.Generator(device="cuda").manual_seed(5)
    tokens = torch.randint(0, 300, (20000,), generator=g, device="cuda").int()
    dy = torch.randn(20000, 40, generator=g, device="cuda").bfloat16()
    x, dx = (torch.randn(40, 9000, generator=g, device="cuda").bfloat16() for _ in range(2))
    z, zl = torch.randn(600, 5000, generator=g, device="cuda"), torch.randn(3, 70001, generator=g, device="cuda").half()
    _, mean, rstd = learn.layer_norm(x)

    def step():
        out = [learn.embedding_backward(dy, tokens, 300), learn.embedding(tokens, dy)]
        out += learn.layer_norm(x)
        out += learn.layer_norm_backward(dx, x, mean, rstd)
        for logits in (z, zl):
            top, index = logits[:, :50].float() + 1, torch.arange(50, device="cuda", dtype=torch.int32).expand(logits.shape[0], 50)
            out += learn.distill_loss(logits, index.contiguous(), top)
        return out

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for k in range(4):
        for t in (dy, x, dx, z, zl):
            t.mul_(0.9)
        tokens.add_(7).remainder_(300)
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b), k


def test_two_programs_at_once(learn):
    """Two streams with steps of their own, interleaved: each as alone."""
    batches = [{k: t.cuda() for k, t in data(20 + k).items()} for k in range(2)]

    def start(k):
        par = [p.cuda() for p in parameters(30 + k)]
        return par, learn.AdamW(par, lr=0.01, state_bits=8)

    def step(k, par, opt):
        loss, grads = gradients(learn, batches[k], *par, rms=k == 1)
        opt.step(grads)
        return loss

    want = []
    for k in range(2):
        par, opt = start(k)
        for _ in range(3):
            loss = step(k, par, opt)
        want.append([*par, loss, *opt.moments()])
    both, streams, losses = [start(k) for k in range(2)], [torch.cuda.Stream() for _ in range(2)], [None, None]
    torch.cuda.synchronize()
    for _ in range(3):
        for k in range(2):
            with torch.cuda.stream(streams[k]):
                losses[k] = step(k, *both[k])
    torch.cuda.synchronize()
    for k in range(2):
        par, opt = both[k]
        for a, b in zip([*par, losses[k], *opt.moments()], want[k]):
            assert torch.equal(a, b)


def test_a_networks_policy_rows(kgx, learn, synth):
    """The raw rows that a network left on the device, taught in place by another's top moves."""
    import contextlib

    import numpy as np

    import student_ref as ref
    from test_gpu_distill import close, octaves
    net = kgx.Net(synth.write_model(synth.tiny_nets()["t_res"], 5))
    n = 6
    sp, gl, _ = synth.make_inputs(n, 11, board_sizes=[19, 13, 9, 19])
    with contextlib.closing(kgx.Handle(net, 8, "f32")) as h:
        d_bin, d_glob, _, _ = h.device_buffers()
        for pointer, rows in ((d_bin, sp), (d_glob, gl)):
            torch.as_tensor(kgx.DeviceArray(None, pointer, (rows.size,), (1,)), device="cuda").copy_(torch.from_numpy(rows.reshape(-1)))
        torch.cuda.synchronize()
        out = np.empty((n, net.row_len), np.float32)
        h.run(n, out)
        h.run(n)
        h.sync()
        rows = torch.as_tensor(h.policy_rows(n, 0), device="cuda")
        z = torch.from_numpy(out)[:, :362]
        g = torch.Generator().manual_seed(2)
        teacher = z + torch.randn(n, 362, generator=g)
        top, index = teacher.topk(16, 1)
        lse = torch.logsumexp(teacher, 1)
        got = learn.distill_loss(rows, index.int().cuda(), top.cuda(), teacher_lse=lse.cuda())
        loss, grad, lsize, gsize = ref.distill(z, index, top, lse=lse)
        x = octaves(z, 1.0)
        close(got.loss, loss, lsize, 3 * x + 362 / 64 + 20, "loss")
        close(got.grad, grad, gsize, 5 * x + 362 / 64 + 20, "grad")
        assert rows.stride(0) == net.row_len and torch.equal(rows.cpu(), z)
