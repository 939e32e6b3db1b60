"""The policy and preference losses on the GPU against their definitions in float64 (tests/learn_ref.py).

Bounds. A softmax term exp((z - top) s) computed in float is off, relative, by the rounding of its exponent (the difference, the
product and the factor log2 e: 3 U X with X the largest exponent in use, in octaves) and by the exponential itself (a float ulp,
2 U); a sum of V terms over at least 64 threads adds U (V / 64 + 12). K U = (3 X + V / 64 + 20) U bounds the relative error of a
probability, its sum and the other factors of a gradient (a few roundings); logp takes the sum's error, absolutely; the result's
own rounding to its type comes on top. The sides of the clip are decided in double, and no ratio of these inputs lies within 1e-5
of its border (asserted)."""

import importlib
import math

import numpy as np
import pytest
import torch

import learn_ref as ref

pytestmark = pytest.mark.gpu
U = ref.U


@pytest.fixture(scope="module")
def learn():
    return importlib.import_module("katago-rs_amd.learn")


def _k(z, scale, columns, legal=None):
    zz = z.double().clone()
    if legal is not None:
        zz[~legal.bool()] = -torch.inf
    zz[~torch.isfinite(zz)] = math.nan
    span = (zz.nan_to_num(nan=-torch.inf).max(1).values - zz.nan_to_num(nan=torch.inf).min(1).values).nan_to_num(0, 0, 0)
    x = float((span * scale * 1.4427).clamp(max=150).max()) if span.numel() else 0.0
    return 3 * max(x, 0) + columns / 64 + 20


def _close(got, want, size, k, name):
    """|got - want| <= half a step of got's type + k U size."""
    eps, least = ref.half_step(got.dtype)
    got, same = got.cpu().double(), None
    fine = torch.isfinite(want)
    assert torch.equal(torch.isfinite(got), fine), name
    assert torch.equal(got[~fine], want[~fine]), name
    err, bound = (got - want).abs()[fine], (eps * want.abs() + least + k * U * size)[fine]
    bad = err > bound
    assert not bad.any(), (name, int(bad.sum()), float((err / bound.clamp(min=1e-300)).max()), same)


def _inputs(n, v, dtype, seed, ld=None, shift=0, spread=2.0):
    g = torch.Generator().manual_seed(seed)
    ld = v if ld is None else ld
    full = (torch.randn(n, ld + shift, generator=g) * spread).to(dtype)
    return g, full


def _policy_case(learn, n, v, dtype, kl, legal, seed, ld=None, shift=0, scale=1.0, edit=None, grad_ld=0, kl_coef=0.3):
    g, full = _inputs(n, v, dtype, seed, ld, shift)
    z = full[:, shift:shift + v]
    actions = torch.randint(0, v, (n,), generator=g, dtype=torch.int32)
    mask = None
    if legal:
        mask = torch.rand(n, v, generator=g) < 0.6
        mask.scatter_(1, actions[:, None].long(), True)
    refl = (z.float() + 0.4 * torch.randn(n, v, generator=g)).to(dtype) if kl == "full" else None
    adv, weight = torch.randn(n, generator=g), torch.rand(n, generator=g)
    lp = ref.log_softmax(z.double() * scale, mask)[torch.arange(n), actions.long()]
    old = (lp + 0.25 * torch.randn(n, generator=g)).float()
    rlp = (lp + 0.5 * torch.randn(n, generator=g)).float() if kl == "estimate" else None
    if edit:
        edit(z, actions, mask, refl)
    lp = ref.log_softmax(z.double() * scale, mask)[torch.arange(n), actions.long().clamp(0, v - 1)]
    for border in (math.log(0.8), math.log(1.3)):
        assert not ((lp - old.double() - border).abs() < 1e-5).any()
    want = ref.policy(z, actions, old, adv, mask, weight, scale, (0.2, 0.3), kl_coef, refl, rlp)
    d = full.cuda()
    dev = lambda t: None if t is None else t.cuda()  # noqa: E731
    grad = None
    if grad_ld:
        grad = torch.full((n, v + grad_ld), 7.0, dtype=dtype, device="cuda")
    got = learn.policy_loss(d[:, shift:shift + v], dev(actions), dev(old), dev(adv), legal=dev(mask), weight=dev(weight),
                            logit_scale=scale, clip=(0.2, 0.3), kl_coef=kl_coef, ref_logits=dev(refl), ref_logp=dev(rlp),
                            grad=None if grad is None else grad[:, 1:1 + v])
    k = _k(z, scale, v, mask) + (_k(refl, scale, v, mask) if kl == "full" else 0)
    loss, logp, klw, gw, size = want
    _close(got.logp, logp, torch.ones(n), k, "logp")
    # kl: sums of p |log p/r| (estimate: of e^d and d), each off by K U; the loss adds the ratio's part.
    ksize = (klw.abs() + 2) * 2 if kl != "estimate" else torch.exp((rlp.double() - logp).clamp(-50, 50)).nan_to_num(0, 0, 0) + 10
    _close(got.kl, klw, ksize, k, "kl")
    ratio = torch.exp((logp - old.double()).clamp(-50, 50)).nan_to_num(0, 0, 0)
    _close(got.loss, loss, weight * (ratio * adv.abs() + kl_coef * ksize), k, "loss")
    _close(got.grad, gw, size * (1 + (torch.exp((rlp.double() - logp).clamp(-50, 50)).nan_to_num(0, 0, 0)[:, None] if rlp is not None else 0)),
           k, "grad")
    if grad is not None:
        assert torch.all(grad[:, 0] == 7) and torch.all(grad[:, 1 + v:] == 7)
    return got


WIDTHS = [1, 2, 3, 7, 8, 9, 63, 65, 361, 362, 363, 511, 1025, 2048, 2049, 4097, 8193, 16384, 16385, 33001, 65537, 131073]


@pytest.mark.parametrize("v", WIDTHS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_policy_loss_widths(learn, v, dtype):
    for i, (kl, legal) in enumerate([("none", False), ("estimate", True), ("full", False), ("full", True)]):
        _policy_case(learn, 5 if v < 5000 else 2, v, dtype, kl, legal, 100 * v + i, ld=v + i, shift=i)


@pytest.mark.parametrize("v,dtype,kl,legal", [(16500, torch.float32, "full", True), (41001, torch.float32, "estimate", False),
                                              (33001, torch.bfloat16, "full", False), (33001, torch.float16, "none", True)])
def test_policy_loss_many_long_rows(learn, v, dtype, kl, legal):
    """More long rows than are cut into parts, and one fewer than that."""
    for n in (385, 384):
        _policy_case(learn, n, v, dtype, kl, legal, n + v)


def test_policy_loss_few_long_rows_captured(learn):
    """Rows cut into parts, two captured calls with a workspace each, replayed in turn."""
    g = torch.Generator(device="cuda").manual_seed(1)
    n, v = 3, 70001
    zs = [torch.randn(n, v, generator=g, device="cuda").bfloat16() for _ in range(3)]
    refl = torch.randn(n, v, generator=g, device="cuda").bfloat16()
    act = torch.tensor([5, -1, 70000], dtype=torch.int32, device="cuda")
    old, adv = torch.full((n,), -11.0, device="cuda"), torch.tensor([1.0, 2.0, -1.0], device="cuda")

    def call(z):
        return list(learn.policy_loss(z, act, old, adv, kl_coef=0.2, ref_logits=refl))

    want = [[t.clone() for t in call(z)] for z in zs]
    graphs = []
    for _ in range(2):
        buf = zs[0].clone()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = call(buf)
        graphs.append((gr, buf, out))
    for k in range(3):
        for j, (gr, buf, _) in enumerate(graphs):
            buf.copy_(zs[(k + j) % 3])
            gr.replay()
        torch.cuda.synchronize()
        for j, (_, _, out) in enumerate(graphs):
            assert all(torch.equal(a, b) for a, b in zip(out, want[(k + j) % 3]))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_policy_loss_rows_temperature_and_strided_gradient(learn, dtype):
    for n in (1, 3, 4, 61):
        _policy_case(learn, n, 362, dtype, "full", True, n, ld=1094, scale=0.7, grad_ld=3)
        _policy_case(learn, n, 2500, dtype, "estimate", False, 50 + n, scale=1.9, grad_ld=2)


@pytest.mark.parametrize("v", [362, 3001, 20001, 70001])
def test_policy_loss_masks_and_values(learn, v):
    def edit(z, actions, legal, refl):
        actions[0], actions[1], actions[2] = -1, v, 2 ** 31 - 1   # padding
        legal[3, actions[3]] = False                              # an illegal action
        legal[4] = False                                          # no legal move
        z[5, :] = -torch.inf                                      # nothing possible
        z[6, actions[6]] = -torch.inf                             # the action alone impossible
        z[7, ~legal[7]] = torch.nan                               # what illegal columns hold does not matter
        refl[7, ~legal[7]] = torch.inf
        z[8, ~legal[8]] = torch.finfo(torch.float32).max
        z[9, :] = torch.finfo(torch.float32).min                  # a mask of the lowest value everywhere: uniform
        refl[9, :] = 0
        z[10, (torch.arange(v) % 3 == 0) & (torch.arange(v) != actions[10])] = torch.finfo(torch.float32).min
        z[11, :] += 5000.0                                        # far from 0
        refl[11, :] += 5000.0
        keep = actions[12]
        legal[12] = False
        legal[12, keep] = True                                    # one legal move
        z[13, (torch.arange(v) % 2 == 0) & (torch.arange(v) != actions[13])] = -torch.inf  # impossible ones, with a reference
    got = _policy_case(learn, 14, v, torch.float32, "full", True, v, edit=edit)
    assert torch.equal(got.logp[:3].cpu(), torch.zeros(3)) and torch.all(got.logp[3:7].cpu() == -torch.inf)
    for t in (got.loss, got.kl):
        assert torch.all(t[:7] == 0)
    assert torch.all(got.grad[:7] == 0) and abs(float(got.logp[12])) == 0


def test_policy_loss_nan_stays_in_its_row(learn):
    z = torch.randn(3, 362, device="cuda")
    z[1, 40] = torch.nan
    a = torch.zeros(3, dtype=torch.int32, device="cuda")
    r = learn.policy_loss(z, a, torch.full((3,), -6.0, device="cuda"), torch.ones(3, device="cuda"))
    assert torch.isnan(r.loss).tolist() == [False, True, False] and torch.isnan(r.logp).tolist() == [False, True, False]
    assert torch.isnan(r.grad[1]).all() and torch.isfinite(r.grad[[0, 2]]).all()


def test_policy_loss_without_gradient_and_without_rows(learn):
    z = torch.randn(7, 362, device="cuda")
    a, f = torch.zeros(7, dtype=torch.int32, device="cuda"), torch.randn(7, device="cuda")
    full = learn.policy_loss(z, a, f, f)
    part = learn.policy_loss(z, a, f, f, want_grad=False)
    assert part.grad is None and torch.equal(part.loss, full.loss)
    none = learn.policy_loss(z[:0], a[:0], f[:0], f[:0])
    assert none.loss.shape == (0,) and none.grad.shape == (0, 362)


def test_policy_gradient_is_the_slope_of_the_loss(learn):
    """Central differences of the returned losses, on few columns: the step's error is of second order (h^2 / 6 times the third
    derivative, below 10 here) and the losses' own rounding (a few U of values near 1) is divided by 2 h."""
    n, v, h = 6, 5, 2.0 ** -7
    g = torch.Generator().manual_seed(5)
    z, adv = torch.randn(n, v, generator=g).cuda(), torch.randn(n, generator=g).cuda()
    refl, a = torch.randn(n, v, generator=g).cuda(), torch.arange(n, dtype=torch.int32, device="cuda") % v
    old = torch.log_softmax(z, 1)[torch.arange(n), a.long()] + 0.02
    call = lambda t: learn.policy_loss(t, a, old, adv, kl_coef=0.5, ref_logits=refl)  # noqa: E731
    grad = call(z).grad
    for j in range(v):
        d = torch.zeros(v, device="cuda")
        d[j] = h
        slope = (call(z + d).loss.double() - call(z - d).loss.double()) / (2 * h)
        assert torch.all((slope - grad[:, j].double()).abs() <= 10 * h * h / 6 + 32 * U * 4 / (2 * h))


def _preference_case(learn, lens, v, dtype, average, seed, ld=None, shift=0, before=0, behind=0, smooth=0.1, edit=None, grad_ld=0):
    t = before + sum(lens) + behind
    g, full = _inputs(t, v, dtype, seed, ld, shift)
    z = full[:, shift:shift + v]
    labels = torch.randint(0, v, (t,), generator=g, dtype=torch.int32)
    if t:
        labels[torch.rand(t, generator=g) < 0.2] = -1
    if edit:
        edit(z, labels)
    offsets = torch.tensor([before] + lens).cumsum(0).to(torch.int32)
    pairs = len(lens) // 2
    lp = ref.log_softmax(z) if t else z.double()
    seq = []
    for q in range(2 * pairs):
        rows = [i for i in range(int(offsets[q]), int(offsets[q + 1])) if 0 <= int(labels[i]) < v]
        s = sum(float(lp[i, int(labels[i])]) for i in rows)
        seq.append(s / max(1, len(rows)) if average else s)
    rlp = (torch.tensor(seq, dtype=torch.float64) + torch.randn(2 * pairs, generator=g)).float()
    weight = torch.rand(pairs, generator=g) + 0.5
    loss, margin, want_seq, gw, size = ref.preference(z, labels, offsets, rlp, 0.4, smooth, average, weight)
    grad = torch.full((t, v + grad_ld), 7.0, dtype=dtype, device="cuda") if grad_ld else None
    got = learn.preference_loss(full.cuda()[:, shift:shift + v], labels.cuda(), offsets.cuda(), rlp.cuda(), beta=0.4,
                                label_smoothing=smooth, average=average, weight=weight.cuda(),
                                grad=None if grad is None else grad[:, :v])
    k = _k(z, 1.0, v) if t else 1.0
    count = max(lens) if lens and not average else 1
    _close(got.seq_logp, want_seq, torch.full((2 * pairs,), float(count)), k, "seq_logp")
    _close(got.margin, margin, 0.8 * torch.full((pairs,), float(count)), k, "margin")
    _close(got.loss, loss, weight * 0.8 * count, k, "loss")
    _close(got.grad, gw, size * (1 + 0.8 * count), k, "grad")
    if grad is not None:
        assert torch.all(grad[:, v:] == 7)
    return got, offsets, labels


@pytest.mark.parametrize("v", [1, 2, 9, 362, 2049, 16385, 40001, 131073])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_preference_loss_widths(learn, v, dtype):
    lens = [3, 5, 0, 2] if v < 5000 else [2, 1]
    for average in (False, True):
        _preference_case(learn, lens, v, dtype, average, v, ld=v + 3, shift=1, before=1, behind=2)


@pytest.mark.parametrize("lens", [[], [0, 0], [1, 0], [0, 1], [1, 1], [400, 3], [3, 300, 0, 0, 17, 1], [2] * 130])
def test_preference_loss_lengths(learn, lens):
    for average in (False, True):
        got, offsets, labels = _preference_case(learn, lens, 362, torch.float32, average, 9, ld=1094, before=2, behind=3, grad_ld=1)
        out = torch.ones(len(labels), dtype=torch.bool)
        out[int(offsets[0]):int(offsets[-1])] = labels[int(offsets[0]):int(offsets[-1])] < 0
        assert torch.all(got.grad.cpu()[out] == 0)


@pytest.mark.parametrize("v,dtype", [(33001, torch.bfloat16), (16500, torch.float32)])
def test_preference_loss_many_long_rows(learn, v, dtype):
    """More long rows than are cut into parts (129), and as many as are."""
    for lens in ([70, 54], [70, 53]):
        _preference_case(learn, lens, v, dtype, False, v, before=3, behind=2)


def test_preference_loss_values(learn):
    v = 700

    def edit(z, labels):
        z[0] += 3000.0
        z[1] = torch.finfo(torch.float32).min
        z[2, torch.arange(v) != 5] = -torch.inf   # one possible token
        labels[0], labels[1], labels[2], labels[3], labels[4] = 3, 4, 5, v, -7
        z[3] = torch.nan                          # rows that are not counted may hold anything
    _preference_case(learn, [4, 3], v, torch.float32, False, 4, edit=edit)


def test_preference_large_margins_saturate(learn):
    """A margin far from 0: the loss is its size on one side and 0 on the other, and no exponential overflows."""
    z = torch.zeros(2, 4, device="cuda")
    lab, off = torch.zeros(2, dtype=torch.int32, device="cuda"), torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    for sign in (1.0, -1.0):
        r = learn.preference_loss(z, lab, off, torch.tensor([-sign * 4000.0, sign * 4000.0], device="cuda"), beta=1.0)
        assert abs(float(r.margin) - sign * 8000.0) <= 1e-3 and float(r.loss) == (0.0 if sign > 0 else float(-r.margin))
        assert torch.isfinite(r.grad).all() and (sign < 0 or torch.all(r.grad == 0))


def test_preference_offsets_out_of_range_stay_inside(learn):
    z = torch.randn(5, 40, device="cuda")
    lab = torch.zeros(5, dtype=torch.int32, device="cuda")
    r = learn.preference_loss(z, lab, torch.tensor([-9, 2, 400], dtype=torch.int32, device="cuda"), torch.zeros(2, device="cuda"))
    want = ref.preference(z.cpu(), lab.cpu(), [0, 2, 5], torch.zeros(2))
    _close(r.grad, want[3], want[4] * 2, _k(z.cpu(), 1.0, 40), "grad")


def test_rows_past_2_31_elements(learn):
    """Row offsets of more than 31 bits: the last rows equal the same rows among fewer, bit for bit. (Among 400: fewer long rows
    are cut into parts, whose sums are added in another order.)"""
    n, v, few = 66000, 33000, 400
    z = torch.zeros(n, v, dtype=torch.bfloat16, device="cuda")
    tail = torch.randn(8, v, device="cuda").bfloat16()
    z[-8:] = tail
    act = torch.full((n,), -1, dtype=torch.int32, device="cuda")
    act[-8:] = torch.arange(8, dtype=torch.int32, device="cuda") * 4000
    f = torch.full((n,), -10.0, device="cuda")
    got = learn.policy_loss(z, act, f, f, grad=None)
    small = torch.zeros(few, v, dtype=torch.bfloat16, device="cuda")
    small[-8:] = tail
    alone = learn.policy_loss(small, act[-few:].clone(), f[:few], f[:few])
    assert torch.equal(got.grad[-8:], alone.grad[-8:]) and torch.equal(got.loss[-8:], alone.loss[-8:]) and not got.grad[:100].any()
    del got
    off = torch.tensor([n - 8, n - 3, n], dtype=torch.int32, device="cuda")
    lab = act.clone()
    p = learn.preference_loss(z, lab, off, torch.zeros(2, device="cuda"))
    q = learn.preference_loss(small, lab[-few:].clone(), off - (n - few), torch.zeros(2, device="cuda"))
    assert torch.equal(p.grad[-8:], q.grad[-8:]) and torch.equal(p.loss, q.loss)


def test_losses_on_another_stream_and_captured(learn):
    """Captured calls read new inputs at each replay, two graphs side by side keep their own workspaces, and a call on another
    stream than the tensors' gives the same bits."""
    g = torch.Generator().manual_seed(1)
    n, v = 33, 362
    zs = [torch.randn(n, v, generator=g).cuda() for _ in range(4)]
    act = torch.randint(0, v, (n,), generator=g, dtype=torch.int32).cuda()
    f = torch.full((n,), -6.0, device="cuda")
    off = torch.tensor([0, 7, 19, 19, 30], dtype=torch.int32, device="cuda")
    rlp = torch.full((4,), -60.0, device="cuda")

    def both(z):
        p = learn.policy_loss(z, act, f, f)
        q = learn.preference_loss(z, act, off, rlp)
        return [*p, *q]

    want = [[t.clone() for t in both(z)] for z in zs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = both(zs[1])
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(other, want[1]))
    graphs = []
    for _ in range(2):
        buf = zs[0].clone()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = both(buf)
        graphs.append((gr, buf, out))
    for k in range(4):
        for j, (gr, buf, out) in enumerate(graphs):
            buf.copy_(zs[(k + j) % 4])
        for gr, _, _ in graphs:
            gr.replay()
        eager = both(zs[k])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(eager, want[k]))
        for j, (_, _, out) in enumerate(graphs):
            assert all(torch.equal(a, b) for a, b in zip(out, want[(k + j) % 4])), (k, j)


def test_losses_refuse_on_the_gpu(learn):
    z = torch.randn(4, 10, device="cuda")
    a, f = torch.zeros(4, dtype=torch.int32, device="cuda"), torch.zeros(4, device="cuda")
    KgError = importlib.import_module("katago-rs_amd").KgError
    with pytest.raises(ValueError, match="actions"):
        learn.policy_loss(z, a.long(), f, f)
    with pytest.raises(ValueError, match="old_logp"):
        learn.policy_loss(z, a, f.cpu(), f)
    with pytest.raises(ValueError, match="legal"):
        learn.policy_loss(z, a, f, f, legal=torch.ones(4, 9, dtype=torch.bool, device="cuda"))
    with pytest.raises(ValueError, match="ref_logits"):
        learn.policy_loss(z, a, f, f, ref_logits=z.half())
    with pytest.raises(KgError, match="not both"):
        learn.policy_loss(z, a, f, f, ref_logits=z.clone(), ref_logp=f)
    with pytest.raises(KgError, match="row stride"):
        learn.policy_loss(z[:1].expand(4, 10), a, f, f)
    with pytest.raises(KgError, match="overlap"):
        learn.policy_loss(z, a, f, f, grad=z)
    with pytest.raises(ValueError, match="odd length"):
        learn.preference_loss(z, a, a, f)
    with pytest.raises(ValueError, match="labels"):
        learn.preference_loss(z, a[:3], torch.zeros(3, dtype=torch.int32, device="cuda"), f[:2])
    assert np.isfinite(learn.policy_loss(z, a, f, f).loss.cpu().numpy()).all()
