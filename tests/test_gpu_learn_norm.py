"""Group norm with an activation on the GPU, forward and backward, against its definition in float64 (tests/learn_ref.py).

Bounds, with K U the relative error of a sum over a group (a thread's own sequence of N / 64 terms or fewer, its joins, and
the few operations around it): mean is off by K U (|mean| + the largest deviation), rstd by K U relative, the normalised value
by K U (1 + |xh|), and what is multiplied to it by the same again; the result's rounding to its type comes on top. act and its
slope are at most 1.1 in slope; the float exponentials inside are off by 8 U of their result."""

import importlib

import pytest
import torch

import learn_ref as ref

pytestmark = pytest.mark.gpu
U = ref.U


@pytest.fixture(scope="module")
def learn():
    return importlib.import_module("katago-rs_amd.learn")


def _close(got, want, size, k, name):
    eps, least = ref.half_step(got.dtype)
    got = got.detach().cpu().double().reshape(want.shape)
    assert torch.isfinite(got).all(), name
    err, bound = (got - want).abs(), eps * want.abs() + least + k * U * size
    assert (err <= bound).all(), (name, int((err > bound).sum()), float((err / bound).max()))


def _case(learn, b, points, c, groups, dtype, act, mask, seed, affine=True, shift=1.0, ld=None, edit=None):
    g = torch.Generator().manual_seed(seed)
    shape = (b, *points, c) if isinstance(points, tuple) else (b, points, c)
    wide = torch.randn(*shape[:-1], c if ld is None else ld, generator=g)
    x = (wide * 1.5 + shift * torch.randn(c, generator=g).repeat(2)[:1]).to(dtype)
    dy = torch.randn(*shape[:-1], c if ld is None else ld, generator=g).to(dtype)
    gamma = 1 + 0.3 * torch.randn(c, generator=g) if affine else None
    beta = 0.5 * torch.randn(c, generator=g) if affine else None
    mk = (torch.rand(shape[:-1], generator=g) < 0.7).float() if mask else None
    if edit:
        edit(x, dy, mk)
    dev = lambda t: None if t is None else t.cuda()  # noqa: E731
    xd, dyd = x.cuda()[..., :c], dy.cuda()[..., :c]
    x, dy = x[..., :c], dy[..., :c]
    y, mean, rstd = learn.group_norm(xd, groups, dev(gamma), dev(beta), mask=dev(mk), eps=1e-5, act=act)
    wy, wm, wr = ref.group_norm(x, groups, gamma, beta, mk, 1e-5, act)
    n = shape[1:-1].numel() if hasattr(shape[1:-1], "numel") else 1
    for s in shape[1:-1]:
        n *= s
    k = n * (c // groups) / 64 + 64
    on = torch.ones(b, n, 1, dtype=torch.bool) if mk is None else (mk.reshape(b, n, 1) != 0)
    xz = torch.where(on, x.double().reshape(b, n, c), 0.0).reshape(b, n, groups, -1)
    dev_max = torch.where(on[..., None], (xz - wm[:, None, :, None]).abs(), 0.0).amax((1, 3))
    _close(mean, wm, wm.abs() + dev_max, k, "mean")
    # (A group of one value has no deviation: what rounding leaves of it is below U times the value, squared.)
    _close(rstd, wr, wr * (1 + (wr * U * 8 * (wm.abs() + dev_max)) ** 2 / U), k, "rstd")
    gm = torch.ones(c).double() if gamma is None else gamma.double()
    bt = torch.zeros(c).double() if beta is None else beta.double()
    xh = ((xz - wm[:, None, :, None]) * wr[:, None, :, None])
    far = ((wm.abs() + dev_max) * wr)[:, None, :, None]  # |x| in units of the deviation
    a_size = ((1 + xh.abs() + far).reshape(b, n, c) * gm.abs() + bt.abs())
    _close(y.reshape(b, n, c), wy, 1.1 * a_size, k + 16, "y")
    assert torch.all(y.reshape(b, n, c)[~on.squeeze(-1).cuda()] == 0)

    dx, dgamma, dbeta = learn.group_norm_backward(dyd, xd, mean, rstd, groups, dev(gamma), dev(beta), mask=dev(mk), act=act)
    stats = (mean.cpu(), rstd.cpu())
    wdx, wdg, wdb = ref.group_norm(x, groups, gamma, beta, mk, 1e-5, act, dy, stats)
    # da's own error: the slope changes by at most 1.1 per unit of its argument. ReLU: not at all for float inputs, whose side of
    # 0 is decided in double; with 16-bit inputs the argument is computed in float, from a difference, two products and a sum
    # (4 U of terms whose sizes a_size adds up), so below 8 U a_size either side is right and da is off by at most dy.
    dyz = torch.where(on, dy.double().reshape(b, n, c), 0.0).abs()
    da_size = dyz * (1.2 + 1.1 * a_size)
    if act == "relu" and dtype != torch.float32:
        a = xh.reshape(b, n, c) * gm + bt
        da_size = da_size + torch.where(on & (a.abs() < 8 * U * a_size), dyz, 0.0) / (k * U)
    xa = xh.abs().reshape(b, n, c)
    _close(dgamma, wdg, (da_size * (xa + far.expand(-1, -1, -1, c // groups).reshape(b, -1, c) + 1)).sum((0, 1)), k * b ** 0 + 64, "dgamma")
    _close(dbeta, wdb, da_size.sum((0, 1)), k + 64, "dbeta")
    d4 = (da_size * gm.abs()).reshape(b, n, groups, -1)
    cnt = (on.sum(1).double() * (c // groups)).clamp(min=1)[:, :, None, None]
    m1 = d4.sum((1, 3), keepdim=True) / cnt
    m2 = (d4 * xh.abs()).sum((1, 3), keepdim=True) / cnt
    size = wr[:, None, :, None] * (d4 + m1 + (xh.abs() + far) * m2 + far * m2)
    _close(dx.reshape(b, n, c), wdx, size.reshape(b, n, c), k + 64, "dx")
    assert torch.all(dx.reshape(b, n, c)[~on.squeeze(-1).cuda()] == 0)


SHAPES = [(1, 1, 1, 1), (2, 1, 8, 2), (3, 5, 3, 3), (2, 361, 384, 32), (3, 361, 128, 8), (2, 361, 75, 5), (1, 300, 25, 5), (2, 70, 44, 4),
          (5, 33, 1024, 64), (2, 9, 2056, 8), (1, 40, 4100, 1), (1, 13, 2048, 2048), (2, 4096, 16, 2), (1, 9001, 2, 1), (70, 7, 30, 3),
          (2, 50, 96, 96), (1, 20011, 7, 7),
          # Rows in shares, columns that are not whole, groups wider than a share's workgroup joins.
          (2, 5000, 96, 4), (1, 12001, 45, 3), (2, 16385, 33, 1), (1, 30000, 20, 4), (2, 700, 500, 1), (2, 700, 1000, 1), (3, 50, 17, 1),
          # More workgroups than CUs: four points a thread.
          (40, 37, 189, 21), (300, 3, 33, 1), (270, 1, 40, 2)]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_group_norm_shapes(learn, shape, dtype):
    b, p, c, g = shape
    for i, (act, mask) in enumerate([("identity", False), ("mish", True), ("silu", False)]):
        _case(learn, b, p, c, g, dtype, act, mask, 7 * i + b + p, affine=i > 0, ld=c + i)


@pytest.mark.parametrize("act", ["identity", "relu", "mish", "silu"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_group_norm_activations_on_boards(learn, act, dtype):
    _case(learn, 3, (19, 19), 96, 8, dtype, act, True, 3)


def test_group_norm_far_mean_and_masked_values(learn):
    def edit(x, dy, mk):
        x += 300.0                     # a mean of hundreds of deviations
        mk[1] = 0                      # a row without a point
        mk[2] = 0
        mk[2, 17] = 1                  # one point
        off = mk == 0
        x[off], dy[off] = torch.nan, torch.inf   # masked points may hold anything
    _case(learn, 4, 361, 48, 6, torch.float32, "mish", True, 5, edit=edit)


def test_group_norm_empty(learn):
    x = torch.zeros(0, 9, 8, device="cuda")
    y, mean, rstd = learn.group_norm(x, 2)
    assert y.shape == (0, 9, 8) and mean.shape == (0, 2)
    dx, dg, db = learn.group_norm_backward(x, x.clone(), mean, rstd, 2)
    assert dx.shape == (0, 9, 8) and torch.all(dg == 0) and torch.all(db == 0)
    x = torch.zeros(3, 0, 8, device="cuda")
    y, mean, rstd = learn.group_norm(x, 2, eps=0.25)
    assert torch.all(mean == 0) and torch.all(rstd == 2)
    _, dg, db = learn.group_norm_backward(x.clone(), x, mean, rstd, 2)
    assert torch.all(dg == 0) and torch.all(db == 0)


def test_group_norm_backward_is_the_slope(learn):
    """Central differences of sum(y dy) in x and gamma: second-order error h^2 / 6 times a third derivative below 40, and the
    rounding of sums of 40 values near 1 over 2 h."""
    g = torch.Generator().manual_seed(2)
    x, dy = torch.randn(2, 5, 4, generator=g).cuda(), torch.randn(2, 5, 4, generator=g).cuda()
    gm, bt = (1 + 0.2 * torch.randn(4, generator=g)).cuda(), torch.randn(4, generator=g).cuda()
    call = lambda x, gm: (learn.group_norm(x, 2, gm, bt, act="mish")[0].double() * dy.double()).sum()  # noqa: E731
    _, mean, rstd = learn.group_norm(x, 2, gm, bt, act="mish")
    dx, dg, _ = learn.group_norm_backward(dy, x, mean, rstd, 2, gm, bt, act="mish")
    h = 2.0 ** -6
    bound = 40 * h * h / 6 + 40 * 16 * U / (2 * h)
    for i in range(x.numel()):
        e = torch.zeros_like(x)
        e.view(-1)[i] = h
        assert abs(float((call(x + e, gm) - call(x - e, gm)) / (2 * h)) - float(dx.view(-1)[i])) <= bound
    for i in range(4):
        e = torch.zeros_like(gm)
        e[i] = h
        assert abs(float((call(x, gm + e) - call(x, gm - e)) / (2 * h)) - float(dg[i])) <= bound


def test_group_norm_captured_and_on_another_stream(learn):
    g = torch.Generator().manual_seed(4)
    xs = [torch.randn(3, 361, 64, generator=g).bfloat16().cuda() for _ in range(3)]
    dy = torch.randn(3, 361, 64, generator=g).bfloat16().cuda()
    gm = torch.rand(64, device="cuda")

    def both(x):
        y, mean, rstd = learn.group_norm(x, 8, gm, act="silu")
        return [y, mean, rstd, *learn.group_norm_backward(dy, x, mean, rstd, 8, gm, act="silu")]

    want = [[t.clone() for t in both(x)] for x in xs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = both(xs[2])
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want[2]))
    graphs = []
    for _ in range(2):
        buf = xs[0].clone()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = both(buf)
        graphs.append((gr, buf, out))
    for k in range(3):
        for j, (gr, buf, out) in enumerate(graphs):
            buf.copy_(xs[(k + j) % 3])
        for gr, _, _ in graphs:
            gr.replay()
        eager = both(xs[k])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(eager, want[k]))
        for j, (_, _, out) in enumerate(graphs):
            assert all(torch.equal(a, b) for a, b in zip(out, want[(k + j) % 3]))


def test_group_norm_refuses_on_the_gpu(learn):
    x = torch.randn(2, 9, 12, device="cuda")
    KgError = importlib.import_module("katago-rs_amd").KgError
    with pytest.raises(KgError, match="multiple of groups"):
        learn.group_norm(x, 5)
    with pytest.raises(KgError, match="overlap"):
        learn.group_norm(x, 3, y=x)
    with pytest.raises(KgError, match="eps"):
        learn.group_norm(x, 3, eps=0.0)
    with pytest.raises(ValueError, match="act"):
        learn.group_norm(x, 3, act="tanh")
    with pytest.raises(ValueError, match="mask"):
        learn.group_norm(x, 3, mask=torch.ones(2, 8, device="cuda"))
    with pytest.raises(ValueError, match="gamma"):
        learn.group_norm(x, 3, torch.ones(12, device="cuda").half())
    with pytest.raises(ValueError, match="mean"):
        learn.group_norm_backward(x, x.clone(), torch.zeros(2, 4, device="cuda"), torch.zeros(2, 3, device="cuda"), 3)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shape", [(40, 361, 45, 3), (6, 9000, 27, 3), (64, 81, 250, 2)])
def test_group_norm_again_is_the_same(learn, shape, dtype):
    """Widths whose last column of 16 bytes is not whole: two threads compute its first channels, and both store them."""
    b, p, c, groups = shape
    g = torch.Generator(device="cuda").manual_seed(9)
    x, dy = (torch.randn(b, p, c, generator=g, device="cuda").to(dtype) for _ in range(2))
    gm, bt = (torch.randn(c, generator=g, device="cuda") for _ in range(2))
    for act in ("mish", "silu"):
        first = None
        for _ in range(8):
            y, mean, rstd = learn.group_norm(x, groups, gm, bt, act=act)
            got = [y, mean, rstd, *learn.group_norm_backward(dy, x, mean, rstd, groups, gm, bt, act=act)]
            first = first or got
            assert all(torch.equal(a, b) for a, b in zip(got, first))
