"""The distillation loss on the GPU against its definition in float64 (tests/student_ref.py).

Bounds. The columns that are not listed are summed in float: a term exp((z - top) s) is off, relative, by the rounding of its
exponent (3 U X with X the largest exponent in use, in octaves) and by the exponential (2 U); a sum of V terms over at least 64
threads adds U (V / 64 + 12). K U = (3 X + V / 64 + 20) U bounds the relative error of that sum, of R and of every probability
(the rest is double, a listed column's exponent too). The gradient's own exponentials have log2 e in one float, 2 U X more.
A result's rounding to its type comes on top."""

import importlib
import math

import pytest
import torch

import learn_ref
import student_ref as ref

pytestmark = pytest.mark.gpu
U = learn_ref.U
TYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.fixture(scope="module")
def learn():
    return importlib.import_module("katago-rs_amd.learn")


def octaves(z, scale, legal=None):
    """The largest span of a row's finite legal logits, in octaves of its probabilities, cut where a float's end."""
    on = torch.isfinite(z) if legal is None else torch.isfinite(z) & legal.bool()
    z = z.double()
    high = torch.where(on, z, -math.inf).max(1).values
    low = torch.where(on, z, math.inf).min(1).values
    span = ((high - low) * scale * 1.4427).clamp(0, 150)
    return float(span.max())


def close(got, want, size, k, name):
    """|got - want| <= half a step of got's type + k U size; infinite and NaN in the same places."""
    eps, least = learn_ref.half_step(got.dtype)
    got = got.cpu().double()
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), name
    assert torch.equal(got[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)]), name
    err, bound = (got - want).abs()[fine], (eps * want.abs() + least + k * U * size)[fine]
    assert not (err > bound).any(), (name, int((err > bound).sum()), float((err / bound.clamp(min=1e-300)).max()))


def make(n, v, k, dtype, top_type, seed, legal=False, rest=False, scale=1.0, ld=0, spread=2.0):
    g = torch.Generator().manual_seed(seed)
    full = (torch.randn(n, v + ld, generator=g) * spread).to(dtype)
    z = full[:, ld // 2:ld // 2 + v]
    teacher = z.float() + 0.7 * torch.randn(n, v, generator=g)
    mask = None
    if legal:
        mask = torch.rand(n, v, generator=g) < 0.6
        mask.scatter_(1, teacher.argmax(1, keepdim=True), True)
    kk = min(k, v)
    top, index = teacher.topk(kk, 1)
    index = torch.cat([index, torch.full((n, k - kk), -1)], 1).int()
    top = torch.cat([top, torch.zeros(n, k - kk)], 1).to(top_type)
    order = torch.randperm(k, generator=g)
    index, top = index[:, order].contiguous(), top[:, order].contiguous()
    lse = None
    if rest:
        # The stored logits are rounded: a normaliser of all columns with them in place.
        t = teacher.double()
        t.scatter_(1, index.long().clamp(min=0), torch.where(index >= 0, top.double(), t.gather(1, index.long().clamp(min=0))))
        lse = torch.logsumexp(t * scale, 1).float()
    return {"full": full, "z": z, "index": index, "top": top, "legal": mask, "weight": torch.rand(n, generator=g) + 0.1, "lse": lse,
            "scale": scale, "at": ld // 2}


def run(learn, c, **more):
    dev = {k: t.cuda() if torch.is_tensor(t) else t for k, t in c.items()}
    z = dev["full"][:, c["at"]:c["at"] + c["z"].shape[1]]
    return learn.distill_loss(z, dev["index"], dev["top"], legal=dev["legal"], weight=dev["weight"], logit_scale=c["scale"],
                              teacher_lse=dev["lse"], **more)


def check(learn, c, **more):
    got = run(learn, c, **more)
    loss, grad, lsize, gsize = ref.distill(c["z"], c["index"], c["top"], c["legal"], c["weight"], c["scale"], c["lse"])
    x = octaves(c["z"], c["scale"], c["legal"])
    k = 3 * x + c["z"].shape[1] / 64 + 20
    close(got.loss, loss, lsize, k, "loss")
    if got.grad is not None:
        close(got.grad, grad, gsize, k + 2 * x, "grad")
    return got


WIDTHS = [1, 2, 3, 4, 7, 8, 9, 63, 64, 65, 361, 362, 363, 511, 512, 1023, 1025, 2048, 2049, 4096, 4097, 8191, 16384, 16385, 32768, 32775, 70001]


@pytest.mark.parametrize("v", WIDTHS)
@pytest.mark.parametrize("dtype", TYPES)
def test_widths(learn, v, dtype):
    n = 7 if v < 5000 else 3
    for i, (k, top_type, legal, rest) in enumerate([(1, torch.float32, False, False), (min(v, 24), torch.float16, True, True),
                                                    (64, torch.bfloat16, False, True), (5, torch.float32, True, False)]):
        check(learn, make(n, v, k, dtype, top_type, 10 * v + i, legal, rest, 0.5 if rest else 1.0, ld=2 * i))


@pytest.mark.parametrize("k", [1, 2, 63, 64, 65, 200, 512, 1023, 1024])
@pytest.mark.parametrize("v,dtype", [(1100, torch.float32), (1100, torch.bfloat16), (9000, torch.float32), (40000, torch.float16)])
def test_entries(learn, k, v, dtype):
    check(learn, make(3, v, k, dtype, torch.float32, k, legal=k % 2 == 0, rest=k > 2))


@pytest.mark.parametrize("n", [1, 2, 31, 500, 5000])
def test_rows(learn, n):
    check(learn, make(n, 362, 12, torch.float32, torch.float16, n, True, n % 2 == 0, ld=732))


def test_every_column_listed(learn):
    """Nothing is left for the rest, however the normaliser was rounded."""
    for v in (2, 5, 40, 600):
        for rest in (False, True):
            check(learn, make(6, v, v, torch.float32, torch.float32, v, rest=rest))


def test_rows_that_take_no_part(learn):
    inf = math.inf
    for v, dtype in ((5, torch.float32), (362, torch.bfloat16), (9000, torch.float16), (20000, torch.float32)):
        for rest in (False, True):
            c = make(8, v, 4, dtype, torch.float32, v, legal=True, rest=rest)
            c["legal"][0] = False                      # no legal column
            c["index"][1] = -1                         # padding
            c["index"][2] = torch.tensor([v, -7, 2 ** 31 - 1, -2 ** 31])
            c["legal"][3, c["index"][3].long().clamp(0, v - 1)] = False  # only illegal entries
            c["legal"][3, :] &= True
            c["z"][4] = -inf                           # no mass anywhere
            c["top"][5] = -inf                         # the teacher's mass is elsewhere
            c["legal"][6] = True
            got = check(learn, c)
            for i in (0, 1, 2, 3, 4) + (() if rest else (5,)):
                assert float(got.loss[i]) == 0 and not got.grad[i].any()


def test_masks_and_garbage(learn):
    """Illegal columns may hold anything; masked logits at the type's lowest value; -infinity where a column has no mass."""
    for v, dtype in ((362, torch.float32), (5000, torch.bfloat16), (20001, torch.float16)):
        for rest in (False, True):
            c = make(6, v, 9, dtype, torch.float32, v, legal=True, rest=rest)
            bad = ~c["legal"]
            filler = torch.tensor([math.nan, math.inf, -math.inf, torch.finfo(dtype).max])[torch.arange(6 * v).reshape(6, v) % 4]
            c["z"].copy_(torch.where(bad, filler.to(dtype), c["z"]))
            check(learn, c)
            c = make(6, v, 9, dtype, torch.float32, v + 1, rest=rest)
            others = torch.ones(6, v, dtype=torch.bool).scatter_(1, c["index"].long().clamp(min=0), False)
            c["z"].copy_(torch.where(others & (torch.arange(v) % 3 == 0), -math.inf, c["z"]))
            c["z"][2] = torch.where(others[2], torch.finfo(dtype).min, c["z"][2])
            c["z"][3] = torch.where(others[3], -math.inf, c["z"][3])
            c["z"][4] = torch.where(others[4], c["z"][4], torch.tensor(-30.0, dtype=dtype))
            if rest:
                c["z"][2] = torch.where(others[2], -120.0 + c["z"][2], c["z"][2])  # R past float's least number: 2^-150 and less
            check(learn, c)


def test_listed_without_mass(learn):
    c = make(3, 400, 6, torch.float32, torch.float32, 3)
    c["z"][0, c["index"][0, 2].long()] = -math.inf
    got = check(learn, c)
    assert float(got.loss[0]) == math.inf and torch.isfinite(got.grad[0]).all()
    c["top"][0, 2] = -math.inf  # and the teacher has none there either
    assert math.isfinite(float(check(learn, c).loss[0]))


def test_not_numbers(learn):
    for v in (6, 400, 20000):
        for where in ("listed", "other", "teacher"):
            c = make(3, v, 4, torch.float32, torch.float32, 4)
            others = torch.ones(v, dtype=torch.bool)
            others[c["index"][1].long()] = False
            if where == "teacher":
                c["top"][1, 2] = math.nan
            else:
                c["z"][1, int(others.nonzero()[0]) if where == "other" else int(c["index"][1, 0])] = math.nan
            got = run(learn, c)
            assert math.isnan(float(got.loss[1])) and torch.isnan(got.grad[1]).all()
            c2 = {k: t[::2].contiguous() if torch.is_tensor(t) else t for k, t in c.items()}
            again = check(learn, c2)
            assert torch.equal(got.loss[::2], again.loss) and torch.equal(got.grad[::2], again.grad)


@pytest.mark.parametrize("v", [3, 300, 5000, 40000])
def test_columns_listed_twice(learn, v):
    for seed in range(3):
        c = make(5, v, 40, torch.float32, torch.float32, seed, legal=seed == 1, rest=seed == 2)
        g = torch.Generator().manual_seed(seed)
        c["index"] = c["index"].gather(1, torch.randint(0, 40, (5, 40), generator=g)).contiguous()
        c["index"][4] = c["index"][4, 0].clone()
        if c["lse"] is not None:  # (the first entry of a column has any of the logits: a normaliser above them all)
            c["lse"] = torch.logsumexp(c["top"].double(), 1).float() + 1
        got = check(learn, c)
        for _ in range(3):
            again = run(learn, c)
            assert torch.equal(got.loss, again.loss) and torch.equal(got.grad, again.grad)


def test_scales(learn):
    for scale in (2.0 ** -64, 2.0 ** -7, 0.37, 5.0, 2.0 ** 20):
        for rest in (False, True):
            check(learn, make(4, 700, 8, torch.float32, torch.float32, 9, legal=True, rest=rest, scale=scale))


def test_far_from_zero(learn):
    c = make(4, 500, 8, torch.float32, torch.float32, 9)
    c["z"] += 1e4
    c["top"] -= 3e4
    check(learn, c)


def test_given_gradient_and_none(learn):
    c = make(5, 777, 8, torch.bfloat16, torch.float32, 9)
    whole = torch.full((5, 790), 3.0, dtype=torch.bfloat16, device="cuda")
    got = check(learn, c, grad=whole[:, 3:780])
    assert got.grad.data_ptr() == whole.data_ptr() + 6 and (whole[:, :3] == 3).all() and (whole[:, 780:] == 3).all()
    assert check(learn, c, want_grad=False).grad is None


def test_strided_entries_and_mask(learn):
    c = make(6, 100, 7, torch.float32, torch.float16, 9, legal=True)
    want = run(learn, c)
    index, top = torch.full((6, 11), 5, dtype=torch.int32), torch.full((6, 9), 50.0, dtype=torch.float16)
    legal = torch.ones(6, 107, dtype=torch.uint8)
    index[:, 2:9], top[:, 1:8], legal[:, 4:104] = c["index"], c["top"], c["legal"]
    got = learn.distill_loss(c["z"].cuda(), index.cuda()[:, 2:9], top.cuda()[:, 1:8], legal=legal.cuda()[:, 4:104], weight=c["weight"].cuda())
    assert torch.equal(got.loss, want.loss) and torch.equal(got.grad, want.grad)


def test_no_rows(learn):
    z = torch.zeros(0, 50, device="cuda")
    got = learn.distill_loss(z, torch.zeros(0, 3, dtype=torch.int32, device="cuda"), torch.zeros(0, 3, device="cuda"))
    assert got.loss.shape == (0,) and got.grad.shape == (0, 50)


@pytest.mark.parametrize("rest", [False, True])
def test_differences(learn, rest):
    """The gradient against differences of the definition, 1e-5 either way in float64: off by the third derivative's 1e-10."""
    c = make(3, 50, 6, torch.float32, torch.float32, 21, legal=True, rest=rest, scale=0.7)
    grad = run(learn, c).grad.cpu().double()
    g = torch.Generator().manual_seed(1)
    for _ in range(5):
        d = torch.randn(3, 50, generator=g, dtype=torch.float64)
        up, down = (ref.distill(c["z"].double() + s * d, c["index"], c["top"], c["legal"], c["weight"], 0.7, c["lse"])[0].sum()
                    for s in (1e-5, -1e-5))
        assert abs(float((up - down) / 2e-5) - float((grad * d).sum())) < 1e-5
