"""A student's operators where a number passes a type's range: infinite entries of the teacher's, rows shorter than
16 bytes about a mean near float's largest, rows whose sum float does not hold."""

import importlib
import math

import pytest
import torch

import learn_ref
import test_gpu_distill as distill
import test_gpu_layer_norm as norm

pytestmark = pytest.mark.gpu
U = learn_ref.U


@pytest.fixture(scope="module")
def learn():
    return importlib.import_module("katago-rs_amd.learn")


# The widths choose the operator's variants: shorter than a chunk, a wave a row, a wave or workgroup a row with what is known of its
# entries before, in parts.
@pytest.mark.parametrize("v,k,dtype", [(2, 2, torch.float32), (6, 4, torch.float32), (400, 4, torch.bfloat16), (400, 300, torch.float32),
                                       (2000, 4, torch.float32), (9000, 4, torch.float16), (20000, 4, torch.float32)])
@pytest.mark.parametrize("rest", [False, True])
def test_infinite_teacher_logits(learn, v, k, dtype, rest):
    """+infinity in an entry that counts makes its row NaN, with the teacher's normaliser too; in one that does not count, nothing."""
    c = distill.make(4, v, k, dtype, torch.float32, v, rest=rest)
    want = distill.run(learn, c)
    c["top"][1, 1] = math.inf
    c["index"][2, 0], c["top"][2, 0] = v, math.inf
    got = distill.run(learn, c)
    assert math.isnan(float(got.loss[1])) and torch.isnan(got.grad[1]).all()
    distill.check(learn, {name: t[2:3].contiguous() if torch.is_tensor(t) else t for name, t in c.items()})
    for row in (0, 3):
        assert torch.equal(got.loss[row], want.loss[row]) and torch.equal(got.grad[row], want.grad[row])
    assert torch.isnan(distill.run(learn, c, want_grad=False).loss[1]) and not torch.isnan(got.loss[[0, 2, 3]]).any()


@pytest.mark.parametrize("c", [1, 2, 3, 4, 5, 7, 8, 9])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_short_rows_about_large_means_backward(learn, c, dtype):
    """0 less such a mean, times rstd, is infinite: no place behind a row takes part. (h is 0 in rows of equal elements.)"""
    x = torch.tensor([1.0, 1e30, 2e36, -3e38, torch.finfo(dtype).max])[:, None].repeat(1, c).to(dtype)
    dy = torch.randn(5, c, generator=torch.Generator().manual_seed(c)).to(dtype)
    for rstd in (1e-5 ** -0.5, 2.0 ** 63):
        norm.backward(learn, x, dy, x[:, 0].float(), torch.full((5,), rstd), None, 0, c)


@pytest.mark.parametrize("c", [1, 5, 16, 100, 384, 1000, 3000, 6001, 9000, 16384, 16385, 40000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_whose_sum_passes_floats_range(learn, c, dtype):
    """Their mean does not: it is off by the float sum's rounding, at most (c / 64 + 24) U of the elements' size. Equal elements leave
    deviations of that size at most, whose squares are 0 or infinite: y is beta."""
    most = torch.finfo(dtype).max
    x, beta = torch.randn(6, c).to(dtype), torch.randn(c).to(dtype)
    x[1], x[2], x[3], x[4] = most, -most, most / 3, torch.where(torch.arange(c) % 2 == 0, most / 4, most / 2)
    y, mean, rstd = learn.layer_norm(x.cuda(), None, beta.float().cuda())
    want = x.double().mean(1)
    assert ((mean.cpu().double() - want).abs() <= (c / 64 + 24) * U * x.double().abs().mean(1))[1:5].all()
    assert torch.equal(y[1:5].cpu(), beta.expand(4, c))
    # (The other rows have the bits that they have beside ordinary ones: in their places, as rows of odd strides are cut along y's lines.)
    ordinary = learn.layer_norm(torch.cat([x[:1].expand(5, c), x[5:]]).cuda(), None, beta.float().cuda())
    for a, b in zip((y, mean, rstd), ordinary):
        assert torch.equal(a[[0, 5]], b[[0, 5]])
    dx = learn.layer_norm_backward(torch.ones_like(x).cuda(), x.cuda(), mean, rstd)[0]
    assert torch.isfinite(dx).all()
