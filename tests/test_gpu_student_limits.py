"""A student's operators where a number passes a type's range: infinite entries of the teacher's, rows shorter than
16 bytes about a mean near float's largest."""

import importlib
import math

import pytest
import torch

import test_gpu_distill as distill
import test_gpu_layer_norm as norm

pytestmark = pytest.mark.gpu


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
