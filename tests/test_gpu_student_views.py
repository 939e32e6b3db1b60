"""A student's operators on views side by side of one buffer: outputs between an input's rows or columns, which share no element with them.

Rows in other places may be cut along other lines, and their sums added in another order: both results lie within the operators' own bounds
(tests/test_gpu_distill.py, test_gpu_layer_norm.py), so that they differ by at most twice those."""

import importlib

import pytest
import torch

import student_ref as ref
import test_gpu_distill as distill

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def learn():
    return importlib.import_module("katago-rs_amd.learn")


def randn(*shape, seed=1):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).cuda()


@pytest.mark.parametrize("v", [7, 362, 2000, 20001])
def test_logits_and_their_gradient(learn, v):
    raw = randn(5, 2 * v + 3)
    z = raw[:, 1:v + 1].contiguous()
    top, index = z.topk(4, 1)
    index = index.int()
    want = learn.distill_loss(z, index, top)
    before = raw.clone()
    got = learn.distill_loss(raw[:, 1:v + 1], index, top, grad=raw[:, v + 1:2 * v + 1])
    _, _, lsize, gsize = ref.distill(z.cpu(), index.cpu(), top.cpu())
    x = distill.octaves(z.cpu(), 1.0)
    distill.close(got.loss, want.loss.cpu().double(), 2 * lsize, 3 * x + v / 64 + 20, "loss")
    distill.close(got.grad, want.grad.cpu().double(), 2 * gsize, 5 * x + v / 64 + 20, "grad")
    assert torch.equal(raw[:, :v + 1], before[:, :v + 1]) and torch.equal(raw[:, 2 * v + 1:], before[:, 2 * v + 1:])


@pytest.mark.parametrize("c", [5, 96, 1024, 5000])
def test_rows_between_rows(learn, c):
    both = randn(14, c)
    x, gamma = both[::2].contiguous(), randn(c, seed=2)
    want, mean, rstd = learn.layer_norm(x, gamma)
    y = learn.layer_norm(both[::2], gamma, y=both[1::2])[0]
    _, wmean, wrstd, h = ref.layer_norm(x.cpu(), gamma.cpu())
    spread = (x.cpu().double() - wmean[:, None]).abs().mean(1)
    g, w = c / 64 + 24, want.cpu().double()
    distill.close(y, w, 2 * ((h.abs() + (wrstd * spread)[:, None]) * gamma.cpu().double().abs() + w.abs()), 2 * g + 8, "y")
    dx = learn.layer_norm_backward(want, x, mean, rstd, gamma)[0]
    _, sizes = ref.layer_norm_backward(w, x.cpu(), mean.cpu(), rstd.cpu(), gamma.cpu())
    learn.layer_norm_backward(want, both[::2], mean, rstd, gamma, dx=both[1::2])
    distill.close(both[1::2], dx.cpu().double(), 2 * sizes[0], 2 * g + 12, "dx")
    assert torch.equal(both[::2], x)


def test_a_table_beside_its_gradient_and_tokens_rows(learn):
    room = randn(60, 40)
    tokens = (torch.arange(60, device="cuda", dtype=torch.int32) * 7) % 11
    table = room[:11, :16].contiguous()
    want = learn.embedding(tokens, table)
    assert torch.equal(learn.embedding(tokens, room[:11, :16], y=room[:, 16:32]), want) and torch.equal(room[:11, :16], table)
    grad = learn.embedding_backward(want, tokens, 11)
    learn.embedding_backward(room[:, 16:32], tokens, 11, grad=room[:11, :16])
    assert torch.equal(room[:11, :16], grad) and torch.equal(room[:, 16:32], want)
