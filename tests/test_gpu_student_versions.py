"""A student's operators raise the version counters of what they write of the caller's, and of nothing else."""

import importlib

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def learn():
    return importlib.import_module("katago-rs_amd.learn")


def _saves(t):
    """A result whose backward pass needs t as it is now."""
    return (torch.ones(t.shape, dtype=t.dtype, device=t.device, requires_grad=True) * t).sum()


def test_given_outputs_raise_versions(learn):
    z, x, table = torch.randn(4, 30, device="cuda"), torch.randn(6, 16, device="cuda"), torch.randn(9, 16, device="cuda")
    top, index = z.topk(5, 1)
    index, tokens = index.int(), torch.tensor([0, 3, 3, 8, -1, 2], dtype=torch.int32, device="cuda")
    _, mean, rstd = learn.layer_norm(x)
    for like, inputs, call in (
            (z, (z, top), lambda t: learn.distill_loss(z, index, top, grad=t)),
            (x, (x,), lambda t: learn.layer_norm(x, y=t)),
            (x, (x, mean, rstd), lambda t: learn.layer_norm_backward(x.clone(), x, mean, rstd, dx=t)),
            (x, (table,), lambda t: learn.embedding(tokens, table, y=t)),
            (table, (x,), lambda t: learn.embedding_backward(x, tokens, 9, grad=t)),
            (table, (x,), lambda t: learn.embedding_backward(x, tokens, 9, grad=t, accumulate=True))):
        out = torch.zeros_like(like)
        kept, others = _saves(out), [_saves(t) for t in inputs]
        call(out)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            kept.backward()
        for graph in others:
            graph.backward()
