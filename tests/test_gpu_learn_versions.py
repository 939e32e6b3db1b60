"""The learning operators write into tensors of the caller behind autograd's back; its version counters are raised as torch's own
in-place operations raise them, so that a backward pass through a graph that saved such a tensor is refused, not wrong."""

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


def _refused(graph):
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        graph.backward()


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_raises_versions(learn, bits):
    whole = torch.randn(600, device="cuda")
    params = [torch.nn.Parameter(torch.randn(30, device="cuda")), torch.randn(300, device="cuda").bfloat16(), *whole.split([512, 88])]
    masters = [None, params[1].float(), None, None]
    opt = learn.AdamW(params, lr=1e-2, state_bits=bits, masters=masters)
    grads = [torch.ones_like(p) for p in params]
    # (Autograd shares one counter between a tensor and its views.)
    kept = [_saves(t) for t in (*params, masters[1], whole)]
    other = _saves(grads[0])
    before = [p._version for p in params]
    opt.step(grads)
    assert all(p._version > v for p, v in zip(params, before))
    for graph in kept:
        _refused(graph)
    other.backward()
    kept = _saves(params[0])
    with pytest.raises(importlib.import_module("katago-rs_amd").KgError):
        opt.step(step=0)
    kept.backward()  # (nothing was written)


def test_given_outputs_raise_versions(learn):
    z, f = torch.randn(4, 30, device="cuda"), torch.zeros(4, device="cuda")
    act, off = torch.zeros(4, dtype=torch.int32, device="cuda"), torch.tensor([0, 2, 4], dtype=torch.int32, device="cuda")
    x = torch.randn(2, 9, 16, device="cuda")
    _, mean, rstd = learn.group_norm(x, 2)
    for like, call in ((z, lambda t: learn.policy_loss(z, act, f, f, grad=t)),
                       (z, lambda t: learn.preference_loss(z, act, off, f[:2], grad=t)),
                       (x, lambda t: learn.group_norm(x, 2, y=t)),
                       (x, lambda t: learn.group_norm_backward(x.clone(), x, mean, rstd, 2, dx=t))):
        out = torch.zeros_like(like)
        kept, inputs = _saves(out), _saves(like)
        call(out)
        _refused(kept)
        inputs.backward()
