"""Sizes past what the library takes are refused with the errors that the calls name (ValueError or KgError), and at once."""

import importlib
import time

import pytest
import torch


@pytest.fixture(scope="module")
def learn():
    return importlib.import_module("katago-rs_amd.learn")


class _OnGpu(torch.Tensor):
    """A CPU tensor that says it is on GPU 0 and contiguous: its memory is not looked at, and new ones take none."""

    is_cuda = property(lambda self: True)

    def get_device(self):
        return 0

    def is_contiguous(self):
        return True

    def new_empty(self, shape, dtype=None):
        shape = (shape,) if isinstance(shape, int) else tuple(shape)
        if max(shape, default=0) < 100:
            return torch.zeros(shape, dtype=dtype or self.dtype).as_subclass(_OnGpu)
        return _huge(*shape, dtype=dtype or self.dtype)


def _huge(*shape, dtype=torch.float32):
    return torch.zeros((1,) * len(shape), dtype=dtype).expand(shape).as_subclass(_OnGpu)


@pytest.fixture
def no_memory(learn, monkeypatch):
    monkeypatch.setattr(torch, "empty", lambda shape, *, dtype, device: _huge(*((shape,) if isinstance(shape, int) else shape), dtype=dtype))
    monkeypatch.setattr(learn, "_stream", lambda device: 0)


@pytest.mark.parametrize("n", [2 ** 31, 2 ** 32 + 3, 2 ** 63 // 16])
def test_rows_past_31_bits(learn, no_memory, n):
    z, i, i2 = _huge(n, 1), _huge(n, dtype=torch.int32), _huge(n, 1, dtype=torch.int32)
    with pytest.raises(ValueError, match="distill_loss"):
        learn.distill_loss(z, i2, z, want_grad=False)
    with pytest.raises(ValueError, match="layer_norm"):
        learn.layer_norm(z)
    with pytest.raises(ValueError, match="layer_norm_backward"):
        learn.layer_norm_backward(z, z, _huge(n), _huge(n))
    with pytest.raises(ValueError, match="embedding"):
        learn.embedding(i, _huge(4, 1))
    with pytest.raises(ValueError, match="embedding"):
        learn.embedding(_huge(3, dtype=torch.int32), z)
    with pytest.raises(ValueError, match="embedding_backward"):
        learn.embedding_backward(z, i, 4)


def test_rows_past_30_bits(kgx, learn, no_memory):
    n = 2 ** 30 + 1
    z, i, i2 = _huge(n, 1), _huge(n, dtype=torch.int32), _huge(n, 1, dtype=torch.int32)
    for call in (lambda: learn.distill_loss(z, i2, z, want_grad=False), lambda: learn.layer_norm(z),
                 lambda: learn.layer_norm_backward(z, z, _huge(n), _huge(n)), lambda: learn.embedding(i, _huge(4, 1)),
                 lambda: learn.embedding_backward(z, i, 4)):
        with pytest.raises(kgx.KgError, match="2.30"):
            call()


def test_scalars_out_of_range(kgx, learn, no_memory):
    x, i = torch.zeros(3, 8).as_subclass(_OnGpu), _huge(3, dtype=torch.int32)
    for eps in (0.0, -1.0, float("nan"), 1e-60):
        with pytest.raises(kgx.KgError, match="eps"):
            learn.layer_norm(x, eps=eps)
    for scale in (float("inf"), float("nan"), 1e39):
        with pytest.raises(kgx.KgError, match="scale"):
            learn.embedding(i, x, scale=scale)
        with pytest.raises(kgx.KgError, match="scale"):
            learn.embedding_backward(x, i, 5, scale=scale)
    for k in (0, 1025):
        with pytest.raises(kgx.KgError, match="k must"):
            learn.distill_loss(x, torch.zeros(3, k, dtype=torch.int32).as_subclass(_OnGpu), torch.zeros(3, k).as_subclass(_OnGpu))


def test_workspaces_of_any_sizes(kgx):
    L, start = kgx.lib(), time.monotonic()
    top = 2 ** 31 - 1
    for a in (-5, 0, 1, 1000, top):
        for b in (-5, 0, 1, 1000, top):
            L.kg_layer_norm_workspace(a, b)
            for c in (-5, 0, 1, 1000, top):
                L.kg_distill_loss_workspace(a, b, c)
                L.kg_embedding_backward_workspace(a, b, c)
    assert time.monotonic() - start < 1
