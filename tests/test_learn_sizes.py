"""Sizes past 31 bits are refused with the errors that the calls name (ValueError or KgError), and at once."""

import importlib
import time

import pytest
import torch


@pytest.fixture(scope="module")
def learn():
    return importlib.import_module("katago-rs_amd.learn")


class _OnGpu(torch.Tensor):
    """A CPU tensor that says it is on GPU 0 and contiguous: its memory is not looked at."""

    is_cuda = property(lambda self: True)

    def get_device(self):
        return 0

    def is_contiguous(self):
        return True


def _huge(*shape, dtype=torch.float32):
    return torch.zeros((1,) * len(shape), dtype=dtype).expand(shape).as_subclass(_OnGpu)


@pytest.fixture
def no_memory(learn, monkeypatch):
    """Outputs that take no memory, on stream 0."""
    monkeypatch.setattr(torch, "empty", lambda shape, *, dtype, device: _huge(*((shape,) if isinstance(shape, int) else shape), dtype=dtype))
    monkeypatch.setattr(learn, "_stream", lambda device: 0)


@pytest.mark.parametrize("n", [2 ** 31, 2 ** 32 + 3, 2 ** 63 // 8])
def test_rows_past_31_bits(learn, no_memory, n):
    z, i, f = _huge(n, 1), _huge(n, dtype=torch.int32), _huge(n)
    with pytest.raises(ValueError, match="policy_loss"):
        learn.policy_loss(z, i, f, f, want_grad=False)
    with pytest.raises(ValueError, match="preference_loss"):
        learn.preference_loss(z, i, _huge(3, dtype=torch.int32), _huge(2), want_grad=False)
    with pytest.raises(ValueError, match="group_norm"):
        learn.group_norm(_huge(1, n, 1), 1)
    with pytest.raises(ValueError, match="group_norm_backward"):
        learn.group_norm_backward(_huge(1, n, 1), _huge(1, n, 1), _huge(1, 1), _huge(1, 1), 1)


def test_groups(kgx, learn, monkeypatch):
    monkeypatch.setattr(learn, "_stream", lambda device: 0)
    x = torch.zeros(2, 9, 12).as_subclass(_OnGpu)
    for groups, error in ((13, kgx.KgError), (0, kgx.KgError), (-1, kgx.KgError), (2 ** 31 - 1, kgx.KgError), (2 ** 31, ValueError),
                          (2 ** 40, ValueError)):
        with pytest.raises(error, match="group"):
            learn.group_norm(x, groups)


def test_group_norm_workspace_of_any_sizes(kgx):
    """At once, and 0 for groups that no call takes."""
    L, start = kgx.lib(), time.monotonic()
    for groups in (2 ** 31 - 1, 2 ** 31 - 2, 2 ** 31 - 19, 2049):
        assert L.kg_group_norm_workspace(1, 361, 2 ** 31 - 1, groups, 0) == 0
        assert L.kg_group_norm_workspace(1, 361, 2 ** 31 - 1, groups, 1) == 0
    assert L.kg_group_norm_workspace(1, 361, 2048, 2048, 0) >= 2048 * 12
    assert time.monotonic() - start < 1
