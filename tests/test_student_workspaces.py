"""The workspaces that a student's operators ask for: 0 where no call takes the sizes, and never less than their parts; and what
learn.py gives where it does not ask."""

import importlib

import torch

import student_abi as abi


def test_sizes_that_no_call_takes(kgx):
    L, over, top = kgx.lib(), 2 ** 30 + 1, 2 ** 31 - 1
    for n in (0, -1, -2 ** 31, over, top):
        assert L.kg_distill_loss_workspace(n, 2000, 50) == L.kg_distill_loss_workspace(50, n, 300) == L.kg_distill_loss_workspace(50, 2000, n) == 0
        assert L.kg_layer_norm_workspace(n, 16) == L.kg_layer_norm_workspace(16, n) == 0
        assert L.kg_embedding_backward_workspace(n, 16, 16) == L.kg_embedding_backward_workspace(16, n, 16) == 0
        assert L.kg_embedding_backward_workspace(16, 16, n) == 0
    assert L.kg_distill_loss_workspace(50, 2000, 1025) == 0


def test_largest_sizes_do_not_overflow(kgx):
    L, most = kgx.lib(), 2 ** 30
    assert L.kg_distill_loss_workspace(most, most, 1024) >= most * 1024 * 20
    assert L.kg_layer_norm_workspace(most, most) >= most * 16 + 1024 * 2 * most * 4
    assert L.kg_embedding_backward_workspace(most, most, most) >= most * 8 + most // (64 * 4) * 2 * most * 4


def test_short_rows_need_none(kgx):
    for rows in (1, 384, 385, 2 ** 30):
        for columns, k in ((1, 1), (1, 256), (448, 1), (448, 256)):
            assert kgx.lib().kg_distill_loss_workspace(rows, columns, k) == 0


class _OnGpu(torch.Tensor):
    """A CPU tensor that says it is on GPU 0."""

    is_cuda = property(lambda self: True)

    def get_device(self):
        return 0


def test_calls_have_the_workspaces_that_the_library_asks_for(kgx, monkeypatch):
    learn = importlib.import_module("katago-rs_amd.learn")
    given = []

    class Library:
        def __getattr__(self, name):
            return getattr(kgx.lib(), name)

        def kg_distill_loss(self, device, stream, args):
            given.append(abi.DistillArgs.from_buffer_copy(args).workspace)
            return 0

    monkeypatch.setattr(learn, "_library", Library)
    monkeypatch.setattr(learn, "_stream", lambda device: 0)
    for dtype in learn.TYPES:
        for v in (1, 3, 7, 362, 447, 448, 449, 512, 2000, 20000):
            for k in (1, 255, 256, 257, 1024):
                learn.distill_loss(torch.zeros(2, v, dtype=dtype).as_subclass(_OnGpu), torch.zeros(2, k, dtype=torch.int32).as_subclass(_OnGpu),
                                   torch.zeros(2, k).as_subclass(_OnGpu))
                assert bool(given[-1]) == (kgx.lib().kg_distill_loss_workspace(2, v, k) > 0), (v, k)
