"""AdamW refuses parameters and masters that share memory: their workgroups would write one element at once."""

import importlib

import pytest
import torch


@pytest.fixture(scope="module")
def learn():
    return importlib.import_module("katago-rs_amd.learn")


class _OnGpu(torch.Tensor):
    is_cuda = property(lambda self: True)


def _on_gpu(t):
    return t.as_subclass(_OnGpu)


def test_parameters_that_share_memory(learn):
    room, other = _on_gpu(torch.zeros(100)), _on_gpu(torch.zeros(8).bfloat16())
    for params, masters in (([room[:10], room[9:20]], None), ([room[20:40], other, room[5:25]], None), ([room, room[3:4]], None),
                            ([room[:8], other], [None, room[4:12]]), ([room[:8], room[:8]], None), ([room[:8], room[:1]], None),
                            ([room[1:2], room], None)):
        with pytest.raises(ValueError, match="of its own"):
            learn.AdamW(params, lr=1e-3, masters=masters)


def test_neighbours_and_empty_parameters_are_taken(learn):
    room, other = _on_gpu(torch.zeros(100)), _on_gpu(torch.zeros(8).bfloat16())
    learn.AdamW([room[:10], room[10:20], room[15:15], room[20:]], lr=1e-3)
    learn.AdamW([room[92:], other], lr=1e-3, masters=[None, room[84:92]])
