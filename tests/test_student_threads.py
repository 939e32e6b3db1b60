"""A student's operators called from several threads on one stream, and what they take while the library is called: a call's workspace is
its own until its kernels are enqueued."""

import importlib
import threading

import pytest
import torch
from torch.multiprocessing.reductions import StorageWeakRef

import student_abi as abi


@pytest.fixture(scope="module")
def learn():
    return importlib.import_module("katago-rs_amd.learn")


class _OnGpu(torch.Tensor):
    """A CPU tensor that says it is on GPU 0."""

    is_cuda = property(lambda self: True)

    def get_device(self):
        return 0


def _on_gpu(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype).as_subclass(_OnGpu)


def test_workspaces_are_held_until_the_launch(kgx, learn, monkeypatch):
    made, calls = [], []
    kinds = {"kg_distill_loss": abi.DistillArgs, "kg_layer_norm_backward": abi.LayerArgs, "kg_embedding_backward": abi.EmbedArgs}

    class Library:
        def __getattr__(self, name):
            if name not in kinds:
                return getattr(kgx.lib(), name)

            def launch(device, stream, args):
                at = kinds[name].from_buffer_copy(args).workspace
                calls.append((name, any(first <= at < first + size and not ref.expired() for first, size, ref in made)))
                return 0
            return launch

    empty = torch.empty

    def recorded(*args, **kwargs):
        t = empty(*args, **kwargs)
        made.append((t.data_ptr(), t.numel() * t.element_size(), StorageWeakRef(t.untyped_storage())))
        return t

    monkeypatch.setattr(learn, "_library", Library)
    monkeypatch.setattr(learn, "_stream", lambda device: 0)
    monkeypatch.setattr(torch, "empty", recorded)
    learn.distill_loss(_on_gpu(2, 2000), _on_gpu(2, 3, dtype=torch.int32), _on_gpu(2, 3))
    learn.layer_norm_backward(_on_gpu(2, 16), _on_gpu(2, 16), _on_gpu(2), _on_gpu(2))
    learn.embedding_backward(_on_gpu(2, 16), _on_gpu(2, dtype=torch.int32), 9)
    assert calls == [(name, True) for name in kinds]


@pytest.mark.gpu
def test_two_threads_on_one_stream(learn):
    """Each thread's results are those of the same calls alone, bit for bit."""
    def work(seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        x, dy = (torch.randn(3000, 96, generator=g, device="cuda") for _ in range(2))
        z = torch.randn(3, 30011, generator=g, device="cuda")
        top, index = z.topk(20, 1)
        index, tokens = index.int(), torch.randint(0, 50, (3000,), generator=g, device="cuda").int()
        many = torch.randint(0, 500, (12000,), generator=g, device="cuda").int()
        dm = torch.randn(12000, 24, generator=g, device="cuda")

        def step():
            y, mean, rstd = learn.layer_norm(x)
            return [y, *learn.layer_norm_backward(dy, x, mean, rstd), *learn.distill_loss(z, index, top),
                    learn.embedding(tokens, x), learn.embedding_backward(dy, tokens, 50), learn.embedding_backward(dm, many, 500)]
        return step

    steps = [work(seed) for seed in (1, 2)]
    want = [step() for step in steps]
    torch.cuda.synchronize()
    wrong, failed = [0, 0], []

    def run(k):
        try:
            for _ in range(40):
                wrong[k] += sum(not torch.equal(a, b) for a, b in zip(steps[k](), want[k]))
        except Exception as e:  # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=run, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed and wrong == [0, 0]
