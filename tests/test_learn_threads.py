"""The learning operators called from several threads on one stream. A call's workspace has to be its own until its kernels are enqueued:
the library is called without the interpreter's lock, and memory that has gone back to the allocator before that is given to the
next thread that asks, whose kernels may then run between this call's."""

import importlib
import threading

import pytest
import torch
from torch.multiprocessing.reductions import StorageWeakRef

import learn_abi as abi


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


class _Library:
    """The library's workspace sizes; its launches look whether what they were given is still held."""

    def __init__(self, real, made):
        self.real, self.made, self.calls = real, made, []

    def __getattr__(self, name):
        kinds = {"kg_policy_loss": abi.PolicyArgs, "kg_preference_loss": abi.PreferenceArgs, "kg_group_norm": abi.NormArgs,
                 "kg_group_norm_backward": abi.NormArgs}
        if name not in kinds:
            return getattr(self.real, name)

        def launch(device, stream, args):
            at = kinds[name].from_buffer_copy(args).workspace
            held = [first <= at < first + size and not ref.expired() for first, size, ref in self.made]
            self.calls.append((name, any(held)))
            return 0
        return launch


def test_workspaces_are_held_until_the_launch(kgx, learn, monkeypatch):
    made = []
    empty = torch.empty

    def recorded(*args, **kwargs):
        t = empty(*args, **kwargs)
        made.append((t.data_ptr(), t.numel() * t.element_size(), StorageWeakRef(t.untyped_storage())))
        return t

    library = _Library(kgx.lib(), made)
    monkeypatch.setattr(learn, "_library", lambda: library)
    monkeypatch.setattr(learn, "_stream", lambda device: 0)
    monkeypatch.setattr(torch, "empty", recorded)
    f, z, x = _on_gpu(2), _on_gpu(2, 20000), _on_gpu(2, 9000, 16)
    learn.policy_loss(z, _on_gpu(2, dtype=torch.int32), f, f)
    learn.preference_loss(z, _on_gpu(2, dtype=torch.int32), _on_gpu(3, dtype=torch.int32), f)
    learn.group_norm(x, 2)
    learn.group_norm_backward(x, x, _on_gpu(2, 2), _on_gpu(2, 2), 2)
    assert library.calls == [(name, True) for name in ("kg_policy_loss", "kg_preference_loss", "kg_group_norm", "kg_group_norm_backward")]


@pytest.mark.gpu
def test_two_threads_on_one_stream(learn):
    """Each thread's results are those of the same calls alone, bit for bit."""
    def work(seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        x, dy = (torch.randn(3, 5000, 96, generator=g, device="cuda") for _ in range(2))
        z = torch.randn(3, 30011, generator=g, device="cuda")
        act = torch.tensor([5, 30010, 7], dtype=torch.int32, device="cuda")
        off, f = torch.tensor([0, 2, 3], dtype=torch.int32, device="cuda"), torch.full((3,), -10.0, device="cuda")

        def step():
            y, mean, rstd = learn.group_norm(x, 4, act="silu")
            return [y, *learn.group_norm_backward(dy, x, mean, rstd, 4, act="silu"), *learn.policy_loss(z, act, f, f),
                    *learn.preference_loss(z, act, off, f[:2])]
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
