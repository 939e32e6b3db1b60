"""What a student's operators refuse, before a device is touched."""

import ctypes
import importlib

import pytest
import torch

import student_abi as abi


@pytest.fixture(scope="module")
def learn():
    return importlib.import_module("katago-rs_amd.learn")


DISTILL = dict(rows=4, columns=9, k=3, type=0, top_type=1, logits=4096, ld=9, legal=None, ld_legal=0, top_index=4096, ld_index=3,
               top_logits=12288, ld_top=3, teacher_lse=None, weight=None, logit_scale=1.0, loss=4096, grad=8192, ld_grad=9)


@pytest.mark.parametrize("change,text", [
    (dict(rows=-1), "rows must"), (dict(rows=2 ** 30 + 1), "rows must"), (dict(columns=0), "columns"), (dict(columns=2 ** 30 + 1), "columns"),
    (dict(k=0), "k must"), (dict(k=1025), "k must"), (dict(type=3), "type"), (dict(top_type=-1), "type"), (dict(logits=None), "logits is null"),
    (dict(ld=8), "row stride of logits"), (dict(ld=-9), "row stride of logits"), (dict(ld=2 ** 62), "row stride of logits"),
    (dict(logits=4098), "aligned"), (dict(top_index=None), "top_index is null"), (dict(ld_index=2), "row stride of top_index"),
    (dict(top_index=4098), "top_index is not aligned"), (dict(top_logits=None), "top_logits is null"), (dict(top_logits=12289), "aligned"),
    (dict(ld_top=2), "row stride of top_logits"), (dict(legal=4096, ld_legal=8), "legal"), (dict(loss=None), "null argument"),
    (dict(logit_scale=0.0), "logit_scale"), (dict(logit_scale=float("nan")), "logit_scale"), (dict(logit_scale=2.0 ** 65), "logit_scale"),
    (dict(grad=4096), "overlap"), (dict(ld_grad=1), "row stride of grad"),
    (dict(columns=2000, ld=2000, ld_grad=2000), "workspace is null"), (dict(columns=2000, ld=2000, ld_grad=2000, workspace=4104), "workspace is not aligned"),
])
def test_distill_loss_refuses(kgx, change, text):
    assert kgx.lib().kg_distill_loss(0, None, ctypes.byref(abi.DistillArgs(**{**DISTILL, **change}))) == 1
    assert text in kgx.lib().kg_last_error().decode()


@pytest.mark.parametrize("backward", [False, True])
@pytest.mark.parametrize("change,text", [
    (dict(rows=-1), "rows"), (dict(rows=2 ** 30 + 1), "rows"), (dict(channels=0), "channels"), (dict(type=9), "type"), (dict(x=None), "x is null"),
    (dict(ldx=11), "row stride of x"), (dict(x=4098), "aligned"), (dict(mean=None), "mean"), (dict(rstd=None), "rstd"),
    (dict(y=4096, dx=4096), "overlap"), (dict(ldy=3, lddx=3), "row stride"), (dict(dy=None, y=None), "null"),
])
def test_layer_norm_refuses(kgx, change, text, backward):
    base = dict(rows=5, channels=12, type=0, rms=0, eps=1e-5, x=4096, ldx=12, gamma=None, beta=None, mean=4096, rstd=4096, workspace=4096,
                y=8192, ldy=12, dy=16384, lddy=12, dx=8192, lddx=12, dgamma=None, dbeta=None)
    L = kgx.lib()
    args = abi.LayerArgs(**{**base, **change})
    assert (L.kg_layer_norm_backward if backward else L.kg_layer_norm)(0, None, ctypes.byref(args)) == 1
    assert text in L.kg_last_error().decode()
    if backward:
        for change, text in ((dict(workspace=None), "workspace is null"), (dict(workspace=4104), "workspace is not aligned"),
                             (dict(lddy=11), "row stride of dy"), (dict(dx=16384), "overlap")):
            assert L.kg_layer_norm_backward(0, None, ctypes.byref(abi.LayerArgs(**{**base, **change}))) == 1
            assert text in L.kg_last_error().decode()
    else:
        for eps in (0.0, -1.0, float("nan"), float("inf"), 1e-60):
            assert L.kg_layer_norm(0, None, ctypes.byref(abi.LayerArgs(**{**base, "eps": eps}))) == 1
            assert "eps" in L.kg_last_error().decode()


@pytest.mark.parametrize("backward", [False, True])
@pytest.mark.parametrize("change,text", [
    (dict(count=-1), "count"), (dict(count=2 ** 30 + 1), "count"), (dict(vocab=0), "vocab"), (dict(vocab=2 ** 30 + 1), "vocab"),
    (dict(channels=0), "channels"), (dict(type=4), "type"), (dict(tokens=None), "tokens"), (dict(tokens=4098), "tokens"),
    (dict(scale=float("inf")), "scale"), (dict(scale=1e39), "scale"), (dict(table=None, dy=None), "null"), (dict(table=4097, dy=4097), "aligned"),
    (dict(ld_table=7, ld_dy=7), "row stride"), (dict(y=None, grad=None), "null"), (dict(ld_y=7, ld_grad=7), "row stride"),
    (dict(y=16384, grad=16384), "overlap"),
])
def test_embedding_refuses(kgx, change, text, backward):
    base = dict(count=5, vocab=7, channels=8, type=1, tokens=4096, scale=1.0, table=16384, ld_table=8, y=8192, ld_y=8, dy=16384, ld_dy=8,
                grad_type=1, accumulate=0, grad=8192, ld_grad=8, workspace=4096)
    L = kgx.lib()
    args = abi.EmbedArgs(**{**base, **change})
    assert (L.kg_embedding_backward if backward else L.kg_embedding)(0, None, ctypes.byref(args)) == 1
    assert text in L.kg_last_error().decode()
    if backward:
        for change, text in ((dict(workspace=None), "workspace is null"), (dict(workspace=4104), "workspace is not aligned"),
                             (dict(grad_type=2), "grad_type"), (dict(grad_type=0, grad=8194), "aligned")):
            assert L.kg_embedding_backward(0, None, ctypes.byref(abi.EmbedArgs(**{**base, **change}))) == 1
            assert text in L.kg_last_error().decode()


def test_null_structures_are_refused(kgx):
    L = kgx.lib()
    for f in (L.kg_distill_loss, L.kg_layer_norm, L.kg_layer_norm_backward, L.kg_embedding, L.kg_embedding_backward):
        assert f(0, None, None) == 1 and "null argument" in L.kg_last_error().decode()


def test_nothing_to_do_touches_no_device(kgx):
    L = kgx.lib()
    assert L.kg_distill_loss(99, None, ctypes.byref(abi.DistillArgs(columns=5, k=2, logit_scale=1.0))) == 0
    assert L.kg_layer_norm(99, None, ctypes.byref(abi.LayerArgs(channels=5, eps=1e-5))) == 0
    assert L.kg_embedding(99, None, ctypes.byref(abi.EmbedArgs(vocab=5, channels=5))) == 0
    assert L.kg_embedding_backward(99, None, ctypes.byref(abi.EmbedArgs(vocab=5, channels=5, accumulate=1))) == 0


@pytest.mark.parametrize("name", ["DISTILL", "LAYER", "EMBED"])
def test_packed_arguments_lie_as_the_structures_do(learn, name):
    packed, kind = getattr(learn, f"_{name}_ARGS"), getattr(abi, {"DISTILL": "DistillArgs", "LAYER": "LayerArgs", "EMBED": "EmbedArgs"}[name])
    values = [0.5 + i if t is ctypes.c_double else 3 + i for i, (_, t) in enumerate(kind._fields_)]
    got = kind.from_buffer_copy(packed.pack(*values))
    assert packed.size == ctypes.sizeof(kind) and [getattr(got, f) for f, _ in kind._fields_] == values


def test_workspaces(kgx):
    L = kgx.lib()
    assert L.kg_distill_loss_workspace(-1, 100000, 5) == L.kg_distill_loss_workspace(4, 362, 24) == L.kg_distill_loss_workspace(4, 5000, -1) == 0
    assert L.kg_distill_loss_workspace(1, 362, 1024) >= 20 * 1024 and L.kg_distill_loss_workspace(2 ** 30, 2 ** 30, 1024) >= 20 * 2 ** 40
    assert L.kg_layer_norm_workspace(0, 5) == L.kg_layer_norm_workspace(-2, 5) == L.kg_layer_norm_workspace(5, -1) == 0
    assert L.kg_layer_norm_workspace(1, 1) >= 8 and L.kg_layer_norm_workspace(100000, 1024) >= 8192
    assert L.kg_embedding_backward_workspace(0, 5, 5) == L.kg_embedding_backward_workspace(5, 0, 5) == 0
    assert L.kg_embedding_backward_workspace(5, 5, -1) == 0
    for n, v, c in ((1, 1, 1), (2 ** 30, 2 ** 30, 1), (5000, 2 ** 30, 4096)):
        assert 8 * n <= L.kg_embedding_backward_workspace(n, v, c) < 1 << 50


class _Cuda(torch.Tensor):
    """A CPU tensor that says it is on GPU 0."""

    is_cuda = property(lambda self: True)

    def get_device(self):
        return 0


def _gpu(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype).as_subclass(_Cuda)


def test_python_calls_refuse_what_they_cannot_take(learn):
    z, i, i32 = torch.zeros(3, 5), torch.zeros(3, 2, dtype=torch.int32), torch.int32
    with pytest.raises(ValueError, match="on the GPU"):
        learn.distill_loss(z, i, torch.zeros(3, 2))
    with pytest.raises(ValueError, match="top_logits"):
        learn.distill_loss(_gpu(3, 5), _gpu(3, 2, dtype=i32), _gpu(4, 2))
    with pytest.raises(ValueError, match="top_index"):
        learn.distill_loss(_gpu(3, 5), _gpu(3, 2, dtype=torch.int64), _gpu(3, 2))
    with pytest.raises(ValueError, match="top_index"):
        learn.distill_loss(_gpu(3, 5), _gpu(2, 3, dtype=i32).t(), _gpu(3, 2))
    with pytest.raises(ValueError, match="legal"):
        learn.distill_loss(_gpu(3, 5), _gpu(3, 2, dtype=i32), _gpu(3, 2), legal=_gpu(3, 5))
    with pytest.raises(ValueError, match="teacher_lse"):
        learn.distill_loss(_gpu(3, 5), _gpu(3, 2, dtype=i32), _gpu(3, 2), teacher_lse=_gpu(4))
    with pytest.raises(ValueError, match="grad"):
        learn.distill_loss(_gpu(3, 5), _gpu(3, 2, dtype=i32), _gpu(3, 2), grad=_gpu(3, 6))
    with pytest.raises(ValueError, match="on the GPU"):
        learn.layer_norm(torch.zeros(2, 8))
    with pytest.raises(ValueError, match="batch"):
        learn.layer_norm(_gpu(8))
    with pytest.raises(ValueError, match="gamma"):
        learn.layer_norm(_gpu(2, 8), _gpu(7))
    with pytest.raises(ValueError, match="beta"):
        learn.layer_norm(_gpu(2, 8), None, _gpu(8, dtype=torch.float16))
    with pytest.raises(ValueError, match="y must have"):
        learn.layer_norm(_gpu(2, 8), y=_gpu(2, 9))
    with pytest.raises(ValueError, match="dy must have"):
        learn.layer_norm_backward(_gpu(2, 9), _gpu(2, 8), _gpu(2), _gpu(2))
    with pytest.raises(ValueError, match="rstd must"):
        learn.layer_norm_backward(_gpu(2, 8), _gpu(2, 8), None, _gpu(3))
    with pytest.raises(ValueError, match="on the GPU"):
        learn.embedding(torch.zeros(3, dtype=i32), z)
    with pytest.raises(ValueError, match="tokens"):
        learn.embedding(_gpu(3), _gpu(3, 5))
    with pytest.raises(ValueError, match="tokens"):
        learn.embedding(torch.zeros(3, dtype=i32), _gpu(3, 5))
    with pytest.raises(ValueError, match="tokens"):
        learn.embedding(torch.zeros((), dtype=i32).as_subclass(_Cuda), _gpu(3, 5))
    with pytest.raises(ValueError, match="y must be"):
        learn.embedding(_gpu(3, dtype=i32), _gpu(3, 5), y=_gpu(3, 4))
    with pytest.raises(ValueError, match="dy must be"):
        learn.embedding_backward(_gpu(3, 5), _gpu(4, dtype=i32), 9)
    with pytest.raises(ValueError, match="accumulate"):
        learn.embedding_backward(_gpu(3, 5), _gpu(3, dtype=i32), 9, accumulate=True)
    for vocab in (0, -3, 2 ** 31, 2 ** 40):
        with pytest.raises(ValueError, match="vocab"):
            learn.embedding_backward(_gpu(3, 5), _gpu(3, dtype=i32), vocab)
    with pytest.raises(ValueError, match="grad must be"):
        learn.embedding_backward(_gpu(3, 5), _gpu(3, dtype=i32), 9, grad=_gpu(9, 4))
