"""What the learning operators refuse, before a device is touched, and the host-side arithmetic of the AdamW step."""

import ctypes
import importlib

import numpy as np
import pytest
import torch

import learn_abi as abi
import learn_ref as ref


@pytest.fixture(scope="module")
def learn():
    return importlib.import_module("katago-rs_amd.learn")


def _policy_args(learn, **change):
    base = dict(rows=4, columns=9, type=0, logits=4096, ld=9, legal=None, ld_legal=0, action=4096, old_logp=4096,
                advantage=4096, weight=None, ref_logits=None, ld_ref=0, ref_logp=None, logit_scale=1.0, clip_low=0.2,
                clip_high=0.2, kl_coef=0.0, loss=4096, logp=4096, kl=4096, grad=8192, ld_grad=9)
    return abi.PolicyArgs(**{**base, **change})


@pytest.mark.parametrize("change,text", [
    (dict(rows=-1), "rows must"), (dict(rows=2 ** 30 + 1), "rows must"), (dict(columns=0), "columns"), (dict(type=3), "type"), (dict(logits=None), "logits is null"),
    (dict(ld=8), "row stride of logits"), (dict(ld=-9), "row stride of logits"), (dict(ld=2 ** 62), "row stride of logits"),
    (dict(logits=4098), "aligned"), (dict(legal=4096, ld_legal=8), "legal"), (dict(action=None), "null argument"),
    (dict(old_logp=None), "null argument"), (dict(advantage=None), "null argument"), (dict(loss=None), "null argument"),
    (dict(kl=None), "null argument"), (dict(logit_scale=0.0), "logit_scale"), (dict(logit_scale=float("nan")), "logit_scale"),
    (dict(clip_low=1.0), "clip"), (dict(clip_low=-0.1), "clip"), (dict(clip_high=float("inf")), "clip"),
    (dict(kl_coef=float("nan")), "kl_coef"), (dict(ref_logits=4096, ld_ref=9, ref_logp=4096), "not both"),
    (dict(ref_logits=4096, ld_ref=3), "row stride of ref_logits"), (dict(grad=4096), "overlap"), (dict(ld_grad=1), "row stride of grad"),
    (dict(columns=20000, ld=20000, ld_grad=20000), "workspace is null"),
    (dict(columns=20000, ld=20000, ld_grad=20000, workspace=4104), "workspace is not aligned"),
])
def test_policy_loss_refuses(kgx, learn, change, text):
    assert kgx.lib().kg_policy_loss(0, None, ctypes.byref(_policy_args(learn, **change))) == 1
    assert text in kgx.lib().kg_last_error().decode()


@pytest.mark.parametrize("name", ["POLICY", "PREFERENCE", "NORM"])
def test_packed_arguments_lie_as_the_structures_do(learn, name):
    packed, kind = getattr(learn, f"_{name}_ARGS"), getattr(abi, {"POLICY": "PolicyArgs", "PREFERENCE": "PreferenceArgs", "NORM": "NormArgs"}[name])
    values = [0.5 + i if t is ctypes.c_double else 3 + i for i, (_, t) in enumerate(kind._fields_)]
    got = kind.from_buffer_copy(packed.pack(*values))
    assert packed.size == ctypes.sizeof(kind) and [getattr(got, f) for f, _ in kind._fields_] == values


def test_null_structures_are_refused(kgx, learn):
    L = kgx.lib()
    for f in (L.kg_policy_loss, L.kg_preference_loss, L.kg_group_norm, L.kg_group_norm_backward):
        assert f(0, None, None) == 1 and "null argument" in L.kg_last_error().decode()
    assert L.kg_adamw_step(0, None, 1, None, None, None, None) == 1
    assert L.kg_adamw_values(None, None) == 1
    assert L.kg_adamw_moments(0, None, 1, None, 0, None, None) == 1


@pytest.mark.parametrize("change,text", [
    (dict(rows=-1), "rows"), (dict(pairs=-1), "pairs"), (dict(pairs=2 ** 30), "pairs"), (dict(type=7), "type"), (dict(beta=0.0), "beta"),
    (dict(label_smoothing=0.6), "label_smoothing"), (dict(offsets=None), "offsets"), (dict(label=None), "label"),
    (dict(workspace=None), "workspace"), (dict(workspace=4100), "workspace"), (dict(seq_logp=None), "null argument"),
    (dict(grad=4096), "overlap"), (dict(ld=5), "row stride of logits"), (dict(logits=4097), "aligned"),
])
def test_preference_loss_refuses(kgx, learn, change, text):
    base = dict(rows=4, columns=9, type=1, logits=4096, ld=9, label=4096, pairs=1, offsets=4096, ref_logp=4096, weight=None,
                beta=0.1, label_smoothing=0.0, average=0, loss=4096, margin=4096, seq_logp=4096, grad=8192, ld_grad=9,
                workspace=4096)
    args = abi.PreferenceArgs(**{**base, **change})
    assert kgx.lib().kg_preference_loss(0, None, ctypes.byref(args)) == 1
    assert text in kgx.lib().kg_last_error().decode()


@pytest.mark.parametrize("backward", [False, True])
@pytest.mark.parametrize("change,text", [
    (dict(batch=-1), "batch"), (dict(channels=0), "channels"), (dict(groups=0), "groups"), (dict(groups=5), "multiple"),
    (dict(channels=4096, groups=4096, ldx=4096, ldy=4096, lddy=4096, lddx=4096), "2048 groups"),
    (dict(batch=1 << 20, points=1 << 20), "out of range"), (dict(type=-1), "type"), (dict(act=4), "activation"),
    (dict(x=None), "x is null"), (dict(ldx=11), "row stride of x"), (dict(mean=None), "mean"), (dict(workspace=None), "workspace"),
    (dict(workspace=4104), "workspace"), (dict(y=4096, dx=4096), "overlap"),
    (dict(batch=1 << 28, points=1), "batch x groups"), (dict(batch=1 << 25, points=1, channels=3), "batch x groups"),
])
def test_group_norm_refuses(kgx, learn, change, text, backward):
    base = dict(batch=2, points=9, channels=12, groups=3, type=0, act=2, eps=1e-5, x=4096, ldx=12, mask=None, gamma=None,
                beta=None, mean=4096, rstd=4096, workspace=4096, y=8192, ldy=12, dy=16384, lddy=12, dx=8192, lddx=12,
                dgamma=None, dbeta=None)
    args = abi.NormArgs(**{**base, **change})
    L = kgx.lib()
    assert (L.kg_group_norm_backward if backward else L.kg_group_norm)(0, None, ctypes.byref(args)) == 1
    assert text in L.kg_last_error().decode()


def test_group_norm_refuses_eps(kgx, learn):
    args = abi.NormArgs(2, 9, 12, 3, 0, 2, 0.0, 4096, 12)
    assert kgx.lib().kg_group_norm(0, None, ctypes.byref(args)) == 1
    assert "eps" in kgx.lib().kg_last_error().decode()


@pytest.mark.parametrize("tensor,state,hyper,text", [
    (dict(param=None), {}, {}, "tensor 1: null"), (dict(grad=None), {}, {}, "tensor 1: null"), (dict(param=4098), {}, {}, "aligned"),
    (dict(param_type=5), {}, {}, "type"), (dict(elements=-1), {}, {}, "size"), (dict(first_block=-1), {}, {}, "size"),
    (dict(weight_decay=float("inf")), {}, {}, "weight_decay"), ({}, dict(state_bits=16), {}, "state_bits"), ({}, dict(m=None), {}, "moments"),
    ({}, dict(state_bits=8, m_exp=None), {}, "exponents"), ({}, dict(m=4098), {}, "aligned"), ({}, {}, dict(beta1=1.0), "beta1"),
    ({}, {}, dict(eps=0.0), "eps"), ({}, {}, dict(eps=1e-60), "eps"), ({}, {}, dict(step=0), "step"), ({}, {}, dict(lr=float("nan")), "lr"),
    ({}, {}, dict(grad_scale=float("inf")), "grad_scale"),
])
def test_adamw_refuses(kgx, learn, tensor, state, hyper, text):
    good = dict(param=4096, grad=4096, master=None, elements=10, first_block=0, weight_decay=0.1, param_type=0, grad_type=0)
    tensors = (learn._AdamTensor * 2)(learn._AdamTensor(**good), learn._AdamTensor(**{**good, **tensor}))
    st = learn._AdamState(**{**dict(state_bits=32, m=4096, v=4096, m_exp=4096, v_exp=4096), **state})
    hy = learn._AdamHyper(**{**dict(lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, grad_scale=1.0, step=1, seed=0), **hyper})
    L = kgx.lib()
    assert L.kg_adamw_step(0, None, 2, ctypes.byref(tensors), ctypes.byref(st), ctypes.byref(hy), None) == 1
    assert text in L.kg_last_error().decode()


def test_adamw_values(kgx, learn):
    h = learn._AdamHyper(2e-4, 0.9, 0.999, 1e-8, 0.5, 1000, 77)
    v = learn.AdamValues()
    assert kgx.lib().kg_adamw_values(ctypes.byref(h), ctypes.byref(v)) == 0
    want = dict(lr=2e-4, beta1=0.9, beta1_rest=0.1, beta2=0.999, beta2_rest=0.001, eps=1e-8, grad_scale=0.5,
                step_size=2e-4 / (1 - 0.9 ** 1000), root_scale=(1 - 0.999 ** 1000) ** -0.5)
    for k, w in want.items():
        # (One rounding to float; the powers and differences in double are closer than that by far.)
        assert abs(getattr(v, k) - w) <= abs(w) * (ref.U + 1e-12), k
    assert v.seed == 77


def test_workspaces(kgx):
    L = kgx.lib()
    assert L.kg_policy_loss_workspace(-1, 100000) == L.kg_policy_loss_workspace(400, 100000) == L.kg_policy_loss_workspace(4, 362) == 0
    assert L.kg_policy_loss_workspace(1, 100000) >= 64 * 32 and L.kg_policy_loss_workspace(200, 17000) >= 200 * 2 * 32
    assert L.kg_preference_loss_workspace(0) == 0 and L.kg_preference_loss_workspace(-3) == 0
    assert L.kg_preference_loss_workspace(1000) >= 1000 * 20
    assert L.kg_group_norm_workspace(-1, 5, 8, 2, 0) == 0 and L.kg_group_norm_workspace(2, 5, 0, 2, 1) == 0
    for b, p, c, g in ((1, 1, 1, 1), (32, 361, 384, 32), (3, 16384, 1024, 64), (70000, 1, 4, 2)):
        assert L.kg_group_norm_workspace(b, p, c, g, 0) >= b * g * 12
        assert L.kg_group_norm_workspace(b, p, c, g, 1) >= b * (8 * c + 8 * g + 4)
    assert L.kg_group_norm_workspace(2, 5, 3, 2 ** 31 - 1, 1) >= 0  # (at once, also for what no call takes)


def test_python_calls_refuse_what_they_cannot_take(learn):
    z, a, f = torch.zeros(3, 5), torch.zeros(3, dtype=torch.int32), torch.zeros(3)
    with pytest.raises(ValueError, match="on the GPU"):
        learn.policy_loss(z, a, f, f)
    with pytest.raises(ValueError, match="float32, float16 or bfloat16"):
        learn.policy_loss(z.double(), a, f, f)
    with pytest.raises(ValueError, match="contiguous columns"):
        learn.policy_loss(torch.zeros(5, 3).t(), a, f, f)
    with pytest.raises(ValueError, match="on the GPU"):
        learn.preference_loss(z, a, torch.zeros(3, dtype=torch.int32), torch.zeros(2))
    with pytest.raises(ValueError, match="on the GPU"):
        learn.group_norm(torch.zeros(2, 9, 8), 2)
    with pytest.raises(ValueError, match="on the GPU"):
        learn.group_norm_backward(torch.zeros(2, 9, 8), torch.zeros(2, 9, 8), torch.zeros(2, 2), torch.zeros(2, 2), 2)
    with pytest.raises(ValueError, match="parameter 0"):
        learn.AdamW([torch.zeros(4)], lr=1e-3)
    with pytest.raises(ValueError, match="needs a parameter"):
        learn.AdamW([], lr=1e-3)
    with pytest.raises(ValueError, match="evenly spaced"):
        learn._points(_Cuda(torch.zeros(4, 9, 8)[:, :5]), "x")
    with pytest.raises(ValueError, match="contiguous channels"):
        learn._points(_Cuda(torch.zeros(1, 8, 9).transpose(1, 2)), "x")
    assert learn._points(_Cuda(torch.zeros(2, 3, 3, 16)[..., :8]), "x")[1] == 16
    assert learn._points(_Cuda(torch.zeros(2, 1, 8)), "x")[1] == 8


class _Cuda:
    """A CPU tensor that says it is on the GPU: its strides are looked at, its memory is not."""

    is_cuda = True

    def __init__(self, t):
        self.t = t

    def __getattr__(self, name):
        return getattr(self.t, name)


def test_eight_bit_moments_are_unbiased_and_bounded():
    """The rounding of the 8-bit moments (the restatement that the GPU's codes are held to, bit for bit): over many seeds its
    mean is the value, off by at most five standard errors, and never by more than a step; zeros stay 0 and positive roots
    positive."""
    rng = np.random.default_rng(3)
    x = (rng.standard_normal((2, 256)) * np.exp2(rng.integers(-12, 1, (2, 256)))).astype(np.float32)
    x[:, 7] = 0
    x[1] *= np.float32(1e-18)
    seeds = 2000
    for signed in (True, False):
        v = x if signed else np.abs(x)
        total, square = np.zeros(x.shape), np.zeros(x.shape)
        for s in range(seeds):
            um, ur = ref.noise(np.arange(512).reshape(2, 256), s)
            got = (ref.decode_m if signed else ref.decode_v)(*ref.encode(v, um if signed else ur, signed)).astype(np.float64)
            total += got
            square += (got - v) ** 2
            assert np.all(got[:, 7] == 0)
        top = np.abs(v).max(1, keepdims=True)
        # The spacing is at most 2^-3 (2^-5) of the value, or that of the smallest codes.
        step = np.maximum(np.abs(v) * 2.0 ** (-3 if signed else -5), top * 2.0 ** (-16 if signed else -11))
        assert np.all(square / seeds <= step ** 2)
        off, err = np.abs(total / seeds - v), step / 2 / np.sqrt(seeds)
        if not signed:  # (below the smallest code a root is raised to it)
            off = np.where(np.abs(v) < top * 2.0 ** -11, 0, off)
            assert np.all((got > 0) == (v > 0))
        assert np.all(off <= 5 * err), np.max(off / err)
