"""A student's operators refuse outputs that share memory with anything else of a call, and take views side by side of one buffer.

The calls name a device that there is not: what the checks let pass is refused there, before a kernel is launched."""

import ctypes
import importlib
import random

import pytest
import torch

import student_abi as abi

NO_DEVICE = 9999


def overlaps(kgx, name, args):
    """What of the arguments the call says to overlap, or None where it takes them as far as the device."""
    L = kgx.lib()
    assert getattr(L, name)(NO_DEVICE, None, ctypes.byref(args)) == 1
    text = L.kg_last_error().decode()
    return text.split(": ", 1)[1] if "must not overlap" in text else None


DISTILL = dict(rows=4, columns=600, k=300, type=0, top_type=0, logits=1 << 20, ld=700, legal=1 << 21, ld_legal=600, top_index=1 << 22, ld_index=300,
               top_logits=1 << 23, ld_top=300, teacher_lse=1 << 24, weight=(1 << 24) + 16, logit_scale=1.0, loss=(1 << 24) + 32, grad=1 << 25,
               ld_grad=600, workspace=1 << 26)
LAYER = dict(rows=5, channels=12, type=1, rms=0, eps=1e-5, x=1 << 20, ldx=12, gamma=1 << 21, beta=(1 << 21) + 48, mean=1 << 22, rstd=(1 << 22) + 20,
             workspace=1 << 23, y=1 << 24, ldy=24, dy=1 << 25, lddy=12, dx=1 << 26, lddx=24, dgamma=1 << 27, dbeta=(1 << 27) + 48)
EMBED = dict(count=9, vocab=7, channels=8, type=1, tokens=1 << 20, scale=1.0, table=1 << 21, ld_table=8, y=1 << 22, ld_y=8, dy=1 << 23, ld_dy=16,
             grad_type=0, accumulate=1, grad=1 << 24, ld_grad=8, workspace=1 << 25)


@pytest.mark.parametrize("name,kind,base,out,inputs", [
    ("kg_distill_loss", abi.DistillArgs, DISTILL, ("grad", "loss", "workspace"), ("logits", "legal", "top_index", "top_logits", "teacher_lse", "weight")),
    ("kg_layer_norm", abi.LayerArgs, LAYER, ("y", "mean", "rstd"), ("x", "gamma", "beta")),
    ("kg_layer_norm_backward", abi.LayerArgs, LAYER, ("dx", "dgamma", "dbeta", "workspace"), ("x", "dy", "gamma", "mean", "rstd")),
    ("kg_embedding", abi.EmbedArgs, EMBED, ("y",), ("table", "tokens")),
    ("kg_embedding_backward", abi.EmbedArgs, EMBED, ("grad", "workspace"), ("dy", "tokens")),
])
def test_each_output_against_the_rest(kgx, name, kind, base, out, inputs):
    assert overlaps(kgx, name, kind(**base)) is None
    for o in out:
        for r in (*out, *inputs):
            if r != o:
                said = overlaps(kgx, name, kind(**{**base, r: base[o]}))
                assert said is not None and o in said and r in said, (o, r, said)
                if "workspace" not in (o, r):  # (which begins at multiples of 16)
                    assert overlaps(kgx, name, kind(**{**base, r: base[o] + 4})) is not None, (o, r)
    assert overlaps(kgx, name, kind(**{**base, inputs[0]: base[inputs[1]]})) is None


def test_what_a_call_does_not_use_may_lie_anywhere(kgx):
    rms = {**LAYER, "rms": 1}
    for name, out in (("kg_layer_norm", "y"), ("kg_layer_norm_backward", "dx")):
        assert overlaps(kgx, name, abi.LayerArgs(**{**rms, "mean": LAYER[out]})) is None
        assert overlaps(kgx, name, abi.LayerArgs(**{**LAYER, "mean": LAYER[out]})) is not None
    assert overlaps(kgx, "kg_layer_norm_backward", abi.LayerArgs(**{**LAYER, "beta": LAYER["dx"], "y": LAYER["x"]})) is None
    assert overlaps(kgx, "kg_layer_norm", abi.LayerArgs(**{**LAYER, "workspace": LAYER["y"], "dx": LAYER["x"]})) is None
    assert overlaps(kgx, "kg_distill_loss", abi.DistillArgs(**{**DISTILL, "columns": 400, "k": 200, "workspace": DISTILL["grad"]})) is None


def test_rows_of_any_strides(kgx):
    """Against the bytes themselves: rows of dy and of a gradient of another type, width and stride, and tokens."""
    r, met = random.Random(5), [0, 0]
    for _ in range(6000):
        n, vocab, c = r.randint(1, 40), r.randint(1, 40), r.randint(1, 9)
        ld, ld_g, wide = c + r.choice([0, 1, r.randint(0, 30)]), c + r.choice([0, 3, r.randint(0, 60)]), r.random() < 0.5
        if r.random() < 0.3:
            ld_g = ld * r.randint(1, 4)
        size = 4 if wide else 2
        at = (1 << 20) + 4 * r.randint(-400, 400)
        dy = {(1 << 20) + i * ld * 2 + b for i in range(n) for b in range(c * 2)}
        grad = {at + i * ld_g * size + b for i in range(vocab) for b in range(c * size)}
        args = abi.EmbedArgs(**{**EMBED, "count": n, "vocab": vocab, "channels": c, "dy": 1 << 20, "ld_dy": ld, "grad": at, "ld_grad": ld_g,
                                "grad_type": 0 if wide else 1, "tokens": 1 << 12})
        want = bool(dy & grad)
        assert (overlaps(kgx, "kg_embedding_backward", args) is not None) == want, (n, vocab, c, ld, ld_g, wide, at)
        met[want] += 1
    assert min(met) > 1000


def test_large_strides_without_a_loop(kgx):
    """Rows that interleave for 2^30 rows: known by arithmetic. 2 of 3 gaps of 8 bytes are dy's, or one element more is the gradient's too."""
    base = {**EMBED, "count": 2 ** 30, "vocab": 2 ** 30, "channels": 4, "tokens": 1 << 60, "workspace": 1 << 61, "dy": 1 << 40, "type": 1, "grad_type": 1}
    assert overlaps(kgx, "kg_embedding_backward", abi.EmbedArgs(**{**base, "ld_dy": 12, "grad": (1 << 40) + 8, "ld_grad": 24})) is None
    assert overlaps(kgx, "kg_embedding_backward", abi.EmbedArgs(**{**base, "ld_dy": 12, "grad": (1 << 40) + 18, "ld_grad": 24})) is not None
    # Strides of 12 and 13 elements meet after a few rows, of 4096 and 4097 after some thousand.
    for ld in (12, 4096):
        assert overlaps(kgx, "kg_embedding_backward", abi.EmbedArgs(**{**base, "ld_dy": ld, "grad": (1 << 40) + 8, "ld_grad": ld + 1})) is not None


class _OnGpu(torch.Tensor):
    """A CPU tensor that says it is on GPU 0."""

    is_cuda = property(lambda self: True)

    def get_device(self):
        return 0


def test_views_of_one_buffer_that_overlap(kgx, monkeypatch):
    learn = importlib.import_module("katago-rs_amd.learn")
    monkeypatch.setattr(learn, "_stream", lambda device: 0)
    raw = torch.zeros(4, 800).as_subclass(_OnGpu)
    index, top = torch.zeros(4, 3, dtype=torch.int32).as_subclass(_OnGpu), torch.zeros(4, 3).as_subclass(_OnGpu)
    with pytest.raises(kgx.KgError, match="grad must not overlap logits"):
        learn.distill_loss(raw[:, :400], index, top, grad=raw[:, 399:799])
    with pytest.raises(kgx.KgError, match="y must not overlap x"):
        learn.layer_norm(raw[:, :100], y=raw[:, 50:150])
    with pytest.raises(kgx.KgError, match="y must not overlap x"):
        learn.layer_norm(raw[:3], y=raw[1:])
    with pytest.raises(kgx.KgError, match="y must not overlap table"):
        learn.embedding(index[:3, 0].contiguous().as_subclass(_OnGpu), raw[:, :16], y=raw[1:, 8:24])
