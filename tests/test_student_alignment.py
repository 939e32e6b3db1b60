"""A student's operators refuse vectors of floats that do not lie at multiples of 4 bytes, before a device is touched."""

import ctypes

import pytest

import student_abi as abi
from test_student_overlap import DISTILL, LAYER, NO_DEVICE


def said(kgx, name, args):
    assert getattr(kgx.lib(), name)(NO_DEVICE, None, ctypes.byref(args)) == 1
    return kgx.lib().kg_last_error().decode()


@pytest.mark.parametrize("name,kind,base,vectors", [
    ("kg_distill_loss", abi.DistillArgs, DISTILL, ("loss", "weight", "teacher_lse")),
    ("kg_layer_norm", abi.LayerArgs, LAYER, ("gamma", "beta", "mean", "rstd")),
    ("kg_layer_norm_backward", abi.LayerArgs, LAYER, ("gamma", "mean", "rstd", "dgamma", "dbeta")),
])
def test_vectors_that_are_not_aligned(kgx, name, kind, base, vectors):
    for v in vectors:
        for by in (1, 2, 3):
            assert f"{v} is not aligned" in said(kgx, name, kind(**{**base, v: base[v] + (1 << 30) + by}))
        assert "aligned" not in said(kgx, name, kind(**{**base, v: base[v] + (1 << 30) + 4}))


def test_what_a_call_does_not_use_is_not_looked_at(kgx):
    assert "aligned" not in said(kgx, "kg_layer_norm", abi.LayerArgs(**{**LAYER, "rms": 1, "mean": 3, "dgamma": 5, "dbeta": 6}))
    assert "aligned" not in said(kgx, "kg_layer_norm_backward", abi.LayerArgs(**{**LAYER, "rms": 1, "mean": 3, "beta": 7}))


def test_sums_over_no_rows_are_written_too(kgx):
    """dgamma and dbeta: they are looked at without a row as well."""
    none = {**LAYER, "rows": 0, "x": None, "dy": None, "dx": None, "mean": None, "rstd": None, "workspace": None}
    assert "dgamma is not aligned" in said(kgx, "kg_layer_norm_backward", abi.LayerArgs(**{**none, "dgamma": LAYER["dgamma"] + 2}))
    assert "dbeta is not aligned" in said(kgx, "kg_layer_norm_backward", abi.LayerArgs(**{**none, "dbeta": LAYER["dbeta"] + 1}))
    assert "dgamma must not overlap dbeta" in said(kgx, "kg_layer_norm_backward", abi.LayerArgs(**{**none, "dbeta": LAYER["dgamma"] + 44}))
    text = said(kgx, "kg_layer_norm_backward", abi.LayerArgs(**none))
    assert "aligned" not in text and "overlap" not in text
