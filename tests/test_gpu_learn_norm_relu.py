"""Group norm with ReLU in 16 bits on every kernel that it has (boards, shares, rows); bounds as in test_gpu_learn_norm.py."""

import importlib

import pytest
import torch

from test_gpu_learn_norm import _case

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def learn():
    return importlib.import_module("katago-rs_amd.learn")


@pytest.mark.parametrize("shape", [(3, 361, 96, 8), (2, 1, 8, 2), (3, 5, 3, 3), (2, 5000, 96, 4), (2, 700, 1000, 1), (2, 9, 2056, 8),
                                   (1, 9001, 2, 1), (40, 37, 189, 21)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("mask", [False, True])
def test_group_norm_relu(learn, shape, dtype, mask):
    b, p, c, g = shape
    _case(learn, b, p, c, g, dtype, "relu", mask, 31 + p, ld=c + 1)
