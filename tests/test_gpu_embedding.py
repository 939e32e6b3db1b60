"""The embedding on the GPU against its definition in float64 (tests/student_ref.py).

Bounds. Forward: one product in float with scale rounded to float, 2 U, and the result's rounding. Backward: a row's tokens are added
in float, at most 600 one after another (never more than there are), such sums in double, then the scale's rounding and product and,
where it is added to what was there, that sum: (count + 4) U of the terms' sizes."""

import importlib
import math

import pytest
import torch

import learn_ref
import student_ref as ref
from test_gpu_distill import close

pytestmark = pytest.mark.gpu
U = learn_ref.U
TYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.fixture(scope="module")
def learn():
    return importlib.import_module("katago-rs_amd.learn")


def tokens_of(n, vocab, seed, kind="even"):
    g = torch.Generator().manual_seed(seed)
    if kind == "one":
        t = torch.full((n,), min(3, vocab - 1))
    elif kind == "likely":
        t = (vocab ** torch.rand(n, generator=g, dtype=torch.float64)).long().clamp(max=vocab) - 1
    else:
        t = torch.randint(0, vocab, (n,), generator=g)
    pad = torch.rand(n, generator=g) < 0.05
    return torch.where(pad, torch.tensor([-1, vocab, -2 ** 31, 2 ** 31 - 1])[torch.arange(n) % 4], t).int()


def forward(learn, tokens, table, scale):
    y = learn.embedding(tokens.cuda(), table.cuda(), scale=scale)
    on = (tokens >= 0) & (tokens < table.shape[0])
    want = torch.where(on[..., None], table.double()[tokens.long().clamp(0, table.shape[0] - 1)] * scale, 0.0)
    close(y, want, want.abs(), 2, "y")
    return y


def backward(learn, tokens, dy, vocab, scale=1.0, before=None, dtype=None):
    grad = None if before is None else before.cuda()
    got = learn.embedding_backward(dy.cuda(), tokens.cuda(), vocab, scale=scale, grad=grad, dtype=dtype, accumulate=grad is not None)
    want, size, count = ref.embedding_backward(dy, tokens, vocab, scale, before)
    close(got, want, size * (count.clamp(max=600) + 4)[:, None], 1, "grad")
    if before is not None:
        unnamed = count == 0
        assert torch.equal(got.cpu()[unnamed].nan_to_num(9.0), before[unnamed].nan_to_num(9.0))
    else:
        assert not got.cpu()[count == 0].any()
    return got


SIZES = [(1, 1, 1), (1, 5, 3), (3, 2, 8), (7, 100003, 4), (64, 1, 24), (65, 64, 1), (722, 362, 384), (1000, 511, 33), (1025, 512, 130),
         (4095, 513, 64), (4097, 50257, 72), (5000, 4, 96), (8193, 262143, 8), (20000, 262144, 5), (66000, 1000, 16), (66000, 3, 257),
         (200001, 70000, 12)]


@pytest.mark.parametrize("n,vocab,c", SIZES)
@pytest.mark.parametrize("dtype", TYPES)
def test_sizes(learn, n, vocab, c, dtype):
    g = torch.Generator().manual_seed(n + c)
    table = torch.randn(vocab, c, generator=g).to(dtype)
    dy = torch.randn(n, c, generator=g).to(dtype)
    for i, kind in enumerate(["even", "likely", "one"]):
        tokens = tokens_of(n, vocab, 3 * n + i, kind)
        if i < 2:
            forward(learn, tokens, table, math.sqrt(c))
        backward(learn, tokens, dy, vocab, (1.0, 0.3, 2.0 ** -9)[i], dtype=torch.float32 if i == 1 else None)


@pytest.mark.parametrize("dtype,wide", [(torch.float32, False), (torch.float16, True), (torch.bfloat16, False), (torch.bfloat16, True)])
@pytest.mark.parametrize("n,vocab,c", [(0, 30, 16), (1, 30, 16), (3000, 40, 96), (9000, 5000, 7), (70000, 6, 40)])
def test_accumulate(learn, n, vocab, c, dtype, wide):
    g = torch.Generator().manual_seed(n)
    dy, before = torch.randn(n, c, generator=g).to(dtype), torch.randn(vocab, c, generator=g).to(torch.float32 if wide else dtype)
    before[vocab // 2] = math.nan
    tokens = tokens_of(n, vocab, n, "likely")
    tokens[tokens == vocab // 2] = -1
    backward(learn, tokens, dy, vocab, 0.5, before)


def test_padding_alone_and_nothing(learn):
    tokens = torch.full((300,), -1, dtype=torch.int32)
    dy = torch.full((300, 16), math.nan)
    assert not backward(learn, tokens, dy, 40).any()
    assert not forward(learn, tokens, torch.randn(40, 16), 1.0).any()
    empty = torch.zeros(0, dtype=torch.int32)
    assert not backward(learn, empty, torch.zeros(0, 16), 40).any()
    assert forward(learn, empty, torch.randn(40, 16), 1.0).shape == (0, 16)


def test_padding_is_not_read(learn):
    for n in (50, 6000, 70000):
        tokens = tokens_of(n, 30, n)
        dy = torch.randn(n, 24)
        dy[(tokens < 0) | (tokens >= 30)] = math.nan
        backward(learn, tokens, dy, 30)


def test_strides_and_given_outputs(learn):
    g = torch.Generator().manual_seed(3)
    tokens = tokens_of(300, 50, 1).reshape(12, 25).cuda()
    table, dy = torch.randn(50, 60, generator=g).cuda(), torch.randn(12, 25, 70, generator=g).cuda()
    y = learn.embedding(tokens, table[:, 3:43].contiguous(), scale=2.0)
    room = torch.full((12, 25, 48), 7.0, device="cuda")
    out = learn.embedding(tokens, table[:, 3:43], scale=2.0, y=room[..., 1:41])
    assert torch.equal(out, y) and (room[..., 0] == 7).all() and (room[..., 41:] == 7).all()
    want = learn.embedding_backward(dy[..., 5:45].contiguous(), tokens, 50)
    room = torch.full((50, 48), 7.0, device="cuda")
    got = learn.embedding_backward(dy[..., 5:45], tokens, 50, grad=room[:, 1:41])
    assert torch.equal(got, want) and (room[:, 0] == 7).all() and (room[:, 41:] == 7).all()


def test_same_bits_each_time(learn):
    """The order of a row's additions is that of its tokens."""
    for n, vocab in ((700, 20), (6000, 900), (100000, 5), (100000, 20000)):
        tokens, dy = tokens_of(n, vocab, n, "likely").cuda(), torch.randn(n, 40).cuda()
        first = learn.embedding_backward(dy, tokens, vocab)
        for _ in range(3):
            assert torch.equal(learn.embedding_backward(dy, tokens, vocab), first)


def test_large_offsets(learn):
    """Rows whose elements lie past 2^31 of the table's and the gradient's first."""
    vocab, c = 1100000, 2048
    table = torch.zeros(vocab, c, dtype=torch.float16, device="cuda")
    table[-1], table[vocab // 2] = 2.0, 3.0
    tokens = torch.tensor([vocab - 1, 5, vocab // 2, vocab, -1], dtype=torch.int32, device="cuda")
    y = learn.embedding(tokens, table, scale=0.5)
    assert (y[0] == 1).all() and (y[2] == 1.5).all() and not y[[1, 3, 4]].any()
    dy = torch.ones(5, c, dtype=torch.float16, device="cuda")
    learn.embedding_backward(dy, tokens, vocab, grad=table)
    assert (table[-1] == 1).all() and (table[vocab // 2] == 1).all() and (table[5] == 1).all() and float(table.sum(dtype=torch.float64)) == 3 * c
