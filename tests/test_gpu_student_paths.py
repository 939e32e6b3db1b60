"""A student's operators at the sizes that choose their other variants: rows that a workgroup takes one after another, long rows that are
not cut, sums over many rows by slabs, tables that are not cleared beside the sort; and calls without a gradient. The bounds are those
of the operators' own tests."""

import importlib
import math

import pytest
import torch

import test_gpu_distill as distill
import test_gpu_embedding as embedding
import test_gpu_layer_norm as norm

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def learn():
    return importlib.import_module("katago-rs_amd.learn")


@pytest.mark.parametrize("n,v,dtype", [(389, 17001, torch.float32), (386, 33100, torch.bfloat16), (40, 70001, torch.float16),
                                       (390, 32736, torch.float32), (390, 32800, torch.float32), (385, 65473, torch.bfloat16)])
@pytest.mark.parametrize("rest", [False, True])
def test_long_rows(learn, n, v, dtype, rest):
    c = distill.make(n, v, 40, dtype, torch.float32, n, legal=rest, rest=rest, ld=6)
    c["index"][n // 2] = -1
    # (Columns whose chunks lie 4096 apart: lists that may be shared.)
    far = torch.arange(0, v, 4096 * 16 // c["z"].element_size())
    c["index"][1, :len(far)] = far.int()
    distill.check(learn, c)


@pytest.mark.parametrize("n,v,k,dtype", [(5, 3, 2, torch.float32), (9, 362, 24, torch.float32), (9, 362, 300, torch.float32),
                                         (9, 1100, 300, torch.bfloat16), (9, 2000, 50, torch.float16), (5, 9000, 50, torch.float32),
                                         (3, 30000, 50, torch.bfloat16), (3, 70001, 50, torch.float16), (389, 17001, 9, torch.float32)])
def test_no_gradient(learn, n, v, k, dtype):
    c = distill.make(n, v, k, dtype, torch.float32, v, legal=True, rest=True)
    c["legal"] = c["legal"].to(torch.uint8) * (1 + torch.arange(v) % 255).to(torch.uint8)  # (any byte but 0 is legal)
    for _ in range(2):
        assert distill.check(learn, c, want_grad=False).grad is None
    distill.check(learn, c)


# More rows than the most workgroups of a launch, 2^20, of one row or four. The rows come in copies: each has the first one's bits.
@pytest.mark.parametrize("n,v,dtype", [(1100000, 3, torch.float32), (4300000, 5, torch.float32), (4300000, 520, torch.bfloat16),
                                       (1100000, 4200, torch.bfloat16)])
def test_more_rows_than_workgroups(learn, n, v, dtype):
    few = 1000
    g = torch.Generator().manual_seed(v)
    z = torch.randn(few, v, generator=g).to(dtype).cuda()
    index = torch.randint(-1, v, (few, 3), generator=g).int().cuda()
    top, lse = torch.randn(few, 3, generator=g).cuda(), (2.5 + torch.rand(few, generator=g)).cuda()
    want = learn.distill_loss(z, index, top, teacher_lse=lse)
    of = lambda t: t.repeat((n // few,) + (1,) * (t.dim() - 1))  # noqa: E731
    got = learn.distill_loss(of(z), of(index), of(top), teacher_lse=of(lse))
    assert (got.loss.view(-1, few) == want.loss).all()
    assert (got.grad.view(-1, few, v) == want.grad).all()


def test_more_wide_rows_than_workgroups(learn):
    n, few, c = 1100000, 1000, 2200
    x = torch.randn(few, c, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    want = learn.layer_norm(x)
    got = learn.layer_norm(x.repeat(n // few, 1))
    for a, b in zip(got, want):
        assert (a.view(-1, *b.shape) == b).all()


@pytest.mark.parametrize("n,c,dtype", [
    (3001, 1100, torch.bfloat16), (2050, 2500, torch.float16), (1000, 1100, torch.float32), (2050, 2501, torch.float32),
    (600, 5001, torch.float32),                                                              # a workgroup takes several rows
    (33, 4104, torch.bfloat16), (333, 9001, torch.float16), (700, 4097, torch.bfloat16), (130, 20003, torch.float32),
    (1000, 8300, torch.float32)])                                                            # slabs, in parts of whole rows
def test_sums_over_many_rows(learn, n, c, dtype):
    for i, (rms, params, ld) in enumerate([(False, True, 0), (True, False, 5)]):
        norm.both(learn, n, c, dtype, n + i, rms, params, ld)


# Tables of more than 64 MB with more than a quarter as many tokens: rows that no token names are filled by marks or beside the sums.
@pytest.mark.parametrize("n,vocab,c,dtype,wide", [(20001, 70000, 257, torch.float32, False), (40000, 140000, 257, torch.bfloat16, False),
                                                  (20000, 70000, 250, torch.float16, True), (8192, 20000, 900, torch.float32, False),
                                                  (8200, 2000, 8500, torch.bfloat16, True)])
def test_large_tables(learn, n, vocab, c, dtype, wide):
    g = torch.Generator().manual_seed(n)
    dy = torch.randn(n, c, generator=g).to(dtype)
    grad_type = torch.float32 if wide else dtype
    for kind in ("even", "likely"):
        tokens = embedding.tokens_of(n, vocab, n, kind)
        got = embedding.backward(learn, tokens, dy, vocab, 0.5, dtype=grad_type)
        room = torch.full((vocab, c + 7), 7.0, dtype=grad_type, device="cuda")
        given = learn.embedding_backward(dy.cuda(), tokens.cuda(), vocab, scale=0.5, grad=room[:, 3:c + 3])
        assert torch.equal(given, got) and (room[:, :3] == 7).all() and (room[:, c + 3:] == 7).all()


@pytest.mark.parametrize("scale", [0.0, -1.5, 2.0 ** 100])
def test_scales(learn, scale):
    g = torch.Generator().manual_seed(2)
    tokens, table, dy = embedding.tokens_of(900, 70, 1), torch.randn(70, 36, generator=g), torch.randn(900, 36, generator=g)
    embedding.forward(learn, tokens, table, scale)
    embedding.backward(learn, tokens, dy, 70, scale)


@pytest.mark.parametrize("c", [16, 384, 5000, 40000])
def test_rows_past_floats_range(learn, c):
    """Infinity makes a row NaN, or with RMS norm 0 beside it; so large that the squares' sum is infinite: rstd 0."""
    x, beta = torch.randn(4, c), torch.randn(c)
    x[1, 3], x[2] = math.inf, 1e30 * x[2]
    for rms in (False, True):
        y, _, rstd = learn.layer_norm(x.cuda(), None, beta.cuda(), rms=rms)
        y, rstd = y.cpu(), rstd.cpu()
        assert torch.equal(y[2], beta) and rstd[2] == 0 and torch.isfinite(y[[0, 3]]).all() and torch.isnan(y[1, 3])
        if rms:
            others = torch.arange(c) != 3
            assert rstd[1] == 0 and torch.equal(y[1, others], beta[others])
        else:
            assert torch.isnan(y[1]).all()


@pytest.mark.parametrize("v", [3, 362, 2000, 20001])
@pytest.mark.parametrize("rest", [False, True])
def test_infinite_logits_and_weights_of_zero(learn, v, rest):
    c = distill.make(4, v, 3, torch.float32, torch.float32, v, rest=rest)
    c["weight"][0] = 0.0
    got = distill.check(learn, c)
    assert float(got.loss[0]) == 0 and not got.grad[0].any()
    c["weight"][2] = 0.0
    c["z"][2, c["index"][2, 0].long()] = -math.inf
    c["z"][1, v // 2] = math.inf
    got = distill.run(learn, c)
    assert math.isnan(float(got.loss[1])) and math.isnan(float(got.loss[2])) and math.isfinite(float(got.loss[3]))
    assert torch.isfinite(got.grad[3]).all()


# Up to 1024 tokens of up to 8192 rows and slabs of their columns go in one launch.
@pytest.mark.parametrize("vocab", [1, 2, 63, 511, 513, 1025, 8192, 8193, 32769])
@pytest.mark.parametrize("c,dtype,wide", [(1, torch.float32, False), (3, torch.bfloat16, True), (7, torch.float16, False), (31, torch.float16, False),
                                          (36, torch.bfloat16, True), (257, torch.float32, False), (1030, torch.bfloat16, False)])
def test_few_tokens(learn, vocab, c, dtype, wide):
    g = torch.Generator().manual_seed(vocab + c)
    grad_type = torch.float32 if wide else dtype
    before = torch.randn(vocab, c, generator=g).to(grad_type)
    before[vocab - 1] = math.inf
    for n, kind in ((1, "even"), (17, "one"), (600, "likely"), (1023, "even"), (1024, "one"), (1025, "likely")):
        tokens, dy = embedding.tokens_of(n, vocab, n, kind), torch.randn(n, c, generator=g).to(dtype)
        dy[(tokens < 0) | (tokens >= vocab)] = math.nan
        first = embedding.backward(learn, tokens, dy, vocab, 0.3, dtype=grad_type)
        assert torch.equal(embedding.backward(learn, tokens, dy, vocab, 0.3, dtype=grad_type), first)
        tokens[tokens == vocab - 1] = -1
        dy[tokens == -1] = math.nan
        embedding.backward(learn, tokens, dy, vocab, 0.3, before)
        room = torch.full((vocab, c + 7), 7.0, dtype=grad_type, device="cuda")
        given = learn.embedding_backward(dy.cuda(), tokens.cuda(), vocab, scale=0.3, grad=room[:, 3:c + 3])
        assert torch.equal(given, learn.embedding_backward(dy.cuda(), tokens.cuda(), vocab, scale=0.3, dtype=grad_type))
        assert (room[:, :3] == 7).all() and (room[:, c + 3:] == 7).all()


def test_marks_of_other_tokens(learn):
    """What a call left in its workspace, where the next one with other tokens marks its rows: by a graph whose workspace stays."""
    g = torch.Generator(device="cuda").manual_seed(4)
    dy = torch.randn(20000, 40, generator=g, device="cuda")
    tokens = torch.randint(0, 30000, (20000,), generator=g, device="cuda").int()
    grad = torch.empty(30000, 40, device="cuda")
    learn.embedding_backward(dy, tokens, 30000, grad=grad)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        learn.embedding_backward(dy, tokens, 30000, grad=grad)
    for k in range(5):
        tokens.copy_(torch.randint(0, (30000, 9, 15000, 40000, 1)[k], (20000,), generator=g, device="cuda") - k)
        grad.fill_(math.nan)
        graph.replay()
        want = learn.embedding_backward(dy, tokens, 30000)
        torch.cuda.synchronize()
        assert torch.equal(grad, want)
        named = torch.zeros(30000, dtype=torch.bool, device="cuda")
        named[tokens[(tokens >= 0) & (tokens < 30000)].long()] = True
        assert not grad[~named].any() and grad[named].any(1).all()
