"""The measured cases of the operators that a student network learns with (katago-rs_amd/learn.py): the distillation loss from a
teacher's top logits with its gradient, layer norm and RMS norm forward and backward, and the embedding of tokens with its
gradient.

Sizes are those of the networks' own policy rows (362 moves inside raw rows of 1094 floats), boards (361 points) and channel
counts, and generic ones: vocabularies, token counts and widths of a language policy. `run` computes a case with elementary
torch operations in 32 bits, or, where `own` is set, with the library's operators.
"""

import importlib
import math

import numpy as np
import torch

own = False

MOVES = 362            # a board's policy row, pass last
ROW = 1094             # floats of a raw row that holds two policy channels, value, scores and ownership
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-5
DEV = "cuda"


# ------------------------------------------------------------------------------------------------------------ cases

def listed():
    def distill(name, rows, vocab, ld, dtype, k, top, rest, legal):
        return {"name": name, "op": "distill", "rows": rows, "vocab": vocab, "ld": ld, "dtype": dtype, "k": k,
                "top_type": top, "rest": rest, "legal": legal}

    def norm(name, back, rows, channels, dtype, rms):
        return {"name": name, "op": "norm_back" if back else "norm", "rows": rows, "channels": channels, "dtype": dtype,
                "rms": rms}

    def embed(name, back, tokens, vocab, channels, dtype, wide, even):
        return {"name": name, "op": "embed_back" if back else "embed", "tokens": tokens, "vocab": vocab,
                "channels": channels, "dtype": dtype, "wide": wide, "even": even}

    return [
        # One batch of positions as the network answers it, against the larger network's best moves.
        distill("distill-board-b32", 32, MOVES, ROW, "f32", 24, "f32", False, True),
        # Tokens of a language policy, an odd count; the teacher's rows were stored as 64 logits and their normaliser.
        distill("distill-tokens-bf16", 4093, 32768, 32768, "bf16", 64, "f16", True, False),
        # A short batch over a large vocabulary of odd size.
        distill("distill-f16-odd", 301, 100003, 100003, "f16", 50, "bf16", True, False),
        # The points of one batch of boards through a transformer trunk.
        norm("norm-trunk-bf16", False, 32 * 361, 384, "bf16", False),
        # Wide rows of an odd length.
        norm("norm-wide-f16-odd", False, 2047, 10007, "f16", False),
        # A small trunk's gradient, float.
        norm("norm-back-f32", True, 8 * 361, 128, "f32", False),
        # A large learning batch of tokens, RMS norm as the transformer networks have it.
        norm("rms-back-bf16", True, 65521, 1024, "bf16", True),
        # Move sequences of a few games.
        embed("embed-moves-f32", False, 722, MOVES, 384, "f32", False, True),
        # Tokens of a language policy, a large batch.
        embed("embed-tokens-bf16", False, 65536, 50257, 1024, "bf16", False, False),
        # The gradients of both; the large one in float for masters, the small one where few rows are named often.
        embed("embed-back-moves-f32", True, 722, MOVES, 384, "f32", False, True),
        embed("embed-back-tokens-bf16", True, 65536, 50257, 1024, "bf16", True, False),
        # A step's worth of tokens over a large vocabulary, most of whose rows stay 0.
        embed("embed-back-sparse-f16", True, 5003, 100003, 512, "f16", False, False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["distill", "norm", "norm_back", "embed", "embed_back"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    if op == "distill":
        board = rng.random() < 0.4
        vocab = MOVES if board else _log(rng, 2, 131072)
        most = max(1, min(16384, 130000000 // vocab))
        return {"op": op, "rows": _log(rng, 1, most), "vocab": vocab,
                "ld": rng.choice([MOVES, ROW]) if board else vocab + rng.choice([0, 0, 1, 6, 8]), "dtype": dtype,
                "k": _log(rng, 1, min(256, vocab)), "top_type": rng.choice(["f32", "f16", "bf16"]),
                "rest": rng.random() < 0.5, "legal": board or rng.random() < 0.2}
    if op in ("norm", "norm_back"):
        channels = _log(rng, 16, 16384)
        return {"op": op, "rows": _log(rng, 1, min(262144, 60000000 // channels)), "channels": channels, "dtype": dtype,
                "rms": rng.random() < 0.5}
    channels = _log(rng, 1, 4096)
    return {"op": op, "tokens": _log(rng, 1, min(1048576, 60000000 // channels)),
            "vocab": _log(rng, 2, min(131072, 50000000 // channels)), "channels": channels, "dtype": dtype,
            "wide": op == "embed_back" and rng.random() < 0.5, "even": rng.random() < 0.3}


# ----------------------------------------------------------------------------------------------------------- inputs

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device=DEV, dtype=dtype)


def _rand(g, *shape):
    return torch.rand(*shape, generator=g, device=DEV)


def _prepare_distill(c, g):
    n, v, k, t = c["rows"], c["vocab"], c["k"], TYPES[c["dtype"]]
    z = _randn(g, n, c["ld"], dtype=t).mul_(2)[:, :v]
    s = {"logits": z, "legal": None, "lse": None, "scale": 0.5 if c["rest"] else 1.0}
    # The teacher agrees in the main; it has no illegal moves.
    teacher = z.float() + 0.7 * _randn(g, n, v)
    if c["legal"]:
        s["legal"] = _rand(g, n, v) < 0.7
        s["legal"].scatter_(1, teacher.argmax(1, keepdim=True), True)
        teacher.masked_fill_(~s["legal"], -math.inf)
    top, index = teacher.topk(k, 1)
    top = top.to(TYPES[c["top_type"]])
    # What was stored is rounded; the normaliser is of all columns.
    lse = torch.logsumexp(teacher.scatter(1, index, top.float()).mul_(s["scale"]), 1)
    if c["rest"]:
        s["lse"] = lse
    # Some rows were stored with fewer entries, and a padded batch leaves rows out.
    count = torch.where(_rand(g, n) < 0.2, (_rand(g, n) * k).long() + 1, k)
    if n > 1:
        count = torch.where(_rand(g, n) < 0.03, 0, count)
    at = torch.arange(k, device=DEV)
    s["top_index"] = torch.where((at < count[:, None]) & (top > -math.inf), index, -1).int()
    s["top_logits"] = top
    # (Gradients of half precision are scaled, as a training loop does, or most would fall below its range.)
    s["weight"] = _rand(g, n) * (64.0 if c["dtype"] == "f16" else 1 / n)
    return s


def _prepare_norm(c, g):
    n, ch, t = c["rows"], c["channels"], TYPES[c["dtype"]]
    s = {"rms": c["rms"]}
    spread, shift = 0.5 + _rand(g, ch), _randn(g, ch)
    s["x"] = ((_randn(g, n, ch) * spread + shift) * (0.5 + _rand(g, n, 1))).to(t)
    s["gamma"], s["beta"] = 1 + 0.2 * _randn(g, ch), None if c["rms"] else 0.3 * _randn(g, ch)
    if c["op"] == "norm_back":
        s["dy"] = _randn(g, n, ch, dtype=t)
        s["mean"], s["rstd"] = _stats(s["x"].double(), c["rms"])
        s["mean"], s["rstd"] = None if c["rms"] else s["mean"].float(), s["rstd"].float()
    return s


def _likely(c):
    """The probability of each token: moves are about even, words are not."""
    p = np.ones(c["vocab"]) if c["even"] else 1 / (np.arange(c["vocab"]) + 3.0)
    return p / p.sum()


def _prepare_embed(c, g):
    n, v, ch, t = c["tokens"], c["vocab"], c["channels"], TYPES[c["dtype"]]
    edges = torch.from_numpy(np.cumsum(_likely(c))).to(DEV)
    tokens = torch.searchsorted(edges, torch.rand(n, generator=g, device=DEV, dtype=torch.float64)).clamp(max=v - 1).int()
    if n > 1:  # padding names no token
        tokens = torch.where(_rand(g, n) < 0.02, -1, tokens)
    s = {"tokens": tokens, "scale": math.sqrt(ch)}
    if c["op"] == "embed":
        s["table"] = (_randn(g, v, ch) / math.sqrt(ch)).to(t)
    else:
        s["dy"], s["vocab"] = _randn(g, n, ch, dtype=t).mul_(0.125), v
        s["grad_type"] = torch.float32 if c["wide"] else t
    return s


def prepare(case, seed):
    g = _gen(seed)
    s = {"distill": _prepare_distill, "norm": _prepare_norm, "norm_back": _prepare_norm, "embed": _prepare_embed,
         "embed_back": _prepare_embed}[case["op"]](case, g)
    s["op"] = case["op"]
    return s


# ------------------------------------------------------------------------------------------------------ plain forms

def _plain_distill(s):
    z, scale, dtype = s["logits"].float(), s["scale"], s["logits"].dtype
    n, v = z.shape
    if s["legal"] is not None:
        z = torch.where(s["legal"], z, -math.inf)
    # An entry counts where it names a legal column that none before it names.
    index = s["top_index"].long()
    counts = (index >= 0) & (index < v)
    at = torch.where(counts, index, 0)
    if s["legal"] is not None:
        counts = counts & s["legal"].gather(1, at)
    order = torch.where(counts, index, -1).sort(dim=1, stable=True)
    again = torch.cat([torch.zeros_like(counts[:, :1]), order.values.diff(dim=1) == 0], 1)
    counts = counts & ~torch.zeros_like(counts).scatter(1, order.indices, again)
    zt = z.gather(1, at).double() * scale
    listed = torch.zeros(n, v + 1, dtype=torch.bool, device=DEV).scatter_(1, torch.where(counts, at, v), True)[:, :v]
    # The columns that are not listed relative to their own maximum; a row's few scalars in 64 bits.
    other = torch.where(listed, -math.inf, z)
    top = other.max(1, keepdim=True).values
    e = torch.exp((other - torch.where(top == -math.inf, 0.0, top)) * scale)
    total = e.sum(1, keepdim=True).double()
    lo = torch.where(total > 0, top.double() * scale + torch.log(total), -math.inf)
    own_max = torch.maximum(torch.where(counts, zt, -math.inf).max(1, keepdim=True).values, lo)
    own_max = torch.where(own_max == -math.inf, 0.0, own_max)
    lse = own_max + torch.log((torch.where(counts, torch.exp(zt - own_max), 0.0)).sum(1, keepdim=True) + torch.exp(lo - own_max))
    t = torch.where(counts, s["top_logits"].double() * scale, -math.inf)
    if s["lse"] is None:
        t_max = t.max(1, keepdim=True).values
        t = t - torch.where(t_max == -math.inf, 0.0, t_max)
        norm = torch.log(torch.exp(t).sum(1, keepdim=True))
        part = counts.any(1, keepdim=True) & (norm > -math.inf)
    else:
        norm, part = s["lse"].double()[:, None], counts.any(1, keepdim=True)
    part = part & (lse > -math.inf)
    lq = torch.where(counts & part, t - norm, -math.inf)
    q = torch.exp(lq)
    rest = torch.zeros_like(lse) if s["lse"] is None else (1 - q.sum(1, keepdim=True)).clamp(min=0)
    rest = torch.where(lo > -math.inf, rest, 0.0)
    mass = q.sum(1, keepdim=True) + rest
    loss = torch.where(q > 0, q * (lq - (zt - lse)), 0.0).sum(1, keepdim=True)
    loss = loss + torch.where(rest > 0, rest * (torch.log(rest) - (lo - lse)), 0.0)
    w = s["weight"].double()[:, None]
    each = w * scale * (mass * torch.exp(lo - lse) - rest) / torch.where(total > 0, total, 1.0)
    hot = w * scale * (mass * torch.exp(zt - lse) - q)
    grad = torch.where(part, e * each.float(), 0.0)
    grad.scatter_add_(1, at, torch.where(counts & part, hot, 0.0).float())
    return {"loss": torch.where(part, w * loss, 0.0).squeeze(1).float(), "grad": grad.to(dtype)}


def _stats(x, rms):
    mean = torch.zeros_like(x[:, 0]) if rms else x.sum(1) / x.shape[1]
    d = x - mean[:, None]
    return mean, 1 / torch.sqrt((d * d).sum(1) / x.shape[1] + EPS)


def _plain_norm(s):
    x = s["x"].float()
    mean, rstd = _stats(x, s["rms"])
    y = (x - mean[:, None]) * rstd[:, None] * s["gamma"]
    if s["beta"] is not None:
        y = y + s["beta"]
    out = {"y": y.to(s["x"].dtype), "rstd": rstd}
    return out if s["rms"] else out | {"mean": mean}


def _plain_norm_back(s):
    dy, rstd = s["dy"].float(), s["rstd"][:, None]
    h = s["x"].float()
    h = (h if s["mean"] is None else h - s["mean"][:, None]) * rstd
    d = dy * s["gamma"]
    dx = d - h * ((d * h).sum(1, keepdim=True) / d.shape[1])
    if s["mean"] is not None:
        dx = dx - d.sum(1, keepdim=True) / d.shape[1]
    return {"dx": (dx * rstd).to(s["x"].dtype), "dgamma": (dy * h).sum(0), "dbeta": dy.sum(0)}


def _plain_embed(s):
    tokens = s["tokens"].long()
    named = (tokens >= 0) & (tokens < s["table"].shape[0])
    y = s["table"][torch.where(named, tokens, 0)].float() * s["scale"]
    return torch.where(named[:, None], y, 0.0).to(s["table"].dtype)


def _plain_embed_back(s):
    tokens, vocab = s["tokens"].long(), s["vocab"]
    at = torch.where((tokens >= 0) & (tokens < vocab), tokens, vocab)
    grad = torch.zeros(vocab + 1, s["dy"].shape[1], device=DEV).index_add_(0, at, s["dy"].float())[:vocab]
    return (grad * s["scale"]).to(s["grad_type"])


# -------------------------------------------------------------------------------------------------------------- run

def _run_own(s):
    learn = importlib.import_module("katago-rs_amd.learn")
    if s["op"] == "distill":
        r = learn.distill_loss(s["logits"], s["top_index"], s["top_logits"], legal=s["legal"], weight=s["weight"],
                               logit_scale=s["scale"], teacher_lse=s["lse"])
        return {"loss": r.loss, "grad": r.grad}
    if s["op"] == "norm":
        y, mean, rstd = learn.layer_norm(s["x"], s["gamma"], s["beta"], eps=EPS, rms=s["rms"])
        return {"y": y, "rstd": rstd} if s["rms"] else {"y": y, "rstd": rstd, "mean": mean}
    if s["op"] == "norm_back":
        dx, dgamma, dbeta = learn.layer_norm_backward(s["dy"], s["x"], s["mean"], s["rstd"], s["gamma"])
        return {"dx": dx, "dgamma": dgamma, "dbeta": dbeta}
    if s["op"] == "embed":
        return learn.embedding(s["tokens"], s["table"], scale=s["scale"])
    return learn.embedding_backward(s["dy"], s["tokens"], s["vocab"], scale=s["scale"], dtype=s["grad_type"])


def run(state):
    if own:
        return _run_own(state)
    return {"distill": _plain_distill, "norm": _plain_norm, "norm_back": _plain_norm_back, "embed": _plain_embed,
            "embed_back": _plain_embed_back}[state["op"]](state)


# ------------------------------------------------------------------------------------------------------------- work

def work(case):
    """Bytes and operations of one pass: each input read once, each output written once."""
    t = SIZE[case["dtype"]]
    if case["op"] == "distill":
        n, v = case["rows"], case["vocab"]
        return {"bytes": n * v * (2 * t + (1 if case["legal"] else 0)) + n * case["k"] * (4 + SIZE[case["top_type"]]) + 12 * n,
                "flops": n * v * 8}
    if case["op"] in ("norm", "norm_back"):
        n, ch, back = case["rows"], case["channels"], case["op"] == "norm_back"
        return {"bytes": n * ch * t * (3 if back else 2) + 8 * n + ch * (12 if back else 8), "flops": n * ch * (14 if back else 8)}
    n, v, ch = case["tokens"], case["vocab"], case["channels"]
    if case["op"] == "embed":
        # Each row that is named is read once.
        seen = float((-np.expm1(0.98 * n * np.log1p(-np.minimum(_likely(case), 1 - 1e-9)))).sum())
        return {"bytes": (n + min(seen, n)) * ch * t + 4 * n, "flops": n * ch}
    return {"bytes": n * ch * t + v * ch * (4 if case["wide"] else t) + 4 * n, "flops": n * ch + v * ch}


# ------------------------------------------------------------------------------------------------------------ exact

def _exact_distill(s):
    z = s["logits"].double().requires_grad_()
    n, v = z.shape
    zs = z * s["scale"]
    if s["legal"] is not None:
        zs = zs.masked_fill(~s["legal"], -math.inf)
    lsm = torch.log_softmax(zs, 1)
    index = s["top_index"].long()
    part = (index >= 0).any(1)
    loss = torch.zeros(n, device=DEV, dtype=torch.float64)
    if bool(part.any()):
        lsm, index = lsm[part], index[part]
        there = index >= 0
        at = index.clamp(min=0)
        t = (s["top_logits"].double()[part] * s["scale"]).masked_fill(~there, -math.inf)
        lq = torch.log_softmax(t, 1) if s["lse"] is None else t - s["lse"].double()[part, None]
        value = torch.special.xlogy(lq.exp(), lq.exp()).sum(1)
        value = value - (lq.exp() * torch.where(there, lsm.gather(1, at), 0.0)).sum(1)
        if s["lse"] is not None:
            free = torch.isfinite(lsm.detach())
            rows = torch.arange(index.shape[0], device=DEV)[:, None].expand_as(index)
            free[rows[there], index[there]] = False
            r = torch.where(free.any(1), (1 - lq.exp().sum(1)).clamp(min=0), 0.0)
            left = torch.logsumexp(torch.where(free | ~free.any(1, keepdim=True), lsm, -math.inf), 1)
            value = value + torch.special.xlogy(r, r) - torch.where(r > 0, r * left, 0.0)
        loss = loss.index_put((part.nonzero().squeeze(1),), s["weight"].double()[part] * value)
    grad, = torch.autograd.grad(loss.sum() + 0.0 * z[:, 0].sum(), z)
    return {"loss": loss.detach(), "grad": grad}


def _exact_norm(s, back):
    x, gamma = s["x"].double(), s["gamma"].double()
    if not back:
        mean = x.mean(1)
        rstd = (x.square().mean(1) if s["rms"] else x.var(1, unbiased=False)).add(EPS).rsqrt()
        y = gamma * rstd[:, None] * (x if s["rms"] else x - mean[:, None])
        return {"y": y, "rstd": rstd} if s["rms"] else {"y": y + s["beta"].double(), "rstd": rstd, "mean": mean}
    rstd, dy = s["rstd"].double()[:, None], s["dy"].double()
    h = rstd * (x if s["rms"] else x - s["mean"].double()[:, None])
    g = dy * gamma
    g_mean = 0.0 if s["rms"] else g.mean(1, keepdim=True)
    return {"dx": rstd * (g - g_mean - h * (g * h).mean(1, keepdim=True)), "dgamma": (dy * h).sum(0), "dbeta": dy.sum(0)}


def _exact_embed(s):
    tokens = s["tokens"].long()
    if s["op"] == "embed":
        y = torch.zeros(tokens.numel(), s["table"].shape[1], device=DEV, dtype=torch.float64)
        y[tokens >= 0] = s["scale"] * s["table"].double()[tokens[tokens >= 0]]
        return y
    # The sums of the tokens in order, as differences of running sums at the ends of each token's share.
    order = tokens.argsort(stable=True)
    ends = torch.searchsorted(tokens[order], torch.arange(-1, s["vocab"], device=DEV), right=True)
    grad = torch.empty(s["vocab"], s["dy"].shape[1], device=DEV, dtype=torch.float64)
    step = max(1, 20000000 // max(1, tokens.numel()))
    for c in range(0, s["dy"].shape[1], step):
        running = s["dy"][:, c:c + step].double()[order].cumsum(0)
        running = torch.cat([torch.zeros_like(running[:1]), running])
        grad[:, c:c + step] = s["scale"] * running[ends].diff(dim=0)
    return grad


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "distill":
        return _exact_distill(s)
    if case["op"] in ("norm", "norm_back"):
        return _exact_norm(s, case["op"] == "norm_back")
    return _exact_embed(s)
