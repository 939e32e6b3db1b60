"""A student's operators from their definitions, in float64 on the CPU, each with the sizes that its float error goes by."""

import math

import torch


def distill(logits, top_index, top_logits, legal=None, weight=None, scale=1.0, lse=None):
    """(loss, grad, sizes of their terms) of kg_distill_loss: a probability's relative error moves them by that much of their size."""
    n, v = logits.shape
    z = logits.double() * scale
    if legal is not None:
        z = z.masked_fill(~legal.bool(), -math.inf)
    loss, grad = torch.zeros(n, dtype=torch.float64), torch.zeros(n, v, dtype=torch.float64)
    lsize, gsize = torch.zeros(n, dtype=torch.float64), torch.zeros(n, v, dtype=torch.float64)
    for i in range(n):
        entries = {}
        for c, t in zip(top_index[i].tolist(), top_logits[i].double().tolist()):
            if 0 <= c < v and (legal is None or bool(legal[i, c])) and c not in entries:
                entries[c] = t
        if not entries or bool((z[i] == -math.inf).all()):
            continue
        at = torch.tensor(list(entries))
        t = torch.tensor(list(entries.values()), dtype=torch.float64) * scale
        if lse is None and bool((t == -math.inf).all()):
            continue
        lp = torch.log_softmax(z[i], 0)
        p = torch.exp(lp)
        lq = torch.log_softmax(t, 0) if lse is None else t - float(lse[i])
        q = torch.exp(lq)
        w = 1.0 if weight is None else float(weight[i])
        rest, share = 0.0, torch.zeros(v, dtype=torch.float64)  # of the others' mass, which may be below any number
        if lse is not None:
            others = lp.clone()
            others[at] = -math.inf
            if bool((others > -math.inf).any()):
                rest = float((1 - q.sum()).clamp(min=0))
                if rest > 0:
                    left = torch.logsumexp(others, 0)
                    loss[i] += rest * (math.log(rest) - left)
                    lsize[i] += rest * (abs(math.log(rest)) + left.abs() + 1)
                    share = rest * torch.softmax(others, 0)
        d = torch.where(q > 0, lq - lp[at], 0.0)
        loss[i] += (q * d).sum()
        lsize[i] += (q * (1 + torch.where(q > 0, d.abs(), 0.0))).sum()
        mass = q.sum() + rest
        g, size = mass * p - share, mass * p + share
        g[at], size[at] = mass * p[at] - q, mass * p[at] + q
        loss[i], lsize[i] = w * loss[i], abs(w) * lsize[i]
        grad[i], gsize[i] = w * scale * g, abs(w) * scale * size
    return loss, grad, lsize, gsize


def layer_norm(x, gamma=None, beta=None, eps=1e-5, rms=False):
    """(y, mean, rstd, h) of kg_layer_norm on rows [n, c]."""
    x = x.double()
    mean = torch.zeros(x.shape[0], dtype=torch.float64) if rms else x.mean(1)
    rstd = 1 / torch.sqrt(((x - mean[:, None]) ** 2).mean(1) + eps)
    h = (x - mean[:, None]) * rstd[:, None]
    y = h if gamma is None else h * gamma.double()
    return y if beta is None else y + beta.double(), mean, rstd, h


def layer_norm_backward(dy, x, mean, rstd, gamma=None):
    """(dx, dgamma, dbeta, and the sizes of their terms) of kg_layer_norm_backward for the given statistics (mean None: RMS)."""
    dy, rstd = dy.double(), rstd.double()[:, None]
    h = (x.double() - (0.0 if mean is None else mean.double()[:, None])) * rstd
    d = dy if gamma is None else dy * gamma.double()
    m2, a2 = (d * h).mean(1, keepdim=True), (d * h).abs().mean(1, keepdim=True)
    m1, a1 = d.mean(1, keepdim=True), d.abs().mean(1, keepdim=True)
    if mean is None:
        m1, a1 = 0.0, 0.0
    dx = rstd * (d - m1 - h * m2)
    return (dx, (dy * h).sum(0), dy.sum(0)), (rstd * (d.abs() + a1 + h.abs() * a2), (dy * h).abs().sum(0), dy.abs().sum(0))


def embedding_backward(dy, tokens, vocab, scale=1.0, before=None):
    """(grad, size of its terms, tokens of each row)."""
    tokens, dy = tokens.reshape(-1).long(), dy.double().reshape(tokens.numel(), dy.shape[-1])
    on = (tokens >= 0) & (tokens < vocab)
    grad = torch.zeros(vocab, dy.shape[1], dtype=torch.float64)
    size = grad.index_add(0, tokens[on], dy[on].abs()) * abs(scale)
    grad = grad.index_add(0, tokens[on], dy[on]) * scale
    if before is not None:
        grad, size = grad + before.double(), size + before.double().abs()
    return grad, size, torch.bincount(tokens[on], minlength=vocab)
