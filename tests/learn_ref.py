"""The learning operators from their definitions, in float64 on the CPU, and float32 restatements of the 8-bit moments' rounding
(every step of it is exact or one rounding, so the codes are compared bit for bit)."""

import numpy as np
import torch

U = 2.0 ** -24  # half a step of float32, relative


def half_step(dtype):
    """A rounding to dtype is off by at most this much, relative, and by `least` where the result is subnormal."""
    least = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}[dtype]
    return torch.finfo(dtype).eps / 2, least


def log_softmax(z, legal=None):
    z = z.double().clone()
    if legal is not None:
        z[~legal.bool()] = -torch.inf
    top = z.max(1, keepdim=True).values
    e = torch.exp(z - torch.where(top == -torch.inf, 0.0, top))
    e[z == -torch.inf] = 0
    return torch.where(z == -torch.inf, -torch.inf, z - top - torch.log(e.sum(1, keepdim=True)))


def policy(logits, actions, old, adv, legal=None, weight=None, scale=1.0, clip=(0.2, 0.2), kl_coef=0.0, ref=None, ref_logp=None):
    """(loss, logp, kl, grad, bound of grad's float error in units of U * K) of kg_policy_loss."""
    n, v = logits.shape
    lsm = log_softmax(logits.double() * scale, legal)
    p = torch.exp(lsm)
    loss, logp, kl = (torch.zeros(n, dtype=torch.float64) for _ in range(3))
    grad, size = torch.zeros(n, v, dtype=torch.float64), torch.zeros(n, v, dtype=torch.float64)
    rsm = None if ref is None else log_softmax(ref.double() * scale, legal)
    for i in range(n):
        a = int(actions[i])
        if not 0 <= a < v:
            continue
        logp[i] = lsm[i, a]
        if logp[i] == -torch.inf:
            continue
        w = 1.0 if weight is None else float(weight[i])
        ratio, ad = torch.exp(lsm[i, a] - float(old[i])), float(adv[i])
        free, held = ratio * ad, ratio.clamp(1 - clip[0], 1 + clip[1]) * ad
        c = -free if free <= held else torch.zeros(())
        hot = torch.zeros(v, dtype=torch.float64)
        hot[a] = 1
        extra, esize = 0.0, 0.0
        if ref_logp is not None:
            d = float(ref_logp[i]) - lsm[i, a]
            kl[i] = torch.exp(d) - d - 1
            c = c + kl_coef * (1 - torch.exp(d))
        if ref is not None:
            d = torch.where(p[i] > 0, lsm[i] - rsm[i], 0.0)
            kl[i] = (p[i] * d).sum()
            extra = kl_coef * p[i] * (d - kl[i])
            esize = abs(kl_coef) * p[i] * (d.abs() + kl[i].abs() + 1)
        loss[i] = w * (kl_coef * kl[i] - min(free, held))
        grad[i] = w * scale * (c * (hot - p[i]) + extra)
        size[i] = abs(w * scale) * (abs(c) * (hot + p[i]) + esize)
    return loss, logp, kl, grad, size


def preference(logits, labels, offsets, ref_logp, beta=0.1, smooth=0.0, average=False, weight=None):
    """(loss, margin, seq_logp, grad, its size) of kg_preference_loss."""
    t, v = logits.shape
    lsm = log_softmax(logits)
    p = torch.exp(lsm)
    pairs = (len(offsets) - 1) // 2
    seq, rows = torch.zeros(2 * pairs, dtype=torch.float64), []
    for q in range(2 * pairs):
        rows.append([i for i in range(int(offsets[q]), int(offsets[q + 1])) if 0 <= int(labels[i]) < v])
        s = sum((lsm[i, int(labels[i])] for i in rows[q]), torch.zeros((), dtype=torch.float64))
        seq[q] = s / max(1, len(rows[q])) if average else s
    loss, margin = torch.zeros(pairs, dtype=torch.float64), torch.zeros(pairs, dtype=torch.float64)
    grad, size = torch.zeros(t, v, dtype=torch.float64), torch.zeros(t, v, dtype=torch.float64)
    ls = torch.nn.functional.logsigmoid
    for i in range(pairs):
        h = beta * ((seq[2 * i] - float(ref_logp[2 * i])) - (seq[2 * i + 1] - float(ref_logp[2 * i + 1])))
        w = 1.0 if weight is None else float(weight[i])
        margin[i] = h
        loss[i] = -w * ((1 - smooth) * ls(h) + smooth * ls(-h))
        dh = w * beta * (smooth * torch.sigmoid(h) - (1 - smooth) * torch.sigmoid(-h))
        for q, sign in ((2 * i, 1.0), (2 * i + 1, -1.0)):
            for r in rows[q]:
                f = sign * dh / (max(1, len(rows[q])) if average else 1)
                grad[r] = -f * p[r]
                grad[r, int(labels[r])] += f
                size[r] = f.abs() * p[r]
                size[r, int(labels[r])] += f.abs()
    return loss, margin, seq, grad, size


def group_norm(x, groups, gamma=None, beta=None, mask=None, eps=1e-5, act="identity", dy=None, stats=None):
    """kg_group_norm in float64: (y, mean, rstd); with dy, (dx, dgamma, dbeta) for the given (mean, rstd)."""
    b, c = x.shape[0], x.shape[-1]
    x = x.double().reshape(b, -1, groups, c // groups)
    on = torch.ones(x.shape[:2], dtype=torch.bool) if mask is None else mask.reshape(b, -1) != 0
    on = on[:, :, None, None]
    gm = (torch.ones(c) if gamma is None else gamma).double().reshape(groups, -1)
    bt = (torch.zeros(c) if beta is None else beta).double().reshape(groups, -1)
    x = torch.where(on, x, 0.0)
    n = (on.sum((1, 3)).double() * (c // groups)).clamp(min=1)
    if stats is None:
        mean = x.sum((1, 3)) / n
        var = torch.where(on, (x - mean[:, None, :, None]) ** 2, 0.0).sum((1, 3)) / n
        rstd = 1 / torch.sqrt(var + eps)
    else:
        mean, rstd = (s.double() for s in stats)
    xh = torch.where(on, (x - mean[:, None, :, None]) * rstd[:, None, :, None], 0.0)
    a = (xh * gm + bt).requires_grad_(dy is not None)
    f = torch.nn.functional
    y = {"identity": lambda t: t * 1, "relu": f.relu, "mish": f.mish, "silu": f.silu}[act](a)
    if dy is None:
        return torch.where(on, y, 0.0).reshape(b, -1, c), mean, rstd
    da, = torch.autograd.grad(y, a, torch.where(on, dy.double().reshape(x.shape), 0.0))
    d, k = da * gm, n[:, None, :, None]
    m1, m2 = d.sum((1, 3), keepdim=True) / k, (d * xh).sum((1, 3), keepdim=True) / k
    dx = torch.where(on, rstd[:, None, :, None] * (d - m1 - xh * m2), 0.0)
    return dx.reshape(b, -1, c), (da * xh).sum((0, 1)).reshape(-1), da.sum((0, 1)).reshape(-1)


# ---- the 8-bit moments, in float32 as the library rounds them ----

def mix32(x):
    x = np.asarray(x, np.uint64) & 0xFFFFFFFF
    x = ((x ^ (x >> 16)) * 0x9E3779B9) & 0xFFFFFFFF
    x = ((x ^ (x >> 15)) * 0xB7E15163) & 0xFFFFFFFF
    return x ^ (x >> 16)


def noise(index, seed):
    index = np.asarray(index, np.uint64)
    h = mix32(index + mix32((index >> np.uint64(32)) + mix32(seed)))
    return (h & 0xFFFF).astype(np.float32) * np.float32(2 ** -16), (h >> 16).astype(np.float32) * np.float32(2 ** -16)


def encode(x, u, signed):
    """(codes, exponents) of float32 x [blocks, 256]."""
    bits, bias, least, carry = (3, 135, 9, 0x1FFFFF) if signed else (5, 138, 12, 0x03FFFF)
    mag = np.abs(x)
    top = mag.view(np.uint32).max(1)
    exp = np.clip((top + np.uint32(carry)) >> 23, least, 255).astype(np.int64)
    y = (mag * np.exp2(bias - np.minimum(exp, 254).astype(np.float64)).astype(np.float32)[:, None]).astype(np.float32)
    low = -6 if signed else 5
    e = np.maximum((y.view(np.uint32) >> 23).astype(np.int64) - 127, low)
    t = (y * np.exp2((bits - e).astype(np.float64)).astype(np.float32)).astype(np.float32)
    n = np.floor(t + u).astype(np.int64)
    if not signed:
        n = np.where((n == 0) & (y > 0), 1, n)
    code = ((e - low) << bits) + n
    if signed:
        code = code | np.where(np.signbit(x), 0x80, 0)
    return code.astype(np.uint8), exp.astype(np.uint8)


def decode_m(code, exp):
    c = code.astype(np.int64)
    e, f = (c >> 3) & 15, c & 7
    v = np.where(e > 0, (8 + f) * np.exp2(e - 10.0), f * np.exp2(-9.0)) * np.where(c & 0x80, -1.0, 1.0)
    return (v * np.exp2(exp.astype(np.float64) - 135)[:, None]).astype(np.float32)


def decode_v(code, exp):
    c = code.astype(np.int64)
    n = np.where(c < 64, c, ((c & 31) | 32) << np.maximum((c >> 5) - 1, 0))
    return (n * np.exp2(exp.astype(np.float64) - 138)[:, None]).astype(np.float32)


def adamw(p, g, m, v, step, lr=1e-3, b1=0.9, b2=0.999, eps=1e-8, wd=0.0, grad_scale=1.0):
    """One step in float64: (p, m, v)."""
    g = g.double() * grad_scale
    m = b1 * m.double() + (1 - b1) * g
    v = b2 * v.double() + (1 - b2) * g * g
    upd = lr / (1 - b1 ** step) * m / (torch.sqrt(v / (1 - b2 ** step)) + eps)
    return p.double() * (1 - lr * wd) - upd, m, v
