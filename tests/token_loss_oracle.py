"""The token losses in 64 bits, written from their definitions one sequence at a time and differentiated by
autograd, and how far fp32 arithmetic may be from them."""

import math

import torch


def log_probs(x, labels, ignore=-100, temperature=1.0):
    """x in 64 bits [..., V] -> lp of the labels' shape, 0 where ignored (those rows are not looked at)."""
    on = labels != ignore
    # log_softmax: NaN for a row that holds an infinity above or nothing but ones below (logsumexp alone has a value there)
    lp = torch.log_softmax(x[on] / temperature, -1).gather(-1, labels[on].long().unsqueeze(-1)).squeeze(-1)
    return torch.zeros(labels.shape, dtype=torch.float64).masked_scatter(on, lp)


def spans(labels, cu=None):
    if cu is not None:
        cu = [int(c) for c in cu]
        return list(zip(cu, cu[1:]))
    if labels.dim() == 1:
        return [(0, labels.numel())]
    n = labels.shape[1]
    return [(i * n, (i + 1) * n) for i in range(labels.shape[0])]


def sums(lp, labels, ignore=-100, cu=None, average=False):
    lp, on = lp.reshape(-1), (labels != ignore).view(-1)
    out = []
    for a, b in spans(labels, cu):
        n = int(on[a:b].sum())
        out.append(lp[a:b].sum() / (max(n, 1) if average else 1))
    return torch.stack(out)


def preference(x, labels, ref, beta=0.1, smoothing=0.0, kind="sigmoid", average=False, cu=None, ignore=-100):
    gain = sums(log_probs(x, labels, ignore), labels, ignore, cu, average) - ref.double()
    n = gain.numel() // 2
    losses = []
    for b in range(n):
        d = gain[b] - gain[n + b]
        if kind == "sigmoid":
            losses.append(-(1 - smoothing) * torch.nn.functional.logsigmoid(beta * d)
                          - (smoothing * torch.nn.functional.logsigmoid(-beta * d) if smoothing else 0))
        elif kind == "ipo":
            losses.append((d - 1 / (2 * beta)) ** 2)
        else:
            losses.append(torch.relu(1 - beta * d))
    return torch.stack(losses).mean(), (beta * gain).detach()


def policy(x, labels, old, adv, ref=None, low=0.2, high=0.2, kl=0.0, temperature=1.0, reduction="token", cu=None, ignore=-100):
    lp = log_probs(x, labels, ignore, temperature)
    flat, on = lp.reshape(-1), (labels != ignore).view(-1)
    by_row = adv.shape == labels.shape
    each = torch.zeros(labels.numel(), dtype=torch.float64)
    means, total, tokens = [], 0.0, 0
    for s, (a, b) in enumerate(spans(labels, cu)):
        at = torch.arange(a, b)[on[a:b]]
        l = flat[at]
        A = adv.reshape(-1)[at].double() if by_row else adv[s].double()
        ratio = torch.exp(l - (l.detach() if old is None else old.reshape(-1)[at].double()))
        loss = -torch.minimum(ratio * A, ratio.clamp(1 - low, 1 + high) * A)
        if ref is not None and kl:
            d = ref.reshape(-1)[at].double() - l
            loss = loss + kl * (torch.exp(d) - d - 1)
        each = each.index_put((at,), loss)
        means.append(loss.sum() / max(1, at.numel()))
        total, tokens = total + loss.sum(), tokens + at.numel()
    out = {"token": lambda: total / max(1, tokens), "sum": lambda: total, "none": lambda: each.view(labels.shape),
           "sequence": lambda: torch.stack(means).mean()}[reduction]()
    return out, lp.detach()


U = 2.0 ** -24  # half a step of fp32, relative


def lp_bound(x, labels, ignore=-100, temperature=1.0):
    """How far one token's lp in fp32 may be, of the labels' shape.

    lp = ((x_y - m) c - log2 s) ln 2 with c = log2(e) / T. Against m, the largest x: the difference, c, the product,
    log2 (one step), the outer difference and product take at most 6 half steps of |x_y - m| / T + log s, and of the
    result. A term exp2((x - m) c) of s is off by 2 + 3 a half steps where a = (m - x) c, and a exp2(-a) is at most
    0.54: under 4 for each term that counts, 2 V for what lies at the far end of a sum of V terms that one lane adds
    (V / 256 of them, and 16 joins). So s is off by V / 128 + 24 half steps, and log s by that.
    """
    z = torch.nan_to_num(x.double() / temperature, nan=0.0, neginf=0.0, posinf=0.0)
    far = z.amax(-1) - z.amin(-1)
    v = x.shape[-1]
    return torch.where(labels != ignore, U * (6 * (2 * far + 2 * math.log(v) + 1) + v / 128 + 24), 0.0)


def grad_bound(x, labels, coef, dtype, ignore=-100, temperature=1.0):
    """How far the logits' gradient f ([v = y] - p), f = coef / T, may be: p is off by at most lp's bound (its exponent
    differs from lp's by the logit alone) relative to it, f by 4 half steps, and the result is rounded once."""
    z = torch.nan_to_num(x.double() / temperature, nan=0.0, neginf=-math.inf)
    p = torch.softmax(z, -1)
    b = lp_bound(x, labels, ignore, temperature).unsqueeze(-1)
    f = torch.where(labels != ignore, coef.double().abs() / temperature, 0.0).unsqueeze(-1)
    y = torch.nn.functional.one_hot(torch.where(labels != ignore, labels, 0).long(), x.shape[-1])
    g = f * (y - p).abs()
    e = torch.finfo(dtype)
    return f * p * (b + 4 * U) + g * (4 * U + e.eps / 2) + e.smallest_normal * e.eps / 2 + 1e-37
