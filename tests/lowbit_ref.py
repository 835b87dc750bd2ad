"""Plain float64 forms of the norm / microscaled product / distillation operators, from their formulas (torch tensors, any device)."""
import math

import torch

GRID = {'e2m1': [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0],
        'e4m3': [m * 2.0 ** -9 for m in range(8)] + [(8 + m) * 2.0 ** (e - 10) for e in range(1, 16) for m in range(8)][:119]}


def quantize(x, fmt):
    """codes [..., blocks, 32] (int64, sign in the top bit), scale bytes [..., blocks] of x along its last axis, filled up to whole
    groups of 128: smallest power of two under which no element exceeds the format's largest, ties to the even code."""
    x = x.double()
    width = -(-x.shape[-1] // 128) * 128
    b = torch.zeros(x.shape[:-1] + (width,), dtype=torch.float64, device=x.device)
    b[..., :x.shape[-1]] = x
    b = b.unflatten(-1, (-1, 32))
    grid = torch.tensor(GRID[fmt], dtype=torch.float64, device=x.device)
    finite = torch.isfinite(b).all(-1)
    amax = torch.where(finite, b.abs().amax(-1), torch.ones_like(b[..., 0]))
    e = torch.ceil(torch.log2((amax / grid[-1]).clamp(min=2.0 ** -400)))
    e = e.clamp(-126, 127)
    scaled = b / torch.exp2(e)[..., None]
    a = scaled.abs()
    middle = (grid[1:] + grid[:-1]) / 2
    below, above = torch.bucketize(a, middle), torch.bucketize(a, middle, right=True)
    code = torch.where(below % 2 == 0, below, above)
    code = code + (torch.signbit(scaled).long() << (7 if fmt == 'e4m3' else 3))
    return code, torch.where(finite, e + 127, torch.full_like(e, 255)).long()


def values(code, byte, fmt, width):
    half = 128 if fmt == 'e4m3' else 8
    grid = torch.tensor(GRID[fmt] + [math.nan] * (half - len(GRID[fmt])), dtype=torch.float64, device=code.device)
    v = grid[code % half] * torch.where(code >= half, -1.0, 1.0).double()
    scale = torch.where(byte == 255, torch.full_like(v[..., 0], math.nan), torch.exp2(byte.double() - 127))
    return (v * scale[..., None]).flatten(-2)[..., :width]


def rounded(x, fmt):
    code, byte = quantize(x, fmt)
    return values(code, byte, fmt, x.shape[-1])


def rms(h, gamma, eps):
    h, gamma = h.double(), gamma.double()
    return h / torch.sqrt((h * h).mean(-1, keepdim=True) + eps) * gamma


def rms_grads(h, gamma, eps, dy, dh=None):
    """dx (without rounding) and dgamma."""
    h, gamma, dy = h.double(), gamma.double(), dy.double()
    s = 1 / torch.sqrt((h * h).mean(-1, keepdim=True) + eps)
    n, g = h * s, dy * gamma
    dx = s * (g - n * (g * n).mean(-1, keepdim=True))
    return (dx if dh is None else dx + dh.double()), (dy * n).flatten(0, -2).sum(0)


def distill(logits, teacher, index, tau=1.0, weight=1.0, row_weight=None, lse=None):
    """loss, gradient and per-class sizes (q + p) * scale that its rounding errors go by; a row at a time."""
    logits, teacher = logits.double(), teacher.double()
    rows, classes = logits.shape
    w = torch.ones(rows, dtype=torch.float64) if row_weight is None else row_weight.double().cpu()
    total = float(w.sum())
    loss, grad, size = 0.0, torch.zeros_like(logits), torch.zeros_like(logits)
    for r in range(rows):
        at = [(int(i), float(t) / tau) for i, t in zip(index[r], teacher[r]) if 0 <= int(i) < classes and float(t) != -math.inf]
        if not at or float(w[r]) == 0 or total == 0:
            continue
        z = logits[r] / tau
        logq = z - torch.logsumexp(z, 0)
        q = torch.exp(logq)
        t = torch.tensor([v for _, v in at], dtype=torch.float64)
        # (differences first: beside the type's lowest value there is no room for the log of a number of entries)
        logp = torch.log_softmax(t - t.max(), 0) if lse is None else t - float(lse[r])
        p = torch.exp(logp)
        rest = 0.0 if lse is None else max(0.0, 1.0 - float(p.sum()))
        mass = float(p.sum()) if lse is not None else 1.0
        l = sum(float(pi) * (float(lp) - float(logq[i])) for (i, _), pi, lp in zip(at, p, logp))
        g, used = mass * q, q.clone()
        if lse is not None:
            outside = torch.ones(classes, dtype=torch.bool, device=z.device)
            outside[[i for i, _ in at]] = False
            lqr = torch.logsumexp(logq[outside], 0) if bool(outside.any()) else torch.tensor(-math.inf)
            if rest > 0 and float(lqr) > -math.inf:
                l += rest * (math.log(rest) - float(lqr))
                # shares of the mass outside add up to 1, also where all of z is the type's lowest value and lqr has no room for
                # the log of their number
                share = torch.where(outside, torch.exp(z - z[outside].max()), torch.zeros_like(q))
                share = share / share.sum()
                # (only here: a loss without the term of the remaining mass has a gradient without it)
                g = g + rest * q - rest * share
                used = used + rest * share
        for (i, _), pi in zip(at, p):
            g[i] -= float(pi)
            used[i] += float(pi)
        scale = weight * tau * float(w[r]) / total
        loss += scale * tau * l
        grad[r], size[r] = g * scale, used * abs(scale)
    return loss, grad, size
