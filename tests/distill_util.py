"""Distillation from stored top logits by its definition in 64 bits on the CPU, with bounds for the kernels' arithmetic.

Bounds.  An exponential is exp2 of (y - max) times a rounded scale: its argument is off by 3 x 2^-24 of itself and the result by
2^-23; with g the largest |y - max| (counted up to 100: beyond, it is 0 in f32) a probability is off by e = (4 g + 8) 2^-24 relative, and the sums over a thread's classes by n 2^-24
with n = V / 256 + 32.  Twice that for a probability over its sum; the gradient is rounded once to its type (u, or half a subnormal step)."""
import math

import torch


def reference(z, values, indices, rest, tau, up):
    """((row losses, bound), (gradient of sum(up * row losses), bound)) in float64; z, values: what the kernel reads"""
    dtype = z.dtype
    u = torch.finfo(dtype).eps / 2
    sub = 0.0 if dtype != torch.float16 else 2.0 ** -25
    z, v, idx, up = z.detach().cpu().double(), values.detach().cpu().double(), indices.cpu().long(), up.cpu().double()
    R, V = z.shape
    losses, grads, e_losses, e_grads = [], [], [], []
    for r in range(R):
        entries = {}
        for i, t in zip(idx[r].tolist(), v[r].tolist()):
            if 0 <= i < V and t > -math.inf:
                entries.setdefault(i, []).append(t / tau)
        y = z[r] / tau
        if not entries:
            losses.append(0.0); e_losses.append(0.0)
            grads.append(torch.zeros(V, dtype=torch.float64)); e_grads.append(torch.zeros(V, dtype=torch.float64))
            continue
        kept = torch.zeros(V, dtype=torch.bool)
        kept[list(entries)] = True
        left = float(rest[r]) if rest is not None and not bool(kept.all()) else -math.inf
        total = torch.logsumexp(torch.tensor([t for ts in entries.values() for t in ts] + [left], dtype=torch.float64), 0)
        log_q = torch.log_softmax(y, 0)
        p = torch.zeros(V, dtype=torch.float64)
        loss = size = 0.0
        for i, ts in entries.items():
            for t in ts:
                pk = math.exp(t - total)
                p[i] += pk
                loss += pk * (t - float(total) - float(log_q[i]))
                size += pk * (abs(t) + abs(float(total)) + abs(float(y[i])) + abs(float(log_q[i])) + 1)
        q = log_q.exp()
        g = q - p
        top = float(torch.stack([(y - y.max()).abs().clamp(max=100).max(), torch.tensor([abs(t - float(total)) for ts in entries.values() for t in ts]).max().clamp(max=100)]).max())
        e = 2 * ((4 * (top + abs(float(y.max()))) + 8) + V / 256 + 32) * 2.0 ** -24
        if left > -math.inf:
            pr, log_rest = math.exp(left - total), float(torch.logsumexp(log_q.masked_fill(kept, -math.inf), 0))
            loss += pr * (left - float(total) - log_rest)
            size += pr * (abs(left) + abs(float(total)) + abs(log_rest) + 1)
            shared = torch.exp(log_q - log_rest) * pr
            g = torch.where(kept, g, q - shared)
            bound = e * torch.where(kept, q + p, q + shared)
        else:
            bound = e * (q + p)
        s = float(up[r]) * tau
        losses.append(loss * tau * tau); e_losses.append(tau * tau * (e * size + 2.0 ** -24 * abs(loss)))
        g, bound = g * s, bound * abs(s)
        grads.append(g); e_grads.append(bound + u * (g.abs() + bound) + sub)
    return (torch.tensor(losses), torch.tensor(e_losses)), (torch.stack(grads), torch.stack(e_grads))


def top(z, k, tau):
    """(values, indices, rest) of a CPU tensor: NaN first, ties by the class"""
    zd = z.double()
    key = torch.where(torch.isnan(zd), math.inf, zd) + 0.0
    values, indices, rest = [], [], []
    for r in range(z.shape[0]):
        row = sorted(range(z.shape[1]), key=lambda i: (not math.isnan(float(zd[r, i])), -float(key[r, i]), i))
        values.append(z[r, row[:k]])
        indices.append(torch.tensor(row[:k], dtype=torch.int32))
        rest.append(torch.logsumexp(zd[r, row[k:]] / tau, 0) if k < len(row) else torch.tensor(-math.inf, dtype=torch.float64))
    return torch.stack(values), torch.stack(indices), torch.stack(rest)
