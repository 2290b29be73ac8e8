"""Plain 64-bit forms of the selective operators and of distillation, token by
token and entry by entry, for the tests to compare with."""
from __future__ import annotations

import math

import torch


def runs(x, lengths):
    """Rows of each sequence of ``[B, T, ...]`` (lengths None) or packed ``[tokens, ...]``."""
    if lengths is None:
        return list(x)
    out, at = [], 0
    for n in lengths:
        out.append(x[at:at + n])
        at += n
    return out


def conv(x, weight, bias, silu, state, lengths=None):
    taps = weight.shape[1]
    ys, finals = [], []
    for i, r in enumerate(runs(x, lengths)):
        past = torch.zeros(taps - 1, x.shape[-1], dtype=x.dtype, device=x.device) if state is None else state[i]
        wide = torch.cat([past, r])
        rows = []
        for t in range(r.shape[0]):
            u = sum(wide[t + j] * weight[:, j] for j in range(taps))
            u = u if bias is None else u + bias
            rows.append(u * torch.sigmoid(u) if silu else u)
        ys.append(torch.stack(rows) if rows else r)
        finals.append(wide[r.shape[0]:])
    return (torch.stack(ys) if lengths is None else torch.cat(ys)), torch.stack(finals)


def scan(values, steps, rates, keys, queries, skip, gate, step_bias, softplus, state, lengths=None):
    channels, n = rates.shape
    repeat = channels // keys.shape[-2]
    d = steps if step_bias is None else steps + step_bias
    if softplus:
        d = torch.log1p(torch.exp(-d.abs())) + d.clamp(min=0)
    parts = [runs(v, lengths) for v in (values, d, keys, queries)]
    reads, finals = [], []
    for i, (x, dt, k, q) in enumerate(zip(*parts)):
        h = torch.zeros(channels, n, dtype=values.dtype, device=values.device) if state is None else state[i]
        rows = []
        for t in range(x.shape[0]):
            h = torch.exp(dt[t, :, None] * rates) * h + (dt[t] * x[t])[:, None] * k[t].repeat_interleave(repeat, 0)
            rows.append((q[t].repeat_interleave(repeat, 0) * h).sum(-1))
        reads.append(torch.stack(rows) if rows else x)
        finals.append(h)
    r = torch.stack(reads) if lengths is None else torch.cat(reads)
    r = r if skip is None else r + skip * values
    r = r if gate is None else r * gate * torch.sigmoid(gate)
    return r, torch.stack(finals)


def distill(logits, teacher, indices, temperature):
    """Loss of every row, and which rows have a teacher."""
    losses, counted = [], []
    for s, t, idx in zip(logits, teacher, indices):
        live = [(float(tk), int(j)) for tk, j in zip(t, idx) if int(j) >= 0 and float(tk) != -math.inf]
        counted.append(bool(live))
        if not live:
            losses.append((s * 0.0).nan_to_num(0.0).sum() * 0.0)
            continue
        z = s / temperature
        log_q = z - torch.logsumexp(z, 0)
        tk = torch.tensor([v for v, _ in live], dtype=torch.float64, device=s.device) / temperature
        log_p = tk - torch.logsumexp(tk, 0)
        where = torch.tensor([j for _, j in live], device=s.device)
        p = torch.exp(log_p)
        losses.append(temperature ** 2 * sum(p[k] * (log_p[k] - log_q[where[k]]) for k in range(len(live))
                                             if float(p[k]) != 0.0))
    return torch.stack(losses), counted
