"""Float64 definition of the head losses: softmax cross entropy and
distillation from a teacher's top logits, straight from hidden states and the
head's weight, row by row where the sparse targets are concerned.

Gradients are written out from the formulas; the CPU tests hold them against
autograd and against differences.
"""
from __future__ import annotations

import math

import torch


def ce_target(target, vocab):
    """(rows that count, dense target distribution, sum p log p) of hard targets."""
    keep = (target >= 0) & (target < vocab)
    p = torch.zeros(len(target), vocab, dtype=torch.float64)
    for i in torch.nonzero(keep)[:, 0].tolist():
        p[i, int(target[i])] = 1.0
    return keep, p, torch.zeros(len(target), dtype=torch.float64)


def distill_target(ids, logits, vocab, temperature):
    """The same of a teacher's entries: absent where the id is negative (or past
    the vocabulary) or the logit is -inf; an id that stands twice adds up."""
    rows, K = ids.shape
    keep = torch.zeros(rows, dtype=torch.bool)
    p = torch.zeros(rows, vocab, dtype=torch.float64)
    plogp = torch.zeros(rows, dtype=torch.float64)
    for i in range(rows):
        there = [(int(ids[i, k]), float(logits[i, k]) / temperature) for k in range(K)
                 if 0 <= int(ids[i, k]) < vocab and float(logits[i, k]) != -math.inf]
        if not there:
            continue
        keep[i] = True
        top = max(y for _, y in there)
        total = sum(math.exp(y - top) for _, y in there)
        for c, y in there:
            q = math.exp(y - top) / total
            p[i, c] += q
            if q > 0:
                plogp[i] += q * (y - top - math.log(total))
    return keep, p, plogp


def head_loss(x, w, keep, p, plogp, scale=1.0, temperature=1.0, grad=None):
    """Returns (loss, lse, dx, dw) in float64; rows that do not count give zeros
    and nothing of their x is looked at."""
    T = temperature
    rows, dim = x.shape
    loss, lse = (torch.zeros(rows, dtype=torch.float64) for _ in range(2))
    dx = torch.zeros(rows, dim, dtype=torch.float64)
    xs, ws, ps = x[keep].double(), w.double(), p[keep]
    u = (scale / T) * (xs @ ws.T)
    l = torch.logsumexp(u, 1) if len(xs) else torch.zeros(0, dtype=torch.float64)
    lse[keep] = l
    loss[keep] = T * T * (plogp[keep] + (ps * (l[:, None] - u)).sum(1))
    g = torch.ones(rows, dtype=torch.float64) if grad is None else grad.double()
    dz = g[keep][:, None] * T * (torch.exp(u - l[:, None]) - ps)
    dx[keep] = scale * (dz @ ws)
    return loss, lse, dx, scale * (dz.T @ xs)


def bounds(x, w, keep, p, scale=1.0, temperature=1.0, grad=None, dz_step=2.0 ** -8):
    """How far the kernels may be from head_loss, entry by entry, by arithmetic:
    returns (loss, lse, dx, dw) bounds without the rounding of the outputs.

    Logits: products of bf16 are exact in fp32; a sum of `dim` of them in steps
    of 16 is off by at most (dim / 16 + 16) * 2^-23 times the sum of the
    products' magnitudes (one truncation a step, and 16 for the alignment
    inside a step): du.  The exponential is off by 2^-22, its argument by 2^-23
    of |u| log2(e), sums of positive terms by 2^-18 (a chain of at most 32
    chunk sums): e = 2^-17 + 2^-22 |u|max in all.
    lse: du + e, and 2^-22 of its size; loss: T^2 times that and du more.
    dz = a (q - p): q off by q * (2 (du + e)), the value rounded to bf16, half a
    step, dz_step = 2^-8 of its size (in two parts: 2^-16).  dx, dw: those times
    |w|, |x| summed, and the fp32 sums' own 2^-16 of the magnitudes (a step of 16
    truncates 2^-23, at most a few hundred steps a product here, and one fp32
    addition a piece).
    """
    T = temperature
    xs, ws, ps = x[keep].double(), w.double(), p[keep]
    u = (scale / T) * (xs @ ws.T)
    mag = float((xs.abs() @ ws.abs().T).max()) * scale / T if len(xs) else 0.0
    du = (x.shape[1] / 16 + 16) * 2.0 ** -23 * mag
    umax = float(u.abs().max()) if len(xs) else 0.0
    e = 2.0 ** -17 + 2.0 ** -22 * umax
    lse_max = umax + math.log(w.shape[0])
    b_lse = du + e + 2.0 ** -22 * lse_max
    b_loss = T * T * (b_lse + du + 2.0 ** -22 * (lse_max + umax + 20))
    g = torch.ones(x.shape[0], dtype=torch.float64) if grad is None else grad.double()
    q = torch.softmax(u, 1)
    a = (g[keep].abs() * T * scale)[:, None]
    dz = a * (q - ps).abs()
    off = a * q * (2 * (du + e)) + dz_step * dz + 2.0 ** -16 * dz + a * 2.0 ** -24
    bdx = torch.zeros(x.shape, dtype=torch.float64)
    bdx[keep] = off @ ws.abs()
    return b_loss, b_lse, bdx, off.T @ xs.abs()
