"""Distillation loss from a teacher's top logits in fp64, one row at a time: the oracle of the kernel."""
from __future__ import annotations

import math

import torch


def row_loss(s: torch.Tensor, ids: list[int], t: list[float], label: int | None, lse: float | None, T: float,
             alpha: float, ignore: int = -100):
    """Loss of one row of fp64 student logits, and whether the row counts."""
    V = s.numel()
    on = [(i, x) for i, x in zip(ids, t) if 0 <= i < V and x != -math.inf]
    if label is not None and (label == ignore or not 0 <= label < V):
        return s.new_zeros(()), False
    if label is None and not on:
        return s.new_zeros(()), False
    loss = s.new_zeros(())
    if on and alpha != 0.0:
        tt = torch.tensor([x for _, x in on], dtype=torch.float64, device=s.device) / T
        logp = tt - (torch.logsumexp(tt, 0) if lse is None else lse)
        at = torch.tensor([i for i, _ in on], device=s.device)
        logq = s / T - torch.logsumexp(s / T, 0)
        p = torch.exp(logp)
        term = torch.where(p > 0, p * (logp - logq[at]), torch.zeros_like(p)).sum()
        if lse is not None:
            rest = torch.ones(V, dtype=torch.bool, device=s.device)
            rest[at] = False
            pr = float(max(0.0, 1.0 - float(p.sum())))
            if pr > 0 and bool(rest.any()):
                term = term + pr * (math.log(pr) - torch.logsumexp(logq[rest], 0))
        loss = loss + alpha * T * T * term
    if label is not None and alpha != 1.0:
        loss = loss + (1 - alpha) * (torch.logsumexp(s, 0) - s[label])
    return loss, True


def scale_of(s, ids, t, lse, T):
    """sum of p (|log p| + |log q|) of a row: what the loss's rounding errors are relative to."""
    V = s.numel()
    on = [(i, x) for i, x in zip(ids, t) if 0 <= i < V and x != -math.inf]
    if not on:
        return 0.0
    tt = torch.tensor([x for _, x in on], dtype=torch.float64, device=s.device) / T
    logp = tt - (torch.logsumexp(tt, 0) if lse is None else lse)
    logq = (s / T - torch.logsumexp(s / T, 0))[torch.tensor([i for i, _ in on], device=s.device)]
    p = torch.exp(logp)
    v = torch.where(p > 0, p * (logp.abs() + logq.abs()), torch.zeros_like(p)).sum()
    return float(v)


def losses(logits, ids, t, labels, lse, T, alpha, ignore=-100):
    """(losses [N] with autograd to fp64 ``logits``, counted [N], rounding scales [N])."""
    out, counted, scale = [], [], []
    ids_l, t_l = ids.tolist(), t.double().tolist()
    lab = None if labels is None else labels.tolist()
    lse_l = None if lse is None else lse.double().tolist()
    for r in range(logits.shape[0]):
        l, c = row_loss(logits[r], ids_l[r], t_l[r], None if lab is None else lab[r],
                        None if lse_l is None else lse_l[r], T, alpha, ignore)
        out.append(l)
        counted.append(c)
        with torch.no_grad():
            scale.append(scale_of(logits[r].detach(), ids_l[r], t_l[r], None if lse_l is None else lse_l[r], T))
    return torch.stack(out), counted, torch.tensor(scale, dtype=torch.float64, device=logits.device)
