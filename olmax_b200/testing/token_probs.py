"""
The definitions of the operators over an LM head's distribution in 64 bits, row by row and class by class where that is plainest:
the oracle of their tests.
"""

from __future__ import annotations

import math

import torch

__all__ = ["scores_64", "score_gradients_64", "distillation_64"]


def _scaled(z, temperature, cap):
    """(y, dy / dz) in 64 bits."""
    z = z.double()
    if cap:
        t = torch.tanh(z / cap)
        return cap * t / temperature, (1 - t * t) / temperature
    return z / temperature, torch.full_like(z, 1 / temperature)


def _log_softmax(y):
    """log p; -inf everywhere for a row without any class."""
    lp = torch.log_softmax(y, -1)
    return torch.where((y == -math.inf).all(-1, keepdim=True), y, lp)


def scores_64(z, ids, top_k, temperature=1.0, cap=0.0, ignore_index=-100):
    """(log p of ids, entropy, top log p, top ids) of logits z [rows, V]."""
    y, _ = _scaled(z, temperature, cap)
    lp = _log_softmax(y)
    p = lp.exp()
    entropy = -torch.where(p == 0, 0.0, p * lp).sum(-1)
    V = z.shape[-1]
    known = (ids != ignore_index) & (ids >= 0) & (ids < V)
    taken = torch.where(known, lp.gather(-1, ids.clamp(0, V - 1)[:, None])[:, 0], 0.0)
    order = z.double().sort(dim=-1, descending=True, stable=True).indices[:, :top_k]
    return taken, entropy, lp.gather(-1, order), order


def score_gradients_64(z, ids, g_log_probs, g_entropy, temperature=1.0, cap=0.0, ignore_index=-100):
    """(gradient, sum of the absolute values of its terms) of sum g_log_probs log p + sum g_entropy H for logits z."""
    y, slope = _scaled(z, temperature, cap)
    lp = _log_softmax(y)
    p = lp.exp()
    V = z.shape[-1]
    known = (ids != ignore_index) & (ids >= 0) & (ids < V)
    one = torch.zeros_like(p).scatter_(-1, ids.clamp(0, V - 1)[:, None], known.double()[:, None])
    gl = (g_log_probs.double() * known)[:, None]
    ge = g_entropy.double()[:, None]
    inner = torch.where(p == 0, 0.0, lp)
    h = -(p * inner).sum(-1, keepdim=True)
    none = (y == -math.inf).all(-1, keepdim=True)
    grad = slope * (gl * (one - p) - ge * p * (inner + h))
    size = slope * (gl.abs() * (one + p) + ge.abs() * p * (inner.abs() + h))
    return torch.where(none, 0.0, grad), torch.where(none, 0.0, size)


def distillation_64(z, teacher_ids, teacher_log_probs, tail, reduction="mean", temperature=1.0, cap=0.0):
    """(loss, its gradient for a unit upstream gradient): each row's divergence from sums over Python lists of its classes."""
    y, slope = _scaled(z, temperature, cap)
    lp = _log_softmax(y)
    rows, V = z.shape
    losses, grads, counted = [], torch.zeros_like(y), []
    for r in range(rows):
        pairs = {}
        for i, t in zip(teacher_ids[r].tolist(), teacher_log_probs[r].double().tolist()):
            if 0 <= i < V and i not in pairs:
                pairs[i] = t
        if tail == "renormalize":
            norm = torch.logsumexp(torch.tensor([t for t in pairs.values()] + [-math.inf], dtype=torch.float64), 0).item()
            pairs = {i: t - norm for i, t in pairs.items()} if norm != -math.inf else {}
        if not pairs:
            losses.append(0.0)
            counted.append(False)
            continue
        counted.append(True)
        index = torch.tensor(list(pairs), device=z.device)
        log_q = torch.tensor(list(pairs.values()), dtype=torch.float64, device=z.device)
        q = log_q.exp()
        outside = torch.ones(V, dtype=torch.bool, device=z.device)
        outside[index] = False
        loss = torch.where(q == 0, 0.0, q * (log_q - lp[r, index])).sum()
        rest_lse = torch.logsumexp(torch.where(outside, y[r], -math.inf), 0)
        rest = max(0.0, 1.0 - q.sum().item()) if tail == "rest" and rest_lse != -math.inf else 0.0
        if rest > 0:
            loss = loss + rest * (math.log(rest) - torch.logsumexp(torch.where(outside, lp[r], -math.inf), 0))
        losses.append(loss.item())
        if not torch.all(y[r] == -math.inf):
            total = q.sum() + rest
            grads[r] = total * lp[r].exp()
            grads[r, index] -= q
            if rest > 0:
                grads[r, outside] -= rest * (y[r, outside] - rest_lse).exp()
    loss = torch.tensor(losses, dtype=torch.float64, device=z.device)
    grads = grads * slope
    if reduction == "none":
        return loss, grads
    n = max(1, sum(counted)) if reduction == "mean" else 1
    return loss.sum() / n, grads / n
