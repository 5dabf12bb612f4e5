"""
Plain PyTorch restatement of every op's math.  It is the numerical oracle of the CUDA kernels (GPU tests compare a
kernel against these functions evaluated in fp32) and it is the implementation used on CPU, where the multi-process
(gloo) tests and the tiny fp32 configuration run.

Semantics follow the reference: RMSNorm upcasts to fp32, multiplies by ``rsqrt(mean(x^2) + eps)`` and by the weight,
then casts back (``olmax/nn/functional.py:51-67``); RoPE is the rotate-half form computed in fp32
(``olmax/nn/rope.py:99-115``); attention is causal soft-max attention with scale ``1/sqrt(head_dim)``, grouped KV
heads and an optional left window (``olmax/nn/attention.py:96-103``) plus an optional tanh soft-cap; the MLP is
``down(act(gate(x)) * up(x))`` (``olmax/nn/mlp.py:69-73``); cross entropy excludes ``ignore_index`` rows from both
numerator and denominator (``olmax/nn/functional.py:70-121``).
"""

from __future__ import annotations

import math
from typing import Optional, Tuple

import torch
import torch.nn.functional as F

__all__ = [
    "rms_norm", "layer_norm", "rope_tables", "apply_rope", "attention", "glu", "cross_entropy", "fused_cross_entropy",
    "softcap", "activation", "token_log_probs", "token_log_probs_bwd", "distillation", "distillation_bwd",
]


def rms_norm(x: torch.Tensor, weight: Optional[torch.Tensor], eps: float = 1e-5,
             bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    dt = x.dtype
    xf = x.float()
    y = xf * torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + eps)
    if weight is not None:
        y = y * weight.float()
    if bias is not None:
        y = y + bias.float()
    return y.to(dt)


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor], bias: Optional[torch.Tensor], eps: float = 1e-5) -> torch.Tensor:
    dt = x.dtype
    xf = x.float()
    mean = xf.mean(-1, keepdim=True)
    var = (xf - mean).pow(2).mean(-1, keepdim=True)
    y = (xf - mean) * torch.rsqrt(var + eps)
    if weight is not None:
        y = y * weight.float()
    if bias is not None:
        y = y + bias.float()
    return y.to(dt)


def rope_tables(seq_len: int, head_dim: int, theta: float, device=None) -> Tuple[torch.Tensor, torch.Tensor]:
    """cos, sin of shape [seq_len, head_dim // 2] in fp32: angle = position * theta^(-2i / head_dim)."""
    inv_freq = 1.0 / (theta ** (torch.arange(0, head_dim, 2, dtype=torch.float32, device=device) / head_dim))
    pos = torch.arange(seq_len, dtype=torch.float32, device=device)
    ang = torch.outer(pos, inv_freq)
    return ang.cos(), ang.sin()


def apply_rope(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, sign: float = 1.0) -> torch.Tensor:
    """x: [B, S, H, D]; out = x * [cos, cos] + rotate_half(x) * [sin, sin]."""
    dt = x.dtype
    S, D = x.shape[1], x.shape[-1]
    xf = x.float()
    c = cos[:S].view(1, S, 1, D // 2)
    s = sin[:S].view(1, S, 1, D // 2) * sign
    lo, hi = xf[..., : D // 2], xf[..., D // 2 :]
    return torch.cat([lo * c - hi * s, hi * c + lo * s], dim=-1).to(dt)


def softcap(x: torch.Tensor, cap: float) -> torch.Tensor:
    return cap * torch.tanh(x / cap) if cap and cap > 0 else x


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, causal: bool = True, window: int = -1,
              logit_softcap: float = 0.0, scale: Optional[float] = None, q_off: int = 0) -> Tuple[torch.Tensor, torch.Tensor]:
    """q [B,S,H,D], k/v [B,Sk,Hkv,D] -> (o [B,S,H,D], lse [B,H,S]).  Query row i sits at position ``q_off + i`` of the
    key axis; window >= 0 keeps keys j >= position - window."""
    B, S, H, D = q.shape
    Hkv = k.shape[2]
    scale = scale if scale is not None else 1.0 / math.sqrt(D)
    qf = q.float().permute(0, 2, 1, 3)
    kf = k.float().permute(0, 2, 1, 3).repeat_interleave(H // Hkv, dim=1)
    vf = v.float().permute(0, 2, 1, 3).repeat_interleave(H // Hkv, dim=1)
    s = torch.matmul(qf, kf.transpose(-1, -2)) * scale
    s = softcap(s, logit_softcap)
    Sk = k.shape[1]
    i = torch.arange(S, device=q.device).view(S, 1) + q_off
    j = torch.arange(Sk, device=q.device).view(1, Sk)
    mask = torch.ones(S, Sk, dtype=torch.bool, device=q.device)
    if causal:
        mask &= j <= i
    if window is not None and window >= 0:
        mask &= j >= i - window
    s = s.masked_fill(~mask, float("-inf"))
    lse = torch.logsumexp(s, dim=-1)
    p = torch.softmax(s, dim=-1)
    o = torch.matmul(p, vf).permute(0, 2, 1, 3)
    return o.to(q.dtype), lse


def attention_bwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, o: torch.Tensor, lse: torch.Tensor,
                  d_o: torch.Tensor, causal: bool = True, window: int = -1, logit_softcap: float = 0.0,
                  scale: Optional[float] = None, q_off: int = 0) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Gradients of one (query block, key block) pair of a softmax whose row statistics are given: ``lse`` [B,H,S] is
    the log-sum-exp over ALL keys of the row (not only this block's) and ``o`` the final output, so the pieces of a
    blockwise / ring attention add up to the gradient of the whole."""
    B, S, H, D = q.shape
    Hkv, Sk = k.shape[2], k.shape[1]
    G = H // Hkv
    scale = scale if scale is not None else 1.0 / math.sqrt(D)
    qf = q.float().permute(0, 2, 1, 3)
    kf = k.float().permute(0, 2, 1, 3).repeat_interleave(G, dim=1)
    vf = v.float().permute(0, 2, 1, 3).repeat_interleave(G, dim=1)
    dof = d_o.float().permute(0, 2, 1, 3)
    raw = torch.matmul(qf, kf.transpose(-1, -2)) * scale
    s = softcap(raw, logit_softcap)
    i = torch.arange(S, device=q.device).view(S, 1) + q_off
    j = torch.arange(Sk, device=q.device).view(1, Sk)
    mask = torch.ones(S, Sk, dtype=torch.bool, device=q.device)
    if causal:
        mask &= j <= i
    if window is not None and window >= 0:
        mask &= j >= i - window
    p = torch.exp(s - lse.float().unsqueeze(-1)).masked_fill(~mask, 0.0)
    delta = (o.float() * d_o.float()).sum(-1).permute(0, 2, 1).unsqueeze(-1)   # [B,H,S,1]
    dv = torch.matmul(p.transpose(-1, -2), dof)
    dp = torch.matmul(dof, vf.transpose(-1, -2))
    ds = p * (dp - delta)
    if logit_softcap and logit_softcap > 0:
        ds = ds * (1.0 - torch.tanh(raw / logit_softcap) ** 2)
    ds = ds * scale
    dq = torch.matmul(ds, kf).permute(0, 2, 1, 3)
    dk = torch.matmul(ds.transpose(-1, -2), qf)
    dk = dk.view(B, Hkv, G, Sk, D).sum(2).permute(0, 2, 1, 3)
    dv = dv.view(B, Hkv, G, Sk, D).sum(2).permute(0, 2, 1, 3)
    return dq.to(q.dtype), dk.to(k.dtype), dv.to(v.dtype)


def activation(name: str, x: torch.Tensor) -> torch.Tensor:
    if name == "silu":
        return F.silu(x)
    if name in ("gelu", "gelu_tanh"):
        return F.gelu(x, approximate="tanh")
    raise ValueError(f"unknown activation '{name}'")


def glu(g: torch.Tensor, u: torch.Tensor, act: str = "silu") -> torch.Tensor:
    return (activation(act, g.float()) * u.float()).to(g.dtype)


def cross_entropy(logits: torch.Tensor, labels: torch.Tensor, ignore_index: int = -100, reduction: str = "mean",
                  logit_softcap: float = 0.0) -> torch.Tensor:
    loss, _ = fused_cross_entropy(logits, labels, ignore_index=ignore_index, reduction=reduction,
                                  logit_softcap=logit_softcap)
    return loss


def fused_cross_entropy(logits: torch.Tensor, labels: torch.Tensor, ignore_index: int = -100, reduction: str = "mean",
                        z_loss_multiplier: float = 0.0, logit_softcap: float = 0.0):
    """(loss, z_loss).  Labels outside [0, V) other than ``ignore_index`` contribute zero loss but still count in the
    mean, as a one-hot of an out-of-range class is all zero (``olmax/nn/functional.py:70-91``)."""
    lf = softcap(logits.float(), logit_softcap)
    V = lf.shape[-1]
    lf2 = lf.reshape(-1, V)
    lab = labels.reshape(-1)
    lse = torch.logsumexp(lf2, dim=-1)
    counted = lab != ignore_index
    in_range = counted & (lab >= 0) & (lab < V)
    tgt = lf2.gather(1, lab.clamp(0, V - 1).view(-1, 1)).view(-1)
    per_tok = torch.where(in_range, lse - tgt, torch.zeros_like(lse))
    z = torch.where(counted, lse.pow(2), torch.zeros_like(lse)) * z_loss_multiplier
    if reduction == "mean":
        n = counted.sum().clamp(min=1)
        return per_tok.sum() / n, z.sum() / n
    if reduction == "sum":
        return per_tok.sum(), z.sum()
    return per_tok.view(labels.shape), z.view(labels.shape)


# ----------------------------------------------------------------------------------------------------------------------
# The LM head's distribution p = softmax(y), y = softcap(z) / temperature of logits z [rows, V]
# ----------------------------------------------------------------------------------------------------------------------
def _distribution(z: torch.Tensor, cap: float, temperature: float):
    """(y, dy/dz, lse) in fp32 (fp64 for fp64 logits)."""
    zf = z if z.dtype == torch.float64 else z.float()
    slope = torch.full_like(zf, 1.0 / temperature)
    if cap and cap > 0:
        t = torch.tanh(zf / cap)
        zf, slope = cap * t, slope * (1.0 - t * t)
    y = zf / temperature
    return y, slope, torch.logsumexp(y, dim=-1)


def _log_p(y: torch.Tensor, lse: torch.Tensor) -> torch.Tensor:
    """log p; a row without any class (lse = -inf) has -inf everywhere."""
    return y - torch.where(lse == -math.inf, torch.zeros_like(lse), lse).unsqueeze(-1)


def token_log_probs(z: torch.Tensor, ids: Optional[torch.Tensor], top_k: int = 0, ignore_index: int = -100, cap: float = 0.0,
                    temperature: float = 1.0):
    """(log p of ids or None, entropy, lse, top log p or None, top ids or None) of logits z [rows, V]: the top classes are
    those with the largest logits, equal ones in the order of their ids."""
    V = z.shape[-1]
    y, _, lse = _distribution(z, cap, temperature)
    lp = _log_p(y, lse)
    entropy = -torch.where(lp > -math.inf, lp.exp() * lp, torch.where(lp.isnan(), lp, torch.zeros_like(lp))).sum(-1)
    taken = None
    if ids is not None:
        known = (ids != ignore_index) & (ids >= 0) & (ids < V)
        taken = torch.where(known, lp.gather(-1, ids.clamp(0, V - 1).unsqueeze(-1)).squeeze(-1), torch.zeros_like(lse))
    if not top_k:
        return taken, entropy, lse, None, None
    top_ids = z.sort(dim=-1, descending=True, stable=True).indices[:, :top_k].contiguous()
    return taken, entropy, lse, lp.gather(-1, top_ids), top_ids


def token_log_probs_bwd(z: torch.Tensor, ids: Optional[torch.Tensor], g_log_probs: Optional[torch.Tensor],
                        g_entropy: Optional[torch.Tensor], ignore_index: int = -100, cap: float = 0.0,
                        temperature: float = 1.0) -> torch.Tensor:
    """d(sum g_log_probs log p + sum g_entropy H) / dz = dy/dz (g_lp (onehot - p) - g_H p (log p + H))."""
    V = z.shape[-1]
    y, slope, lse = _distribution(z, cap, temperature)
    lp = _log_p(y, lse)
    p = lp.exp()
    d = torch.zeros_like(p)
    if g_entropy is not None:
        weighted = torch.where(p > 0, lp, torch.zeros_like(lp))
        entropy = -(p * weighted).sum(-1, keepdim=True)
        d = d - g_entropy.to(p.dtype).unsqueeze(-1) * p * torch.where(p > 0, lp + entropy, torch.zeros_like(lp))
    if g_log_probs is not None:
        known = (ids != ignore_index) & (ids >= 0) & (ids < V)
        g = torch.where(known, g_log_probs.to(p.dtype), torch.zeros_like(lse)).unsqueeze(-1)
        d = (d - g * p).scatter_add(-1, ids.clamp(0, V - 1).unsqueeze(-1), g)
    return (torch.where((lse == -math.inf).unsqueeze(-1), torch.zeros_like(d), d) * slope).to(z.dtype)


def _teacher(teacher_ids: torch.Tensor, values: torch.Tensor, V: int, renormalize: bool):
    """(valid pairs, their masses, log of these, rows with a teacher): of several pairs with one id the first counts."""
    ids = teacher_ids.long()
    first = ~((ids.unsqueeze(-1) == ids.unsqueeze(-2)).tril(-1).any(-1))
    valid = (ids >= 0) & (ids < V) & first
    t = torch.where(valid, values.double(), torch.full_like(values, -math.inf, dtype=torch.float64))
    some = (valid & ~(t == -math.inf)).any(-1) if renormalize else valid.any(-1)
    log_q = t
    if renormalize:
        norm = torch.logsumexp(t, dim=-1, keepdim=True)
        log_q = t - torch.where(norm == -math.inf, torch.zeros_like(norm), norm)
    return valid, log_q.exp(), log_q, some


def _distillation_parts(z, teacher_ids, values, renormalize, cap, temperature):
    V = z.shape[-1]
    y, slope, lse = _distribution(z, cap, temperature)
    valid, q, log_q, some = _teacher(teacher_ids, values, V, renormalize)
    at = torch.where(valid, teacher_ids.long(), torch.full_like(teacher_ids, V, dtype=torch.int64))
    named = torch.zeros(z.shape[0], V + 1, dtype=torch.bool, device=z.device).scatter(-1, at, True)[:, :V]
    rest_lse = torch.logsumexp(y.masked_fill(named, -math.inf), dim=-1)
    rest = torch.zeros_like(q[:, 0])
    if not renormalize:
        rest = torch.where(rest_lse == -math.inf, rest, (1.0 - q.sum(-1)).clamp(min=0.0))
    return y, slope, lse, valid, q, log_q, some, at, named, rest_lse, rest


def distillation(z: torch.Tensor, teacher_ids: torch.Tensor, values: torch.Tensor, renormalize: bool, cap: float = 0.0,
                 temperature: float = 1.0):
    """(loss per row, rows with a teacher) for logits z [rows, V] and a teacher's [rows, k] pairs of class and log probability;
    see ``ops/functional.py: distillation_loss``."""
    y, _, lse, valid, q, log_q, some, at, _, rest_lse, rest = _distillation_parts(z, teacher_ids, values, renormalize, cap, temperature)
    V = z.shape[-1]
    lp = _log_p(y, lse).gather(-1, at.clamp(max=V - 1)).double()
    terms = torch.where(valid & ~(q == 0), q * (log_q - lp), torch.zeros_like(q))
    rest_lp = rest_lse.double() - lse.double()
    loss = terms.sum(-1) + torch.where(rest > 0, rest * (rest.log() - rest_lp), torch.zeros_like(rest))
    return torch.where(some, loss, torch.zeros_like(loss)).to(y.dtype), some


def distillation_bwd(z: torch.Tensor, teacher_ids: torch.Tensor, values: torch.Tensor, g: torch.Tensor, renormalize: bool,
                     cap: float = 0.0, temperature: float = 1.0) -> torch.Tensor:
    """d(sum g loss) / dz: M p - q for the teacher's classes, e^(y - L) (M e^(L - lse) - rest) for the others, whose
    log-sum-exp is L; M = sum q + rest."""
    y, slope, lse, valid, q, _, some, at, named, rest_lse, rest = _distillation_parts(z, teacher_ids, values, renormalize, cap, temperature)
    V = z.shape[-1]
    total = q.sum(-1) + rest
    p = _log_p(y, lse).exp()
    safe = torch.where(rest_lse == -math.inf, torch.zeros_like(rest_lse), rest_lse)
    coef = torch.where(rest_lse == -math.inf, torch.zeros_like(total), total * (safe - lse).double().exp() - rest).to(y.dtype)
    others = (y - safe.unsqueeze(-1)).masked_fill(named, -math.inf).exp() * coef.unsqueeze(-1)
    d = torch.where(named, total.to(y.dtype).unsqueeze(-1) * p, others)
    d = d.scatter_add(-1, at.clamp(max=V - 1), torch.where(valid, -q, torch.zeros_like(q)).to(y.dtype))
    alive = (some & (lse != -math.inf)).unsqueeze(-1)
    return torch.where(alive, d * slope * g.to(y.dtype).unsqueeze(-1), torch.zeros_like(d)).to(z.dtype)
