"""
How exact the kernels over the LM head's distribution are: few classes, where every rounding can be counted, and long rows whose answer a
lost class would change.  A step is 2^-24 of the value, the most that rounding to fp32 changes one.
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from olmax_b200.nn import LMHead
from olmax_b200.nn.module import build_module
from olmax_b200.ops import functional as F
from olmax_b200.parallel import MeshResource
from olmax_b200.testing.token_probs import distillation_64, score_gradients_64, scores_64

DEV = "cuda"
STEP = 2.0 ** -24

# A capped logit y = cap tanh(z / cap).  |z| <= 3/4 cap: z g(s), s = (z / cap)^2: g's polynomial is off by 0.5 step, the four roundings in s move
# g by at most 0.16 as much, Horner's sums by 1.5, the product by 1: below 4 steps of y.  Beyond: cap (1 - 2 w), w = e / (1 + e) <= 0.19, e = e^-2u: e
# is off by 6 steps (its exponent's two roundings count 2 u-fold), of which 2 w (1 - w) <= 0.30 arrive, with the product's five: below 4 steps of cap, 6 of y.
# log p = ln 2 ((y - m) c - log2 s): the difference, c, its product and ln 2 five steps of |y - m|; 2^t 3 steps and its exponent's; the logarithm,
# the difference and the last product 6 steps of |log p| + 1.  With y and m at most `y`: below 24 steps of y and 16 of 1.


def _tol(y):
    return STEP * (24 * y + 16)


def _close(got, want, tol, what=""):
    off = (got.double() - want.double()).abs()
    assert torch.all(off <= tol), (what, float(off.max()), float((off - tol).max()))


def _pairs(cap, dtype):
    """Rows of eight classes: z, 0 and six at the cap's lower end; z on both sides of the cap, small ones among them."""
    z = torch.cat([torch.linspace(-3 * cap, 3 * cap, 301, device=DEV), cap * 2.0 ** -torch.arange(1, 20, device=DEV),
                   -cap * 1.37 ** -torch.arange(1.0, 30, device=DEV), torch.tensor([cap, -cap, 40 * cap, -40 * cap], device=DEV)]).to(dtype)
    rows = torch.full((z.numel(), 8), -100 * cap, device=DEV, dtype=dtype)
    rows[:, 0], rows[:, 1] = z, 0.0
    return rows


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("cap", [5.0, 30.0, 256.0])
def test_capped_logits_are_exact_to_a_few_steps(cap, dtype):
    z = _pairs(cap, dtype)
    y = (cap * torch.tanh(z[:, 0].double() / cap)).abs()
    for part in (z, z[:, :2], z[:, :3]):        # whole vectors, and single classes
        n = part.shape[1]
        for first in (0, 1):
            ids = torch.full((part.shape[0],), first, device=DEV)
            out = F.token_log_probs(part, ids, top_k=2, logit_softcap=cap)
            lp, ent, top, top_ids = scores_64(part, ids, 2, 1.0, cap)
            _close(out.log_probs, lp, _tol(y), (n, first))
            _close(out.top_log_probs, top, _tol(y)[:, None], (n, first))
            # (the other six weigh e^-cap each, their terms cap + y times that)
            _close(out.entropy, ent, _tol(y) + STEP * 64 * cap * math.exp(-cap) * 6, (n, first))
            assert torch.equal(out.top_ids, top_ids)


@pytest.mark.parametrize("cap", [5.0, 30.0, 256.0])
def test_gradients_of_capped_logits_are_exact_to_a_few_steps(cap):
    """In fp32: a probability is off by its exponent's error, the slope 1 - tanh^2 by 24 steps (near the cap's ends 4 w (1 - w))."""
    z = _pairs(cap, torch.float32)
    rows = z.shape[0]
    ids = torch.zeros(rows, dtype=torch.int64, device=DEV)
    y = (cap * torch.tanh(z[:, 0].double() / cap)).abs()[:, None]
    gl, ge = torch.linspace(-1, 1, rows, device=DEV), torch.linspace(1, -0.5, rows, device=DEV)
    for a, b in ((gl, 0 * ge), (0 * gl, ge)):
        leaf = z.clone().requires_grad_(True)
        out = F.token_log_probs(leaf, ids, logit_softcap=cap)
        got, = torch.autograd.grad((out.log_probs, out.entropy), leaf, (a, b))
        want, size = score_gradients_64(z, ids, a, b, 1.0, cap)
        # The entropy's gradient is -p (log p + H) slope, where log p and H may cancel: each is off by a _tol(y), whatever is left of them.  The oracle's own
        # slope: tanh, its square and the difference from 1 are off by half of 2^-52 each, where the kernel's form has no such limit; it stands before
        # terms of |g| (1 + p) + |g| p (|log p| + H) <= 4, p |log p| and H being below 1.1 for two classes.
        part = b.abs()[:, None] * (torch.softmax(cap * torch.tanh(z.double() / cap), -1) * (1 - torch.tanh(z.double() / cap) ** 2))[:, :2]
        _close(got[:, :2], want[:, :2], ((_tol(y) * 2 + 24 * STEP) * size)[:, :2] + 2 * _tol(y) * part + 4 * 1.5 * 2.0 ** -52)
    t_ids = torch.tensor([[0, 1]], device=DEV).expand(rows, 2)
    t = torch.log(torch.tensor([[0.5, 0.25]], device=DEV)).expand(rows, 2)
    for tail in ("rest", "renormalize"):
        leaf = z.clone().requires_grad_(True)
        loss = F.distillation_loss(leaf, t_ids, t, tail=tail, reduction="none", logit_softcap=cap)
        got, = torch.autograd.grad(loss, leaf, torch.ones(rows, device=DEV))
        want, grads = distillation_64(z, t_ids, t, tail, "none", 1.0, cap)
        # the rest's log-sum-exp lies at -cap: a difference of logarithms of that size
        _close(loss.detach(), want, 2 * _tol(y[:, 0] + (cap if tail == "rest" else 0)), tail)
        slope = 1 - torch.tanh(z[:, :2].double() / cap) ** 2
        _close(got[:, :2], grads[:, :2], (2 * _tol(y) + 24 * STEP) * 2 * slope + 2 * 1.5 * 2.0 ** -52, tail)


@pytest.mark.parametrize("rows", [9, 300])
def test_capped_logits_out_of_the_heads_epilogue(rows):
    """Products that are exact (one factor is a power of two, the others zeros), so that the capped logit's error is all there is."""
    V, d, cap = 512, 64, 256.0
    head = build_module(lambda: LMHead(d, V, logit_softcap=cap), mesh_resource=MeshResource.FSDP(1), device=torch.device(DEV))
    w = torch.zeros(V, d, device=DEV)
    w[:, 0] = -60000.0
    w[0, 0], w[1, 0], w[2, 0] = 0.0, 3.0, -1.5
    head.store.load_full("proj.weight", w.to(torch.bfloat16))
    head.store.sync_shadow()
    x = torch.zeros(rows, d, device=DEV)
    x[:, 0] = 2.0 ** -(torch.arange(rows, device=DEV) % 8)
    x = x.to(torch.bfloat16)
    ids = torch.arange(rows, device=DEV) % 3
    z = x.double() @ w.to(torch.bfloat16).double().t()
    lp, ent, _, _ = scores_64(z, ids, 1, 1.0, cap)
    with torch.no_grad():
        out = head.token_log_probs(x, ids)
    _close(out.log_probs, lp, _tol(3.0))
    _close(out.entropy, ent, 2 * _tol(3.0))


@pytest.mark.parametrize("V,k,temperature,cap,dtype", [(50257, 16, 2.0, 0.0, torch.float32), (100352, 64, 2.0, 0.0, torch.float32), (32000, 8, 3.0, 0.0, torch.float32),
                                                       (256000, 128, 2.0, 0.0, torch.bfloat16), (100352, 64, 2.0, 30.0, torch.bfloat16)])
@pytest.mark.parametrize("rows", [2, 64, 200])
def test_a_small_distillation_loss(rows, V, k, temperature, cap, dtype):
    """
    A student near its teacher, most of whose mass P (the teacher's: Q) is the rest's.  The loss is a difference of logarithms of sums, of which the rest's
    is a part of the whole: an error e of the rest's sum counts (1 - P) - (1 - Q) times, one of the named classes' sum P times.  e: the exponential is off by
    2.4 steps, its exponent (|t| <= 12 where the mass lies) by 2.5 ln 2 |t| = 21; a thread adds 16 terms a batch, V / 4096 batches, 256 threads in a tree:
    8 + V / 4096 + 8.  The logits of named classes enter in 64 bits, capped ones off by 4 steps of |y| / T.
    """
    g = torch.Generator(device=DEV).manual_seed(3)
    z = (torch.randn(rows, V, generator=g, device=DEV) * 2).to(dtype)
    y = z.double() + 0.1 * torch.randn(rows, V, generator=g, device=DEV)
    y = cap * torch.tanh(y / cap) if cap else y
    t = torch.log_softmax(y / temperature, -1).topk(k, -1)
    ids, values = t.indices, t.values.float()
    loss = F.distillation_loss(z, ids, values, temperature=temperature, logit_softcap=cap, reduction="none")
    want, _ = distillation_64(z, ids, values, "rest", "none", temperature, cap)
    ys = (cap * torch.tanh(z.double() / cap) if cap else z.double()) / temperature
    named = torch.log_softmax(ys, -1).gather(1, ids).exp().sum(1) + values.double().exp().sum(1)
    e = STEP * (2.4 + 21 + 16 + V / 4096 + (4 * float(ys.abs().max()) if cap else 0))
    _close(loss, want, e * named + 2 * STEP * want)
