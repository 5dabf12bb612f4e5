"""
Long rows whose answer changes when a single class is lost, counted twice or taken from another row: equal logits, whose sum is the number of classes
exactly, and rows with all their mass on one class, at every border of the kernels' slices, batches, vectors and tiles.
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from olmax_b200.nn import LMHead
from olmax_b200.nn.module import build_module
from olmax_b200.ops import functional as F
from olmax_b200.parallel import MeshResource
from olmax_b200.testing.token_probs import distillation_64

DEV = "cuda"
STEP = 2.0 ** -24


def _log_tol(V):
    """Equal logits: exponents of 0, sums of ones, which fp32 holds exactly.  What is left are the logarithm to the base 2 (2 steps), ln 2 (1) and their
    product (1).  A class more or less changes log V by 1 / V, which is more up to V = 2^18."""
    return 4 * STEP * math.log(V)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows", [1, 9, 40, 100, 400])           # clusters of eight CTAs per row, and fewer, down to one
@pytest.mark.parametrize("V", [4099, 50257, 100352, 200003, 256000])
def test_equal_logits(V, rows, dtype):
    buf = torch.full((rows, V + 8), 3.0, device=DEV, dtype=dtype)
    ids = (torch.arange(rows, device=DEV) * 977) % V
    for first in (0, 3):
        z = buf[:, first : first + V]
        for cap, k in ((0.0, 0), (0.0, 5), (30.0, 0)):
            out = F.token_log_probs(z, ids, top_k=k, logit_softcap=cap)
            assert 1.0 / V > _log_tol(V)
            assert float((out.log_probs.double() + math.log(V)).abs().max()) <= _log_tol(V)
            assert float((out.entropy.double() - math.log(V)).abs().max()) <= _log_tol(V)
            if k:
                assert torch.equal(out.top_ids, torch.arange(5, device=DEV).expand(rows, 5))
        # half of the mass on three classes: the other V - 3 have a log-sum-exp of log(V - 3) + 3, of which the loss takes a half
        t_ids = torch.stack([ids, (ids + 1) % V, (ids + V // 2) % V], -1)
        t = torch.full((rows, 3), math.log(1 / 6), device=DEV)
        for cap in (0.0, 30.0):
            leaf = z.detach().requires_grad_(True)
            loss = F.distillation_loss(leaf, t_ids, t, reduction="none", logit_softcap=cap)
            g, = torch.autograd.grad(loss, leaf, torch.ones(rows, device=DEV))
            q = 3 * math.exp(float(t[0, 0]))
            want = q * (float(t[0, 0]) + math.log(V)) + (1 - q) * (math.log(1 - q) + math.log(V) - math.log(V - 3))
            assert float((loss.detach().double() - want).abs().max()) <= 2 * STEP * want and (1 - q) / V > 2 * STEP * want
            slope = 1 - math.tanh(0.1) ** 2 if cap else 1.0
            named, others = (1 / V - q / 3) * slope, (1 / V - (1 - q) / (V - 3)) * slope
            rounding = 2.0 ** -8 if dtype == torch.bfloat16 else 0.0
            # (a probability is off by some steps of log V and of its exponential's argument)
            full = torch.full((rows, V), others, dtype=torch.float64, device=DEV).scatter_(1, t_ids, named)
            size = torch.full((rows, V), 1 / V + (1 - q) / (V - 3), dtype=torch.float64, device=DEV).scatter_(1, t_ids, 1 / V + q / 3)
            assert torch.all((g.double() - full).abs() <= 64 * STEP * size + rounding * full.abs())


def _borders(V, lead):
    """Classes around the borders: a row's ends, its vectors, batches of 256 threads and of all their loads, and the slices of one to eight CTAs."""
    at = {0, V}
    for step in (256 * 4, 256 * 8, 256 * 16):
        at |= {lead + step, lead + 2 * step, lead + V // step * step, lead + (V // step - 1) * step}
    for C in (2, 4, 8):
        at |= {lead + V * i // C for i in range(1, C)}
    found = {p + o for p in at for o in (-9, -8, -5, -4, -3, -2, -1, 0, 1, 2, 3, 4, 7, 8)}
    return sorted(p for p in found if 0 <= p < V)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V,first", [(50257, 1), (100352, 0), (9001, 3)])
def test_all_mass_on_one_class(V, first, dtype):
    lead = -first % (16 // (4 if dtype == torch.float32 else 2))
    at = _borders(V, lead)
    buf = torch.full((len(at), V + 8), -1000.0, device=DEV, dtype=dtype)
    z, ids = buf[:, first : first + V], torch.tensor(at, device=DEV)
    z.scatter_(1, ids[:, None], 2.0)
    n = torch.arange(len(at), device=DEV)
    for part in (slice(0, None), *(slice(r, r + 16) for r in range(0, len(at), 16))):      # a CTA per row; clusters of eight
        zp, ip = z[part], ids[part]
        for k in (0, 3):
            out = F.token_log_probs(zp, ip, top_k=k)
            assert torch.all(out.log_probs == 0) and torch.all(out.entropy == 0)
            if k:
                assert torch.equal(out.top_ids[:, 0], ip) and torch.all(out.top_log_probs[:, 0] == 0)
        # a teacher that names another class: all of the student's mass is the rest's, and as large as the teacher leaves
        other = ((ip + 1) % V)[:, None]
        leaf = zp.detach().requires_grad_(True)
        loss = F.distillation_loss(leaf, other, torch.full_like(other, math.log(0.25), dtype=torch.float32), reduction="none")
        want, _ = distillation_64(zp[:1], other[:1], torch.full((1, 1), math.log(0.25), device=DEV), "rest", "none")
        assert float((loss.detach().double() - want).abs().max()) <= 8 * STEP * float(want)
        g, = torch.autograd.grad(loss, leaf, torch.ones(len(zp), device=DEV))
        m = torch.arange(len(zp), device=DEV)
        # total p - rest = 1 - 3/4 at the student's class, -1/4 at the teacher's, nothing elsewhere
        assert torch.all((g[m, ip].double() - 0.25).abs() <= 2.0 ** -8) and torch.all((g[m, other[:, 0]].double() + 0.25).abs() <= 2.0 ** -8)
        assert torch.all((g != 0).sum(1) == 2)
    assert torch.equal(z.argmax(1), ids) and len(n) > 148


@pytest.mark.parametrize("tokens", [1, 9, 16, 17, 130, 300, 1000])
@pytest.mark.parametrize("V", [4096 + 8, 50304, 100352])
def test_equal_logits_of_the_head(V, tokens):
    """Equal rows of the weight give equal products, whatever the order of their sums."""
    d = 64
    head = build_module(lambda: LMHead(d, V), mesh_resource=MeshResource.FSDP(1), device=torch.device(DEV))
    g = torch.Generator(device=DEV).manual_seed(1)
    head.store.load_full("proj.weight", (torch.randn(d, generator=g, device=DEV) * 0.3).to(torch.bfloat16).expand(V, d))
    head.store.sync_shadow()
    x = torch.randn(tokens, d, generator=g, device=DEV).to(torch.bfloat16)
    with torch.no_grad():
        out = head.token_log_probs(x, (torch.arange(tokens, device=DEV) * 977) % V)
    assert 1.0 / V > _log_tol(V)
    assert float((out.log_probs.double() + math.log(V)).abs().max()) <= _log_tol(V)
    assert float((out.entropy.double() - math.log(V)).abs().max()) <= _log_tol(V)


@pytest.mark.parametrize("tokens", [16, 64, 256])
@pytest.mark.parametrize("V", [8192 + 8, 50304])
def test_all_mass_on_one_class_of_the_head(V, tokens):
    """Token r has a logit of 64 at a class of its own beside a border of the tiles, and 0 elsewhere; a lost class leaves the entropy of V equal ones."""
    step = [0, 64, 128, 256, 512, V - 256, V - 128, V - 64, V - 8, V]
    at = sorted({p + o for p in step for o in (-2, -1, 0, 1, 7, 8, 31, 32, 33) if 0 <= p + o < V})
    at = (at * (tokens // len(at) + 1))[:tokens] if tokens >= len(at) else at[:: len(at) // tokens][:tokens]
    d = 256
    head = build_module(lambda: LMHead(d, V), mesh_resource=MeshResource.FSDP(1), device=torch.device(DEV))
    w = torch.zeros(V, d, device=DEV)
    w[torch.tensor(at, device=DEV), torch.arange(tokens, device=DEV)] = 64.0
    head.store.load_full("proj.weight", w)
    head.store.sync_shadow()
    x = torch.eye(tokens, d, device=DEV).to(torch.bfloat16)
    with torch.no_grad():
        out = head.token_log_probs(x, torch.tensor(at, device=DEV))
    # V e^-64 is below 1e-22
    assert torch.all(out.log_probs.abs() <= 1e-20) and torch.all(out.entropy.abs() <= 1e-18)
