"""How the kernels over the LM head's distribution are called: grad mode, forward-mode derivatives, upstream factors, repeated teachers, masks."""

import math

import pytest
import torch
from torch.autograd import forward_ad

pytestmark = pytest.mark.gpu

from olmax_b200.nn import LMHead
from olmax_b200.nn.module import build_module
from olmax_b200.ops import functional as F
from olmax_b200.ops import kernels as K
from olmax_b200.parallel import MeshResource
from olmax_b200.testing.token_probs import distillation_64, scores_64

DEV = "cuda"


def _head(V=512, d=64, cap=None):
    return build_module(lambda: LMHead(d, V, logit_softcap=cap), mesh_resource=MeshResource.FSDP(1), device=torch.device(DEV))


def _inputs(rows=24, V=512, d=64, k=3, seed=1):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(rows, d, generator=g, device=DEV).to(torch.bfloat16)
    t = torch.randn(rows, V, generator=g, device=DEV).log_softmax(-1).topk(k, dim=-1)
    return x, t.indices, t.values


def test_losses_without_grad_mode_leave_no_gradient():
    head = _head()
    x, ids, t = _inputs()
    x.requires_grad_(True)
    labels = torch.arange(24, device=DEV)
    for call in (lambda: head.distillation_loss(x, ids, t), lambda: head.loss(x, labels)[0]):
        with torch.no_grad():
            loss = call()
        assert not loss.requires_grad and float(head.store.grad.abs().max()) == 0
        # (the cross entropy adds its 24 rows in any order: 24 roundings of the sum)
        assert abs(float(call().detach()) - float(loss)) <= 24 * 2.0 ** -24 * abs(float(loss)) and float(head.store.grad.abs().max()) > 0
        head.store.zero_grad()


def test_forward_mode_derivatives_reach_no_kernel():
    head = _head()
    x, ids, t = _inputs()
    z, lab = torch.randn(24, 512, device=DEV), torch.zeros(24, dtype=torch.int64, device=DEV)
    before = K.launch_count()
    for mode in (torch.no_grad, torch.enable_grad):
        for call in (lambda z, x: F.token_log_probs(z, lab), lambda z, x: head.token_log_probs(x, lab), lambda z, x: F.distillation_loss(z, ids, t),
                     lambda z, x: head.distillation_loss(x, ids, t)):
            with mode(), forward_ad.dual_level(), pytest.raises(NotImplementedError):
                call(forward_ad.make_dual(z, torch.ones_like(z)), forward_ad.make_dual(x, torch.ones_like(x)))
    assert K.launch_count() == before


@pytest.mark.parametrize("int_type", [torch.int64, torch.int32])
def test_a_repeated_class_whose_first_pair_is_nothing_is_no_teacher(int_type):
    """Of several pairs with one id the first counts; renormalised, a row with none above -inf has no teacher and does not enter the mean, neither
    the loss's nor the gradient's, which are divided by counts of their own."""
    head = _head()
    x, ids, t = _inputs(rows=24)
    ids[::3, 1] = ids[::3, 0]
    ids[::3, 2] = -1
    t[::3, 0], t[::3, 1] = -math.inf, -1.0                 # the second pair of these rows does not count
    ids[1, 2], t[1, 0] = ids[1, 1], -math.inf              # here the second does, the third does not
    results = []
    for blank in (False, True):
        i2 = ids.clone()
        if blank:
            i2[::3] = -1
        leaf = x.clone().requires_grad_(True)
        head.store.zero_grad()
        loss = head.distillation_loss(leaf, i2.to(int_type), t, tail="renormalize")
        dx, = torch.autograd.grad(loss, leaf)
        results.append((loss.detach(), dx, head.store.full_gradient("proj.weight").clone()))
    for a, b in zip(*results):
        assert torch.equal(a, b)
    z = x.double() @ head.weight.full().double().t()
    want, dz = distillation_64(z, ids, t, "renormalize")
    # logits of 64 exact products each, off by less than 64 * 2^-24 of the sum of their absolute values; statistics and logarithms some steps of 2^-24
    e = 2.0 ** -24 * (2 * 64 * float((x.double().abs() @ head.weight.full().double().abs().t()).max()) + 64)
    assert abs(float(results[0][0]) - float(want)) <= e * 4
    w = head.weight.full().double()
    size = dz.abs() @ w.abs()
    assert torch.all((results[0][1].double() - dz @ w).abs() <= (2.0 ** -8 + 2.0 ** -12 + 4 * e) * size + 2.0 ** -8 * (dz @ w).abs() + 1e-12)


def test_a_scaled_distillation_loss_of_the_head_is_reported():
    """As on the CPU, but without waiting for the GPU: in the kernels' status word, which the trainer reads every step."""
    from olmax_b200.ops import _lib

    head = _head()
    x, ids, t = _inputs()
    x.requires_grad_(True)
    _lib.check_status()
    (head.distillation_loss(x, ids, t, weight=0.5) + 3 * x.float().square().mean()).backward()
    _lib.check_status()
    (0.5 * head.distillation_loss(x, ids, t)).backward()
    with pytest.raises(_lib.KernelError, match="factor"):
        _lib.check_status()
    _lib.check_status()                                    # told once


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [7, 1003, 40000])
def test_masked_classes_under_a_soft_cap(V, dtype):
    """-cap, as the formula has it: in whole vectors and single classes, of rows of one CTA and of several."""
    cap = 5.0
    z = (torch.randn(4, V, generator=torch.Generator(device=DEV).manual_seed(2), device=DEV) * 3).to(dtype)
    z[0, 1::2], z[1, V // 2:], z[2], z[3, :1] = -math.inf, -math.inf, -math.inf, math.inf
    ids = torch.tensor([1, V - 1, 0, 0], device=DEV)
    k = min(V, 9)
    out = F.token_log_probs(z, ids, top_k=k, logit_softcap=cap)
    lp, ent, top, top_ids = scores_64(z, ids, k, 1.0, cap)
    # steps of 2^-24: a log p is at most 2 cap + log V and off by 24 |y| + 16; the sum of V terms of a CTA of 256 threads by V / 256 + 32
    tol = 2.0 ** -24 * (24 * cap + 16 + V / 256 + 32 + 4 * (2 * cap + math.log(V)))
    assert torch.equal(out.top_ids, top_ids)
    for a, b in ((out.log_probs, lp), (out.entropy, ent), (out.top_log_probs, top)):
        assert float((a.double() - b).abs().max()) <= tol * (1 + math.log(V))
