"""How log probabilities and distillation are called, on CPU: grad mode, upstream factors, forward-mode derivatives, repeated teachers, masks."""

import math

import pytest
import torch
from torch.autograd import forward_ad

from olmax_b200.exceptions import OLMaxConfigurationError
from olmax_b200.nn import LMHead
from olmax_b200.nn.module import build_module
from olmax_b200.ops import functional as F
from olmax_b200.parallel import MeshResource
from olmax_b200.testing.token_probs import scores_64


def _head(V=40, d=16, cap=None):
    return build_module(lambda: LMHead(d, V, logit_softcap=cap), mesh_resource=MeshResource.FSDP(1), device=torch.device("cpu"))


def _inputs(rows=6, V=40, d=16, k=3):
    g = torch.Generator().manual_seed(1)
    x = torch.randn(rows, d, generator=g).requires_grad_(True)
    t = torch.randn(rows, V, generator=g).log_softmax(-1).topk(k, dim=-1)
    return x, t.indices, t.values


def test_a_distillation_loss_without_grad_mode_leaves_no_gradient():
    head = _head()
    x, ids, t = _inputs()
    with torch.no_grad():
        loss = head.distillation_loss(x, ids, t)
    assert not loss.requires_grad and float(head.store.grad.abs().max()) == 0
    again = head.distillation_loss(x, ids, t)
    assert torch.equal(again.detach(), loss) and float(head.store.grad.abs().max()) > 0


def test_forward_mode_derivatives_are_refused():
    """By all of them alike, in either grad mode; a tangent that a kernel never saw would read as zero."""
    head = _head()
    x, ids, t = _inputs()
    x = x.detach()
    z = torch.randn(6, 40)
    lab = torch.zeros(6, dtype=torch.int64)
    for mode in (torch.no_grad, torch.enable_grad):
        for call in (lambda z, x: F.token_log_probs(z, lab), lambda z, x: F.token_log_probs(z, top_k=2), lambda z, x: head.token_log_probs(x, lab),
                     lambda z, x: F.distillation_loss(z, ids, t), lambda z, x: head.distillation_loss(x, ids, t)):
            with mode(), forward_ad.dual_level():
                with pytest.raises(NotImplementedError):
                    call(forward_ad.make_dual(z, torch.ones_like(z)), forward_ad.make_dual(x, torch.ones_like(x)))
                call(z, x)                       # no tangent, no refusal
    with pytest.raises(NotImplementedError):
        torch.func.jvp(lambda z: F.token_log_probs(z, lab).log_probs, (z,), (torch.ones_like(z),))


def test_a_scaled_distillation_loss_of_the_head_is_refused():
    """The weight's gradient is formed in the forward pass: a factor behind it would scale one of the two gradients alone."""
    head = _head()
    x, ids, t = _inputs()
    for factor in (0.5, 0.0, math.nan):
        loss = head.distillation_loss(x, ids, t)
        with pytest.raises(RuntimeError):
            (factor * loss).backward()
        assert x.grad is None
    head.store.zero_grad()
    other = x.square().mean()
    (head.distillation_loss(x, ids, t, weight=0.5) + 3 * other).backward()      # a factor of the other loss is none of its own
    half = [x.grad - 6 * x.detach() / x.numel(), head.store.full_gradient("proj.weight").clone()]
    head.store.zero_grad()
    whole, = torch.autograd.grad(head.distillation_loss(x, ids, t), x)
    # (a few roundings of terms below 1: the mean's, the weight's, the sum's)
    assert float((half[0] - 0.5 * whole).abs().max()) < 8 * 2.0 ** -24
    assert float((half[1] - 0.5 * head.store.full_gradient("proj.weight")).abs().max()) < 8 * 2.0 ** -24


def test_the_trainer_refuses_a_z_loss_beside_a_teacher(tmp_path):
    """The distillation loss has no z-loss: a multiplier that would be dropped is refused."""
    from olmax_b200.models import DefaultTransformerConfig, DefaultTransformerLayerConfig
    from olmax_b200.nn import MultiheadSelfAttentionConfig
    from olmax_b200.optim import AdamWConfig, ConstantSchedule
    from olmax_b200.train import Trainer

    cfg = DefaultTransformerConfig(vocab_size=64, d_model=64, hidden_size=96, num_layers=1,
                                   layer=DefaultTransformerLayerConfig(attention=MultiheadSelfAttentionConfig(n_heads=4, head_dim=16)))
    model = cfg.build(seed=0, mesh_resource=MeshResource.FSDP(1), device=torch.device("cpu"))
    ids = torch.randint(0, 64, (2, 12), generator=torch.Generator().manual_seed(5))
    with torch.no_grad():
        best = model.token_log_probs(ids, top_k=4)
    trainer = Trainer(work_dir=tmp_path, save_folder=tmp_path, optim=AdamWConfig(lr=ConstantSchedule(1e-2)), z_loss_multiplier=1e-4)
    trainer.setup(model, 1)
    with pytest.raises(OLMaxConfigurationError):
        trainer.train_batch([(ids, best.top_ids, best.top_log_probs)])
    trainer.train_batch([(ids, ids)])
    trainer.z_loss_multiplier = 0.0
    trainer.train_batch([(ids, best.top_ids, best.top_log_probs)])


def test_a_soft_cap_makes_a_masked_class_one_of_the_lowest():
    """cap tanh(-inf / cap) = -cap: the formula has no masks, and the documentation says so."""
    z = torch.tensor([[1.0, 2.0, -math.inf], [-math.inf] * 3])
    out = F.token_log_probs(z, torch.tensor([2, 0]), top_k=3, logit_softcap=5.0)
    lp, ent, top, top_ids = scores_64(z, torch.tensor([2, 0]), 3, 1.0, 5.0)
    assert torch.allclose(out.log_probs.double(), lp, atol=2e-6) and torch.allclose(out.entropy.double(), ent, atol=2e-6)
    assert torch.allclose(out.top_log_probs.double(), top, atol=2e-6) and torch.equal(out.top_ids, top_ids)
    assert abs(float(out.log_probs[1]) + math.log(3)) < 2e-6
    # a mask that holds: cap the logits first
    y = torch.where(z == -math.inf, z, 5.0 * torch.tanh(z / 5.0))
    masked = F.token_log_probs(y, torch.tensor([2, 0]))
    assert masked.log_probs[0] == -math.inf and masked.log_probs[1] == -math.inf and masked.entropy[1] == 0


def test_the_heads_weight_gets_a_gradient_when_the_hidden_states_do():
    """As with the cross entropy: hidden states without requires_grad are scored, and nothing is recorded of the weight."""
    head = _head()
    x, ids, t = _inputs()
    for call in (lambda x: head.token_log_probs(x, ids[:, 0]).log_probs.sum(), lambda x: head.distillation_loss(x, ids, t), lambda x: head.loss(x, ids[:, 0])[0]):
        assert not call(x.detach()).requires_grad and float(head.store.grad.abs().max()) == 0
        call(x).backward()
        assert float(head.store.grad.abs().max()) > 0
        head.store.zero_grad()
