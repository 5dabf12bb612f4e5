"""How log probabilities and distillation are called, on CPU: grad mode, upstream factors, forward-mode derivatives, repeated teachers, masks."""

import math

import pytest
import torch

from olmax_b200.nn import LMHead
from olmax_b200.nn.module import build_module
from olmax_b200.ops import functional as F
from olmax_b200.parallel import MeshResource


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
