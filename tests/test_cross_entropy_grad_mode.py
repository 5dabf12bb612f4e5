"""A cross entropy evaluated without grad mode leaves no gradient behind, whatever its input says about itself."""

import pytest
import torch
from torch.autograd import forward_ad

from olmax_b200.nn import LMHead
from olmax_b200.nn.module import build_module
from olmax_b200.parallel import MeshResource
from olmax_b200.testing import run_distributed_test


def _evaluate(head, rows=6, V=40, d=16):
    x = torch.randn(rows, d, generator=torch.Generator().manual_seed(1)).requires_grad_(True)
    labels = torch.arange(rows) % V
    with torch.no_grad():
        loss, _ = head.loss(x, labels)
    assert not loss.requires_grad and float(head.store.grad.abs().max()) == 0
    again, _ = head.loss(x, labels)
    assert torch.equal(again.detach(), loss) and float(head.store.grad.abs().max()) > 0


def test_cross_entropy():
    _evaluate(build_module(lambda: LMHead(16, 40), mesh_resource=MeshResource.FSDP(1), device=torch.device("cpu")))


def _check_vocab_parallel():
    _evaluate(build_module(lambda: LMHead(16, 40, vocab_parallel=True), mesh_resource=MeshResource.FSDP_with_TP(2, 2), device=torch.device("cpu")))


def test_vocabulary_parallel_cross_entropy():
    run_distributed_test(_check_vocab_parallel, world_size=2)


def test_a_forward_mode_derivative_is_refused_in_either_mode():
    head = build_module(lambda: LMHead(16, 40), mesh_resource=MeshResource.FSDP(1), device=torch.device("cpu"))
    x, labels = torch.randn(6, 16), torch.arange(6)
    for mode in (torch.no_grad, torch.enable_grad):
        with mode(), forward_ad.dual_level(), pytest.raises(NotImplementedError):
            head.loss(forward_ad.make_dual(x, torch.ones_like(x)), labels)
