"""
Log probabilities of tokens, top classes and distillation on CPU: values and gradients against the definitions in 64 bits and
against differences, the same through the LM head, the model and the trainer, and what is refused.
"""

import math

import pytest
import torch

from olmax_b200.exceptions import OLMaxConfigurationError
from olmax_b200.models import DefaultTransformerConfig, DefaultTransformerLayerConfig
from olmax_b200.nn import LMHead, LMHeadConfig, MultiheadSelfAttentionConfig
from olmax_b200.nn import functional as NF
from olmax_b200.nn.module import build_module
from olmax_b200.ops import functional as F
from olmax_b200.ops import kernels as K
from olmax_b200.parallel import MeshResource
from olmax_b200.testing import run_distributed_test
from olmax_b200.testing.token_probs import distillation_64, scores_64


def _close(got, want, tol):
    got, want = got.double(), want.double()
    assert torch.equal(got.isnan(), want.isnan())
    same = (got == want) | got.isnan()
    assert torch.all(same | ((got - want).abs() <= tol)), float((got - want)[~same].abs().max())


def _rows(rows, V, seed=0, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(rows, V, generator=g) * 3).to(dtype)


# fp32 evaluation: y, its maximum and the log-sum-exp are rounded a few times relative to |y| <= 16, the sum of V terms in pairwise order
# (log2 V roundings): below 16 * 8 * 2^-24 + 32 * 2^-24 < 1e-5; tanh and the division by the temperature add a few more
TOL = 2e-5


@pytest.mark.parametrize("temperature,cap", [(1.0, 0.0), (0.7, 5.0)])
@pytest.mark.parametrize("rows,V,k", [(1, 1, 1), (3, 2, 2), (4, 33, 5), (5, 300, 128)])
def test_scores_against_64_bits(rows, V, k, temperature, cap):
    z = _rows(rows, V)
    ids = torch.arange(rows) % (V + 1) - 1 + (torch.arange(rows) % 3 == 2) * V   # -1, valid ones and beyond the last class
    out = NF.token_log_probs(z, ids, top_k=k, temperature=temperature, logit_softcap=cap or None)
    lp, ent, top, top_ids = scores_64(z, ids, k, temperature, cap)
    _close(out.log_probs, lp, TOL)
    _close(out.entropy, ent, TOL)
    _close(out.top_log_probs, top, TOL)
    assert torch.equal(out.top_ids, top_ids)
    # leading dimensions, and only what is asked for
    more = NF.token_log_probs(z.expand(2, rows, V), top_k=0, temperature=temperature, logit_softcap=cap)
    assert more.log_probs is None and more.top_ids is None and more.entropy.shape == (2, rows)


def test_scores_of_masked_and_empty_rows():
    z = _rows(5, 12)
    z[0, 3:] = -math.inf
    z[1] = -math.inf
    z[2, ::2] = torch.finfo(torch.float32).min
    z[3] = 1.5                       # every class equal
    z[4, 7] = math.nan
    ids = torch.tensor([0, 4, 1, 2, 3])
    z.requires_grad_(True)
    out = F.token_log_probs(z, ids, top_k=12)
    lp, ent, top, top_ids = scores_64(z.detach(), ids, 12, 1.0, 0.0)
    _close(out.log_probs, lp, TOL)
    _close(out.entropy, ent, TOL)
    _close(out.top_log_probs, top, TOL)
    assert torch.equal(out.top_ids, top_ids) and out.top_ids[3].tolist() == list(range(12))
    assert out.log_probs[1] == -math.inf and out.entropy[1] == 0
    g, = torch.autograd.grad((out.log_probs[:4].sum() + out.entropy[:4].sum()), z)
    assert torch.all(g[1] == 0) and torch.all(g[0, 3:] == 0) and torch.all(g[:4].isfinite())


@pytest.mark.parametrize("cap", [0.0, 4.0])
def test_score_gradients_by_differences(cap):
    z = _rows(6, 17, dtype=torch.float64).requires_grad_(True)
    ids = torch.tensor([0, 16, -100, 17, 3, 3])

    def fn(z):
        out = F.token_log_probs(z, ids, temperature=0.8, logit_softcap=cap)
        return out.log_probs, out.entropy

    assert torch.autograd.gradcheck(fn, (z,))


def _teacher(rows, V, k, seed=1, temperature=1.0):
    out = F.token_log_probs(_rows(rows, V, seed), top_k=k, temperature=temperature)
    return out.top_ids.clone(), out.top_log_probs.clone()


@pytest.mark.parametrize("tail", ["rest", "renormalize"])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_distillation_values_and_gradients(tail, reduction):
    rows, V, k = 7, 40, 6
    ids, t = _teacher(rows, V, k)
    ids[0] = -1                       # no teacher
    ids[1, 2:] = -1                   # a short list
    ids[2, 3] = ids[2, 1]             # a repeated class: the first counts
    ids[3, 0] = V                     # outside
    t[4, 5] = -math.inf
    z = _rows(rows, V, 2).requires_grad_(True)
    loss = NF.distillation_loss(z, ids, t, tail=tail, reduction=reduction, temperature=0.9, logit_softcap=6.0)
    want, grads = distillation_64(z.detach(), ids, t, tail, reduction, 0.9, 6.0)
    _close(loss.detach(), want, TOL)
    up = torch.linspace(-1, 1, rows) if reduction == "none" else torch.tensor(1.5)
    g, = torch.autograd.grad(loss, z, up)
    _close(g, grads * (up.unsqueeze(-1) if reduction == "none" else up), TOL)

    def fn(z):
        return F.distillation_loss(z, ids, t.double(), tail=tail, reduction=reduction, temperature=0.9, logit_softcap=6.0)

    assert torch.autograd.gradcheck(fn, (z.detach().double().requires_grad_(True),))


def test_distillation_of_the_students_own_distribution_is_zero():
    z = _rows(9, 50).requires_grad_(True)
    for k, tail in ((5, "rest"), (50, "rest"), (50, "renormalize")):
        out = F.token_log_probs(z.detach(), top_k=k)
        loss = F.distillation_loss(z, out.top_ids, out.top_log_probs, tail=tail)
        g, = torch.autograd.grad(loss, z)
        assert abs(float(loss.detach())) < TOL and float(g.abs().max()) < TOL


def test_distillation_without_a_teacher_or_without_others():
    z = _rows(4, 8).requires_grad_(True)
    none = torch.full((4, 3), -1)
    loss = F.distillation_loss(z, none, torch.zeros(4, 3))
    g, = torch.autograd.grad(loss, z)
    assert float(loss.detach()) == 0 and torch.all(g == 0)
    # every class outside the teacher's is masked: there is no further class, however little the teacher leaves to it
    ids, t = torch.tensor([[0, 1]]).expand(4, 2), torch.log(torch.tensor([[0.5, 0.4]])).expand(4, 2)
    masked = torch.full((4, 8), -math.inf)
    masked[:, :2] = 0.0
    masked.requires_grad_(True)
    loss = F.distillation_loss(masked, ids, t)
    g, = torch.autograd.grad(loss, masked)
    want = 0.5 * math.log(0.5 / 0.5) + 0.4 * math.log(0.4 / 0.5)
    assert abs(float(loss.detach()) - want) < TOL
    _close(g, torch.tensor([0.45 - 0.5, 0.45 - 0.4] + [0.0] * 6).expand(4, 8) / 4, TOL)
    # a class that the teacher likes and the student has masked
    assert float(F.distillation_loss(masked.detach(), torch.tensor([[3]] * 4), torch.zeros(4, 1))) == math.inf


def _head(V=40, d=16, cap=None):
    return build_module(lambda: LMHead(d, V, logit_softcap=cap), mesh_resource=MeshResource.FSDP(1), device=torch.device("cpu"))


@pytest.mark.parametrize("cap", [None, 5.0])
def test_head_scores_and_distillation_are_those_of_its_logits(cap):
    head = _head(cap=cap)
    w = head.store.full_parameter("proj.weight").clone().requires_grad_(True)
    x = torch.randn(2, 5, 16, generator=torch.Generator().manual_seed(3)).requires_grad_(True)
    ids = torch.arange(10).view(2, 5)
    ids[1, 1] = -100
    out = head.token_log_probs(x, ids, top_k=4, temperature=1.2)
    want = F.token_log_probs(x @ w.t(), ids, top_k=4, temperature=1.2, logit_softcap=cap)
    for a, b in zip(out, want):
        _close(a.detach(), b.detach(), TOL)
    objective = [(o.log_probs * torch.linspace(0, 1, 10).view(2, 5)).sum() + 0.3 * o.entropy.sum() for o in (out, want)]
    gx, = torch.autograd.grad(objective[0], x)
    wx, ww = torch.autograd.grad(objective[1], (x, w))
    _close(gx, wx, TOL)
    _close(head.store.full_gradient("proj.weight"), ww, TOL)
    head.store.zero_grad()
    t_ids, t = out.top_ids.flip(0), out.top_log_probs.detach().flip(0)
    loss = head.distillation_loss(x, t_ids, t, weight=0.25, temperature=1.2)
    want = 0.25 * F.distillation_loss(x @ w.t(), t_ids, t, temperature=1.2, logit_softcap=cap)
    _close(loss.detach(), want.detach(), TOL)
    gx, = torch.autograd.grad(loss, x)
    wx, ww = torch.autograd.grad(want, (x, w))
    _close(gx, wx, TOL)
    _close(head.store.full_gradient("proj.weight"), ww, TOL)


def _model(mesh=None, vocab_parallel=False, tie=False):
    attn = MultiheadSelfAttentionConfig(n_heads=4, head_dim=16)
    cfg = DefaultTransformerConfig(vocab_size=64, d_model=64, hidden_size=96, num_layers=2, ce_chunk_rows=16, tie_embeddings=tie,
                                   layer=DefaultTransformerLayerConfig(attention=attn), lm_head=LMHeadConfig(vocab_parallel=vocab_parallel))
    return cfg.build(seed=0, mesh_resource=mesh or MeshResource.FSDP(1), device=torch.device("cpu"))


@pytest.mark.parametrize("tie", [False, True])
def test_model_scores_its_labels_and_learns_from_a_teacher(tie, tmp_path):
    from olmax_b200.optim import AdamWConfig, ConstantSchedule
    from olmax_b200.train import Trainer

    student, teacher = _model(tie=tie), _model()
    ids = torch.randint(0, 64, (2, 12), generator=torch.Generator().manual_seed(5))
    labels = torch.roll(ids, -1, 1)
    labels[:, -1] = -100
    with torch.no_grad():
        scores = student.token_log_probs(ids, labels)
        loss, _ = student(ids, labels)
        best = teacher.token_log_probs(ids, top_k=8)
    assert scores.log_probs.shape == (2, 12) and best.top_ids.shape == (2, 12, 8) and best.log_probs is None
    assert torch.allclose(-scores.log_probs.sum() / 22, loss, atol=1e-5)
    logits = student(ids)
    want = F.distillation_loss(logits.detach(), best.top_ids, best.top_log_probs)
    got = student.distillation_loss(ids, best.top_ids, best.top_log_probs)
    assert torch.allclose(got.detach(), want, atol=1e-5)
    # the trainer's default loss of a micro-batch (ids, teacher ids, teacher log probabilities)
    student.store.zero_grad()
    trainer = Trainer(work_dir=tmp_path, save_folder=tmp_path, optim=AdamWConfig(lr=ConstantSchedule(1e-2)))
    trainer.setup(student, 1)
    before = student.store.master.clone()
    loss = trainer.train_batch([(ids, best.top_ids, best.top_log_probs)])
    assert torch.allclose(loss, want, atol=1e-5) and not torch.equal(before, student.store.master)
    with pytest.raises(ValueError):
        student.distillation_loss(ids[:, :5], best.top_ids, best.top_log_probs)


def _sharded(rank, world, axis):
    mesh = MeshResource.FSDP(world) if axis == "fsdp" else MeshResource.FSDP_with_TP(world, world)
    model, whole = _model(mesh), None
    ids = torch.randint(0, 64, (4, 16), generator=torch.Generator().manual_seed(7))
    t = torch.randn(4, 16, 64, generator=torch.Generator().manual_seed(8)).log_softmax(-1).topk(6, dim=-1)
    mine = ids.chunk(world)[rank] if axis == "fsdp" else ids
    teach = [x.chunk(world)[rank] if axis == "fsdp" else x for x in (t.indices, t.values)]
    model.store.set_grad_scale(1.0 / world)
    loss = model.distillation_loss(mine, *teach)
    out = model.token_log_probs(mine, mine)
    (loss + out.log_probs.mean() + out.entropy.mean()).backward()
    model.store.finish_backward()
    model.store.reduce_replicated_grads()
    return loss.item(), model.store.full_gradient("lm_head.proj.weight"), model.store.full_gradient("layers.0.attention.q_proj.weight")


def _check_sharded(axis):
    import torch.distributed as dist

    rank, world = dist.get_rank(), dist.get_world_size()
    from olmax_b200.parallel import set_mesh

    loss, *grads = _sharded(rank, world, axis)
    total = torch.tensor(loss)
    dist.all_reduce(total)
    set_mesh(None)
    model = _model(MeshResource.DDP(world))
    ids = torch.randint(0, 64, (4, 16), generator=torch.Generator().manual_seed(7))
    t = torch.randn(4, 16, 64, generator=torch.Generator().manual_seed(8)).log_softmax(-1).topk(6, dim=-1)
    want = model.distillation_loss(ids, t.indices, t.values)
    out = model.token_log_probs(ids, ids)
    (want + out.log_probs.mean() + out.entropy.mean()).backward()
    model.store.finish_backward()
    assert abs(total.item() / world - want.item()) < 1e-5
    for g, name in zip(grads, ("lm_head.proj.weight", "layers.0.attention.q_proj.weight")):
        assert torch.allclose(g, model.store.full_gradient(name), atol=1e-5), (name, float((g - model.store.full_gradient(name)).abs().max()))


@pytest.mark.parametrize("axis", ["fsdp", "tp"])
def test_two_ranks_give_what_one_gives(axis):
    run_distributed_test(_check_sharded, world_size=2, func_args=(axis,))


def _check_vocab_parallel():
    model = _model(MeshResource.FSDP_with_TP(2, 2), vocab_parallel=True)
    ids = torch.zeros((2, 8), dtype=torch.int64)
    with pytest.raises(OLMaxConfigurationError):
        model.token_log_probs(ids, ids)
    with pytest.raises(OLMaxConfigurationError):
        model.distillation_loss(ids, torch.zeros((2, 8, 3), dtype=torch.int64), torch.zeros(2, 8, 3))


def test_a_vocabulary_parallel_head_refuses():
    run_distributed_test(_check_vocab_parallel, world_size=2)


@pytest.mark.parametrize("bad", [
    dict(temperature=0.0), dict(temperature=1e-7), dict(temperature=1e7), dict(logit_softcap=300.0), dict(logit_softcap=1e-4), dict(temperature=-1.0), dict(temperature=math.nan), dict(temperature=math.inf),
    dict(logit_softcap=-1.0), dict(logit_softcap=math.inf), dict(top_k=-1), dict(top_k=11), dict(ids=torch.zeros(5, dtype=torch.int64)),
    dict(ids=torch.zeros(4)), dict(ignore_index=2 ** 32 + 5),
])
def test_refused_scores(bad):
    with pytest.raises(ValueError):
        F.token_log_probs(_rows(4, 10), **bad)


def test_refused_top_classes_beyond_the_limit_and_types():
    with pytest.raises(ValueError):
        F.token_log_probs(_rows(1, 1000), top_k=K.TOP_K_MAX + 1)
    with pytest.raises(ValueError):
        F.token_log_probs(torch.zeros(3, 0))
    with pytest.raises(ValueError):
        F.token_log_probs(torch.zeros(()))
    with pytest.raises(K.KernelError):
        F.token_log_probs(torch.zeros(3, 4, dtype=torch.float16))
    with pytest.raises(K.KernelError):
        F.distillation_loss(torch.zeros(3, 4, dtype=torch.int32), torch.zeros(3, 1, dtype=torch.int64), torch.zeros(3, 1))


@pytest.mark.parametrize("bad", [
    dict(tail="drop"), dict(reduction="max"), dict(temperature=0.0), dict(teacher_ids=torch.zeros(4, 3)),
    dict(teacher_ids=torch.zeros(4, 2, dtype=torch.int64)), dict(teacher_log_probs=torch.zeros(4, 3, dtype=torch.int64)),
    dict(teacher_ids=torch.zeros(3, 3, dtype=torch.int64), teacher_log_probs=torch.zeros(3, 3)),
    dict(teacher_ids=torch.zeros(4, 0, dtype=torch.int64), teacher_log_probs=torch.zeros(4, 0)),
    dict(teacher_ids=torch.zeros(4, 129, dtype=torch.int64), teacher_log_probs=torch.zeros(4, 129)),
])
def test_refused_distillation(bad):
    args = dict(teacher_ids=torch.zeros(4, 3, dtype=torch.int64), teacher_log_probs=torch.zeros(4, 3))
    args.update(bad)
    with pytest.raises(ValueError):
        F.distillation_loss(_rows(4, 200), **args)
    if "reduction" not in bad:
        with pytest.raises(ValueError):
            _head(V=200).distillation_loss(torch.zeros(4, 16), **args)


def test_empty_batches():
    out = F.token_log_probs(torch.zeros(0, 10), torch.zeros(0, dtype=torch.int64), top_k=3)
    assert out.log_probs.shape == (0,) and out.top_ids.shape == (0, 3)
    z = torch.zeros(0, 10, requires_grad=True)
    loss = F.distillation_loss(z, torch.zeros((0, 2), dtype=torch.int64), torch.zeros(0, 2))
    assert float(loss) == 0 and torch.autograd.grad(loss, z)[0].shape == (0, 10)


def test_second_derivatives_are_refused():
    z = _rows(3, 9).requires_grad_(True)
    out = F.token_log_probs(z, torch.zeros(3, dtype=torch.int64))
    with pytest.raises(RuntimeError):
        torch.autograd.grad(out.log_probs.sum(), z, create_graph=True)
    loss = F.distillation_loss(z, torch.zeros((3, 1), dtype=torch.int64), torch.zeros(3, 1))
    with pytest.raises(RuntimeError):
        torch.autograd.grad(loss, z, create_graph=True)
