"""The kernels over the LM head's distribution against the definitions in 64 bits."""

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

# Error of an fp32 evaluation, in units of 2^-24.  The scaled logit y and its distance to the maximum are rounded a few times: 8 max |y|.  An
# exponential is off by about 4 and its argument's rounding.  A thread adds up to V / 64 terms one by one (a block has no fewer than 64
# threads) and the threads' sums are joined in a tree: V / 64 + 64.  A tanh is off by 2e-7, cap / T times that in y.


def _eps(V, y_max, cap=0.0, temperature=1.0):
    return 2.0 ** -24 * (V / 64 + 64 + 8 * y_max) + (4e-7 * cap / temperature if cap else 0.0)


def _close(got, want, tol, what=""):
    got, want = got.double(), want.double()
    assert got.shape == want.shape and torch.equal(got.isnan(), want.isnan()), what
    off = torch.where((got == want) | got.isnan(), 0.0, (got - want).abs())
    assert torch.all(off <= tol), (what, float(off.max()), float((off - tol).max()))


def _logits(rows, V, dtype=torch.float32, seed=0, spread=3.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(rows, V, generator=g, device=DEV) * spread).to(dtype)


def _ids(rows, V, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed + 100)
    ids = torch.randint(0, V, (rows,), generator=g, device=DEV)
    if rows > 3:
        ids[1], ids[2], ids[3] = -100, V, -1   # none of these is scored
    return ids


def _check_scores(z, ids, k, temperature=1.0, cap=0.0):
    out = F.token_log_probs(z, ids, top_k=k, temperature=temperature, logit_softcap=cap)
    z2, i2 = z.reshape(-1, z.shape[-1]), ids.reshape(-1)
    lp, ent, top, top_ids = scores_64(z2, i2, k, temperature, cap)
    y = z2.double()[z2.isfinite()]
    y_max = float(y.abs().max()) / temperature if y.numel() else 0.0
    y_max = min(y_max, cap / temperature) if cap else y_max
    e = _eps(z.shape[-1], y_max, cap, temperature)
    _close(out.log_probs.reshape(-1), lp, e * (1 + 1), "log p")
    _close(out.entropy.reshape(-1), ent, e * (2 + ent.nan_to_num(0).abs()), "entropy")
    if k:
        assert torch.equal(out.top_ids.reshape(-1, k), top_ids)
        _close(out.top_log_probs.reshape(-1, k), top, e * 2, "top log p")
    return out


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,V,k", [(1, 1, 1), (3, 2, 2), (2, 7, 3), (5, 127, 127), (4, 128, 128), (130, 1000, 5), (3, 4097, 64), (1, 50257, 128),
                                      (33, 32000, 20), (7, 100352, 0), (300, 8192, 1), (2, 256000, 128)])
def test_scores(rows, V, k, dtype):
    _check_scores(_logits(rows, V, dtype), _ids(rows, V), k)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("temperature,cap", [(0.5, 0.0), (1.0, 30.0), (2.0, 5.0), (1.0, 256.0), (0.01, 1.0), (1e-6, 0.0), (1e6, 0.0), (1e-6, 30.0), (1.0, 1e-3)])
def test_scores_scaled(temperature, cap, dtype):
    _check_scores(_logits(40, 5003, dtype, spread=8.0), _ids(40, 5003), 16, temperature, cap)


def test_row_starts_strides_and_leading_dimensions():
    big = _logits(64, 1024)
    ids = _ids(64, 1001)
    for first in range(4):                                        # every 4-byte offset of a 16-byte line
        _check_scores(big[:, first : first + 1001], ids, 9)
    _check_scores(big[::2, 3:1004], ids[::2], 9)
    half = _logits(64, 1024, torch.bfloat16)
    for first in range(8):
        _check_scores(half[:, first : first + 999], ids, 9)
    _check_scores(big.view(4, 16, 1024), _ids(64, 1024).view(4, 16), 9)
    _check_scores(big.view(4, 16, 1024).transpose(0, 1), _ids(64, 1024).view(16, 4), 9)     # rows that are no single stride apart
    _check_scores(big[:1].expand(5, 1024), _ids(5, 1024), 9)                                # a broadcast row
    _check_scores(_logits(1000, 70).t(), _ids(70, 1000), 9)                                 # classes that are not contiguous


def test_ties_go_to_the_lowest_class():
    V = 20011
    z = _logits(6, V)
    z[0] = 0.25                                                   # all equal
    z[1] = torch.arange(V, device=DEV) // 300 % 5                 # long runs of few values
    z[2] = torch.arange(V, device=DEV, dtype=torch.float32)       # ascending
    z[3] = -torch.arange(V, device=DEV, dtype=torch.float32)      # descending
    z[4, ::2], z[4, 1::2] = 0.0, -0.0
    z[5] = z[5].to(torch.bfloat16).float()
    for k in (1, 37, 128):
        for dtype in (torch.float32, torch.bfloat16):
            zz = z.to(dtype)
            out = F.token_log_probs(zz, top_k=k)
            want = (zz.float() + 0.0).sort(dim=-1, descending=True, stable=True).indices[:, :k]
            assert torch.equal(out.top_ids, want)


def test_masked_classes_and_rows():
    for V in (12, 4096, 30001):
        for dtype in (torch.float32, torch.bfloat16):
            z = _logits(8, V, dtype)
            z[0, 3:] = -math.inf
            z[1] = -math.inf
            z[2, ::2] = torch.finfo(dtype).min
            z[3, : V - 1] = -math.inf
            z[4, : V // 2] = -math.inf
            z[5, 1] = math.nan
            z[6] = torch.finfo(dtype).min
            ids = torch.tensor([0, 4, 1, V - 1, V - 1, 2, 3, 0], device=DEV)
            # the lowest values of the type overflow the sums that the tolerance is made of: their rows are looked at one by one
            _check_scores(z[[0, 1, 3, 4, 7]], ids[[0, 1, 3, 4, 7]], min(V, 9))
            out = F.token_log_probs(z, ids, top_k=min(V, 128))
            assert out.log_probs[1] == -math.inf and out.entropy[1] == 0 and out.top_ids[1].tolist() == list(range(min(V, 128)))
            assert out.log_probs[5].isnan() and out.entropy[5].isnan() and out.top_ids[5, 0] == 1
            lp, ent, top, top_ids = scores_64(z[[2]], ids[[2]], min(V, 9))
            _close(out.log_probs[2:3], lp, _eps(V, 20.0) * 2)
            _close(out.entropy[2:3], ent, _eps(V, 20.0) * (2 + ent))
            assert torch.equal(out.top_ids[2:3, : min(V, 9)], top_ids)
            _close(out.entropy[6:7], torch.tensor([math.log(V)], device=DEV), _eps(V, 20.0) * (2 + math.log(V)))
            # gradients: none where there is no class, none for a masked class, all finite but for the NaN row
            zz = z.clone().requires_grad_(True)
            out = F.token_log_probs(zz, ids)
            g, = torch.autograd.grad(out.log_probs[:5].sum() + out.entropy.sum(), zz)
            assert torch.all(g[1] == 0) and torch.all(g[0, 3:] == 0) and torch.all(g[[0, 1, 2, 3, 4, 6, 7]].isfinite())
            assert torch.all(g[5].isnan())


def _check_score_gradients(z, ids, temperature=1.0, cap=0.0, dtype_tol=None):
    rows, V = z.shape
    g = torch.Generator(device=DEV).manual_seed(9)
    gl, ge = torch.randn(rows, generator=g, device=DEV), torch.randn(rows, generator=g, device=DEV)
    leaf = z.detach().requires_grad_(True)
    out = F.token_log_probs(leaf, ids, temperature=temperature, logit_softcap=cap)
    for a, b in ((gl, ge), (gl, None), (None, ge)):
        outs = [o for o, u in ((out.log_probs, a), (out.entropy, b)) if u is not None]
        got, = torch.autograd.grad(outs, leaf, [u for u in (a, b) if u is not None], retain_graph=True)
        zero = torch.zeros(rows, device=DEV)
        want, size = score_gradients_64(z, ids, zero if a is None else a, zero if b is None else b, temperature, cap)
        y_max = min(float(z.float().abs().max()), cap or math.inf) / temperature
        e = _eps(V, y_max, cap, temperature) * 4 + (8e-6 if cap else 0.0)
        # (1 - tanh^2 of a capped logit is off by a few roundings of 1)
        tol = e * size + 1e-30 + (2.0 ** -8 * want.abs() if z.dtype == torch.bfloat16 else 0)
        assert got.dtype == z.dtype
        _close(got, want, tol)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,V,temperature,cap", [(1, 1, 1.0, 0.0), (3, 2, 1.0, 0.0), (9, 1000, 0.7, 0.0), (5, 4099, 1.0, 30.0),
                                                    (70, 50257, 1.0, 0.0), (4, 100352, 2.0, 5.0)])
def test_score_gradients(rows, V, temperature, cap, dtype):
    _check_score_gradients(_logits(rows, V, dtype), _ids(rows, V), temperature, cap)


def test_score_gradients_of_views_and_broadcast_rows():
    big = _logits(20, 1030)
    ids = _ids(20, 1001)
    for z in (big[:, 1:1002], big[:, 4:1005], big.to(torch.bfloat16)[:, 3:1004]):
        _check_score_gradients(z, ids)
    row = _logits(1, 777).requires_grad_(True)
    out = F.token_log_probs(row.expand(6, 777), _ids(6, 777))
    g, = torch.autograd.grad(out.log_probs.sum(), row)             # the gradient of a broadcast input is the sum over its rows
    each = [torch.autograd.grad(F.token_log_probs(row, i.view(1)).log_probs.sum(), row)[0] for i in _ids(6, 777)]
    _close(g, sum(e.double() for e in each), 6 * _eps(777, 20.0))


# ------------------------------------------------------------------------------------------------------------ distillation
def _teacher(rows, V, k, seed=5, temperature=1.0):
    t = torch.log_softmax(_logits(rows, V, seed=seed).double() / temperature, -1).topk(k, dim=-1)
    return t.indices, t.values.float()


def _check_distillation(z, ids, t, tail, reduction="mean", temperature=1.0, cap=0.0, up=None):
    rows, V = z.shape
    leaf = z.detach().requires_grad_(True)
    loss = F.distillation_loss(leaf, ids, t, tail=tail, reduction=reduction, temperature=temperature, logit_softcap=cap)
    want, grads = distillation_64(z, ids, t, tail, reduction, temperature, cap)
    y_max = min(float(z.float().abs()[z.isfinite()].max()), cap or math.inf) / temperature
    e = _eps(V, y_max, cap, temperature)
    # a loss is a sum over masses of at most 1 (2 where a bad teacher leaves nothing) of differences of logarithms
    _close(loss.detach(), want, 4 * e * (rows if reduction == "sum" else 1) + 2.0 ** -23 * want.abs())
    if up is None:
        up = torch.ones((), device=DEV) if reduction != "none" else torch.linspace(-1, 2, rows, device=DEV)
    got, = torch.autograd.grad(loss, leaf, up)
    scale = up.double() if reduction != "none" else up.double()[:, None]
    n = max(1, int(((ids >= 0) & (ids < V)).any(1).sum())) if reduction == "mean" else 1
    # a gradient's terms are at most total * p + q + rest * (share of the rest) with masses of at most 1; each is relatively exact
    p = torch.softmax(_y(z, temperature, cap), -1)
    q = torch.zeros(rows, V + 1, dtype=torch.float64, device=DEV)
    q.scatter_(1, ids.long().where((ids >= 0) & (ids < V), V), 1.0)
    size = 2 * p + q[:, :V] + _rest_share(z, ids, temperature, cap)
    tol = (4 * e + (8e-6 if cap else 0)) * size * scale.abs() / n / temperature + 1e-30
    want_g = grads * scale
    if z.dtype == torch.bfloat16:
        tol = tol + 2.0 ** -8 * want_g.abs()
    assert got.dtype == z.dtype
    _close(got, want_g, tol, "gradient")


def _y(z, temperature, cap):
    return (cap * torch.tanh(z.double() / cap) if cap else z.double()) / temperature


def _rest_share(z, ids, temperature, cap):
    named = torch.zeros(z.shape[0], z.shape[1] + 1, dtype=torch.bool, device=DEV)
    named.scatter_(1, ids.long().where((ids >= 0) & (ids < z.shape[1]), z.shape[1]), True)
    return torch.softmax(_y(z, temperature, cap).masked_fill(named[:, :-1], -math.inf), -1).nan_to_num(0.0)


@pytest.mark.parametrize("tail", ["rest", "renormalize"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,V,k", [(1, 1, 1), (2, 5, 5), (3, 40, 1), (9, 1001, 7), (4, 50257, 64), (130, 3000, 128), (3, 256000, 128)])
def test_distillation(rows, V, k, dtype, tail):
    _check_distillation(_logits(rows, V, dtype), *_teacher(rows, V, k), tail)


@pytest.mark.parametrize("tail", ["rest", "renormalize"])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("temperature,cap", [(1.0, 0.0), (2.0, 30.0)])
def test_distillation_reductions_padding_and_repeated_classes(temperature, cap, reduction, tail):
    rows, V, k = 12, 2003, 20
    ids, t = _teacher(rows, V, k, temperature=temperature)
    ids[0] = -1                         # no teacher
    ids[1, 3:] = -1                     # a short list
    ids[2, ::2] = V + 5                 # padding between the pairs
    ids[3, 4] = ids[3, 1]               # repeated: the first counts
    ids[4, 1:] = ids[4, :1]
    t[5, 6:] = -math.inf
    ids[6] = -100
    z = _logits(rows, V)
    z[7, 1000:] = -math.inf
    t[7, (ids[7] >= 1000)] = -math.inf  # masked classes that the teacher does not like either
    _check_distillation(z, ids, t, tail, reduction, temperature, cap)
    _check_distillation(z, ids.int(), t, tail, reduction, temperature, cap)
    _check_distillation(z.to(torch.bfloat16), ids, t, tail, reduction, temperature, cap)
    if reduction != "none":
        _check_distillation(z, ids, t, tail, reduction, temperature, cap, up=torch.tensor(-0.375, device=DEV))


def test_distillation_views_and_borders():
    big = _logits(11, 1030)
    ids, t = _teacher(11, 1001, 9)
    for z in (big[:, 1:1002], big[:, 4:1005], big.to(torch.bfloat16)[:, 3:1004]):
        _check_distillation(z, ids, t, "rest")
    wide_ids, wide_t = torch.full((11, 15), -1, device=DEV), torch.zeros(11, 15, device=DEV)
    wide_ids[:, 3:12], wide_t[:, 3:12] = ids, t
    _check_distillation(big[:, :1001], wide_ids[:, 3:12], wide_t[:, 3:12], "rest")     # teachers of another row stride
    # a student far more certain than its teacher: what it leaves to the rest is below a rounding of 1
    z = _logits(3, 1001)
    z[torch.arange(3), ids[:3, 0]] += 200.0
    _check_distillation(z, ids[:3], t[:3], "rest")
    # the masses of all classes, which leave nothing but a rounding
    _check_distillation(_logits(4, 100), *_teacher(4, 100, 100), "rest")
    # the student's own distribution
    z = _logits(5, 3001)
    own = F.token_log_probs(z, top_k=50)
    leaf = z.requires_grad_(True)
    loss = F.distillation_loss(leaf, own.top_ids, own.top_log_probs)
    g, = torch.autograd.grad(loss, leaf)
    assert abs(float(loss.detach())) < 4 * _eps(3001, 20.0) and float(g.abs().max()) < 4 * _eps(3001, 20.0)


def test_distillation_of_empty_and_masked_rows():
    z = _logits(6, 500)
    z[0] = -math.inf
    z[1, 2:] = -math.inf
    z[2, 5] = math.nan
    z[3, 5] = math.nan
    ids = torch.tensor([[0, 1], [0, 1], [3, 4], [-1, -1], [3, 4], [7, 8]], device=DEV)
    t = torch.log(torch.tensor([[0.5, 0.4]], device=DEV)).expand(6, 2).clone()
    for tail in ("rest", "renormalize"):
        leaf = z.clone().requires_grad_(True)
        loss = F.distillation_loss(leaf, ids, t, tail=tail, reduction="none")
        g, = torch.autograd.grad(loss, leaf, torch.ones(6, device=DEV))
        want, grads = distillation_64(z[[1, 4, 5]], ids[[1, 4, 5]], t[[1, 4, 5]], tail, "none")
        _close(loss.detach()[[1, 4, 5]], want, 4 * _eps(500, 20.0))
        _close(g[[1, 4, 5]], grads, 4 * _eps(500, 20.0))
        assert loss[0] == math.inf and torch.all(g[0] == 0)           # no class to give the teacher's mass to
        assert loss[2].isnan() and torch.all(g[2].isnan())
        assert loss[3] == 0 and torch.all(g[3] == 0)                  # no teacher: whatever the logits are
    none = F.distillation_loss(_logits(4, 30), torch.full((4, 3), -1, device=DEV), torch.zeros(4, 3, device=DEV))
    assert float(none) == 0


# ------------------------------------------------------------------------------------------------------- how they are called
def test_long_offsets():
    """Rows whose distance passes 32 bits."""
    rows, V, ld = 9, 1001, 2 ** 28 + 3
    buf = torch.empty(rows * ld, dtype=torch.bfloat16, device=DEV)
    z = buf.as_strided((rows, V), (ld, 1))
    z.copy_(_logits(rows, V, torch.bfloat16))
    _check_scores(z, _ids(rows, V), 5)
    _check_score_gradients(z, _ids(rows, V))
    _check_distillation(z, *_teacher(rows, V, 5), "rest")


def _pass(z, ids, t_ids, t):
    leaf = z.detach().requires_grad_(True)
    out = F.token_log_probs(leaf, ids, top_k=8)
    kd = F.distillation_loss(leaf, t_ids, t)
    g1, = torch.autograd.grad((out.log_probs.sum() + 0.1 * out.entropy.sum()), leaf)
    g2, = torch.autograd.grad(kd, leaf)
    return [x.detach() for x in (*out, kd, g1, g2)]


def test_streams_repeats_and_captured_graphs():
    sets = []
    for seed, rows in ((0, 6), (1, 300)):
        sets.append((_logits(rows, 9001, seed=seed), _ids(rows, 9001, seed), *_teacher(rows, 9001, 12, seed=seed + 7)))
    eager = [_pass(*s) for s in sets]
    for s, want in zip(sets, eager):
        for a, b in zip(_pass(*s), want):
            assert torch.equal(a, b)                                  # no order of blocks or atomics shows
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = [_pass(*s) for s in sets]
    here = [_pass(*s) for s in sets]                                  # beside the other stream's
    torch.cuda.synchronize()
    graphs = []
    for s in sets:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphs.append((graph, _pass(*s)))
    for s in sets:                                                    # other inputs, then the first ones again
        s[0].mul_(0.5)
    for graph, _ in graphs:
        graph.replay()
    changed = [_pass(*s) for s in sets]
    torch.cuda.synchronize()
    for got, want in ((on_side, eager), (here, eager), ([o for _, o in graphs], changed)):
        for a, b in zip(got, want):
            assert all(torch.equal(x, y) for x, y in zip(a, b))
    for s in sets:
        s[0].mul_(2.0)
    for graph, _ in reversed(graphs):
        graph.replay()
    torch.cuda.synchronize()
    for (_, a), b in zip(graphs, eager):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def _bf16_head(V, d, cap=None):
    return build_module(lambda: LMHead(d, V, logit_softcap=cap, init_std=0.1), mesh_resource=MeshResource.FSDP(1), device=torch.device(DEV))


@pytest.mark.parametrize("rows,chunk,cap", [(1, 2048, None), (13, 2048, None), (100, 40, 30.0), (75, 16, None), (64, 64, None)])
def test_head_scores_distillation_and_their_gradients(rows, chunk, cap):
    V, d = 1000, 256
    head = _bf16_head(V, d, cap)
    w = head.weight.full()
    x = torch.randn(rows, d, generator=torch.Generator(device=DEV).manual_seed(3), device=DEV).to(torch.bfloat16)
    ids = _ids(rows, V)
    # the GEMM's fp32 sums of 256 exact products are off by less than 256 * 2^-24 of the sum of the absolute values, about 15 here
    gemm = 256 * 2.0 ** -24 * float((x.double().abs() @ w.double().abs().t()).max())
    z = x.double() @ w.double().t()
    leaf = x.clone().requires_grad_(True)
    out = head.token_log_probs(leaf, ids, top_k=6, temperature=0.9, chunk_rows=chunk)
    lp, ent, top, _ = scores_64(z, ids, 6, 0.9, cap or 0.0)
    e = _eps(V, 20.0, cap or 0.0, 0.9) + 2 * gemm
    _close(out.log_probs.detach(), lp, 2 * e)
    _close(out.entropy.detach(), ent, (2 + ent) * e)
    _close(out.top_log_probs, top, 2 * e)

    def compare(gx, dz):
        """dz is rounded to bf16 (half a step, 2^-8 relative) before the products, dx after them; all sums are fp32."""
        rounding = 2.0 ** -8 + 2.0 ** -12
        want_x, size_x = dz @ w.double(), dz.abs() @ w.double().abs()
        _close(gx, want_x, rounding * size_x + 2.0 ** -8 * want_x.abs() + e * size_x + 1e-12)
        want_w, size_w = dz.t() @ x.double(), dz.abs().t() @ x.double().abs()
        _close(head.store.full_gradient("proj.weight"), want_w, (rounding + e) * size_w + 1e-12)
        head.store.zero_grad()

    gl, ge = torch.linspace(-1, 1, rows, device=DEV), torch.linspace(0.2, 0.1, rows, device=DEV)
    gx, = torch.autograd.grad((out.log_probs, out.entropy), leaf, (gl, ge))
    dz, _ = score_gradients_64(z, ids, gl, ge, 0.9, cap or 0.0)
    compare(gx, dz)
    t_ids, t = _teacher(rows, V, 10, temperature=0.9)
    t_ids[rows // 2] = -1
    loss = head.distillation_loss(leaf, t_ids, t, weight=0.5, temperature=0.9, chunk_rows=chunk)
    want, dz = distillation_64(z, t_ids, t, "rest", "mean", 0.9, cap or 0.0)
    _close(loss.detach(), 0.5 * want, 4 * e)
    gx, = torch.autograd.grad(loss, leaf)
    compare(gx, 0.5 * dz)
    with torch.no_grad():
        again = head.distillation_loss(x, t_ids, t, weight=0.5, temperature=0.9, chunk_rows=chunk)
    assert torch.equal(again, loss.detach()) and float(head.store.grad.abs().max()) == 0


def test_a_teacher_scores_and_a_student_learns_from_it():
    """The operators one after another, as a distillation step uses them."""
    from olmax_b200.models import DefaultTransformerConfig, DefaultTransformerLayerConfig
    from olmax_b200.nn import MultiheadSelfAttentionConfig

    def model(seed, layers):
        cfg = DefaultTransformerConfig(vocab_size=2048, d_model=512, hidden_size=1024, num_layers=layers, ce_chunk_rows=96,
                                       layer=DefaultTransformerLayerConfig(attention=MultiheadSelfAttentionConfig(n_heads=4, head_dim=128)))
        return cfg.build(seed=seed, mesh_resource=MeshResource.FSDP(1), device=torch.device(DEV))

    teacher, student = model(1, 2), model(2, 1)
    ids = torch.randint(0, 2048, (2, 128), generator=torch.Generator(device=DEV).manual_seed(1), device=DEV)
    with torch.no_grad():
        best = teacher.token_log_probs(ids, top_k=32)
        logits = student(ids)
    loss = student.distillation_loss(ids, best.top_ids, best.top_log_probs)
    loss.backward()
    student.store.finish_backward()
    fused = student.store.full_gradient("lm_head.proj.weight").clone()
    # the same loss from the model's logits, which are rounded to bf16 (half a step, 2^-8 relative); the gradient of a loss with
    # respect to a row's logits has an absolute sum of at most 2
    plain = F.distillation_loss(logits, best.top_ids, best.top_log_probs)
    assert abs(float(loss.detach()) - float(plain)) <= 2 * 2.0 ** -8 * float(logits.abs().max())
    assert float(fused.abs().max()) > 0 and torch.all(fused.isfinite())
    labels = torch.roll(ids, -1, 1)
    labels[:, -1] = -100
    with torch.no_grad():
        scores = student.token_log_probs(ids, labels, top_k=3)
        ce, _ = student(ids, labels)
        logits = student(ids)
    counted = labels != -100
    assert abs(float(-scores.log_probs[counted].mean()) - float(ce)) <= 1e-4 * float(ce)
    # (rounding keeps the order: the largest fp32 logit is among the largest rounded ones)
    assert torch.equal(logits.gather(-1, scores.top_ids[..., :1])[..., 0], logits.amax(-1))


def test_refusals_reach_no_kernel():
    z = _logits(4, 200)
    from olmax_b200.ops import kernels as K

    before = K.launch_count()
    for bad in (dict(top_k=129), dict(top_k=-1), dict(temperature=0.0), dict(ids=torch.zeros(4, dtype=torch.int64))):   # ids on the CPU
        with pytest.raises(ValueError):
            F.token_log_probs(z, **bad)
    with pytest.raises(K.KernelError):
        F.token_log_probs(z.half())
    with pytest.raises(ValueError):
        F.distillation_loss(z, torch.zeros(4, 3, dtype=torch.int64), torch.zeros(4, 3))
    with pytest.raises(K.KernelError):
        _bf16_head(64, 64).token_log_probs(torch.zeros(4, 64, device=DEV))
    out = F.token_log_probs(z[:0], torch.zeros(0, dtype=torch.int64, device=DEV), top_k=2)
    assert out.top_ids.shape == (0, 2) and K.launch_count() == before


def test_infinite_logits():
    """+inf has no distribution (NaN, as the formula gives it), but an order."""
    for V in (40, 9000):
        z = _logits(3, V)
        z[0, 5] = math.inf
        z[1, V - 1] = z[1, 7] = math.inf
        z[1, 20] = math.nan
        out = F.token_log_probs(z, torch.tensor([5, 7, 3], device=DEV), top_k=3)
        assert out.log_probs[:2].isnan().all() and out.entropy[:2].isnan().all() and out.log_probs[2].isfinite()
        best = z.clone()
        best[0, 5] = -math.inf
        assert out.top_ids[0].tolist() == [5, *best[0].topk(2).indices.tolist()]
        assert out.top_ids[1].tolist() == [20, 7, V - 1]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_top_classes_of_long_rows_in_bad_orders(dtype):
    """Rows that keep giving new largest logits, that keep repeating them, or whose largest ones all fall to the same few threads."""
    V = 260011
    i = torch.arange(V, device=DEV)
    z = _logits(7, V)
    z[0] = i                                                        # ascending (in steps of a rounding for bf16)
    z[1] = 7.0
    z[2] = (i // 50000).float()                                     # long runs, ascending
    z[3] = torch.where(i % 2048 < 200, 50.0 + i / V, z[3])          # the largest in the same places of every stretch
    z[4] = (i % 3).float()
    z[5] = torch.where(i > V - 300, 1.0, -1.0)
    z[6] = torch.where(i % 8192 < 8, (i // 8192).float(), -3.0)     # few threads, ascending
    z = z.to(dtype)
    for part in (z, z[:, 1:], z[:1]):                               # (one row: shared by a cluster)
        for k in (1, 64, 128):
            out = F.token_log_probs(part, top_k=k)
            want = part.sort(dim=-1, descending=True, stable=True).indices[:, :k]
            assert torch.equal(out.top_ids, want)


@pytest.mark.parametrize("rows,V,d,cap,temperature", [(1, 8, 64, None, 1.0), (16411, 264, 64, None, 1.0), (7, 264, 128, None, 1.0), (300, 1000, 256, 30.0, 0.7), (2048, 5000, 512, None, 1.0),
                                                      (1100, 20008, 72, None, 2.0), (328, 50304, 128, 30.0, 1.0)])
def test_head_scores_out_of_the_epilogue(rows, V, d, cap, temperature):
    """Tiles of both geometries, ragged in rows, classes and contraction, against the same head's fp32 logits."""
    head = _bf16_head(V, d, cap)
    w = head.weight.full()
    x = torch.randn(rows, d, generator=torch.Generator(device=DEV).manual_seed(3), device=DEV).to(torch.bfloat16)
    ids = _ids(rows, V)
    z = x.double() @ w.double().t()
    gemm = d * 2.0 ** -24 * float((x.double().abs() @ w.double().abs().t()).max())
    y_max = min(float(z.abs().max()), cap or math.inf) / temperature
    lp, ent, _, _ = scores_64(z, ids, 1, temperature, cap or 0.0)
    e = _eps(V, y_max, cap or 0.0, temperature) + 2 * gemm / temperature
    with torch.no_grad():
        out = head.token_log_probs(x, ids, temperature=temperature)
        none = head.token_log_probs(x, temperature=temperature)
        three = head.token_log_probs(x.view(1, rows, d), ids.view(1, rows), temperature=temperature)
    _close(out.log_probs, lp, 2 * e)
    _close(out.entropy, ent, (2 + ent) * e)
    assert none.log_probs is None and torch.equal(none.entropy, out.entropy) and torch.equal(three.log_probs[0], out.log_probs)
    from olmax_b200.ops import _lib

    _lib.check_status()


def test_head_scores_of_weight_shards():
    """B in row blocks a stride apart, as a gathered unit is laid out."""
    from olmax_b200.ops import kernels as K

    M, N, Kd, R, rows = 512, 2400, 256, 4, 509
    g = torch.Generator(device=DEV).manual_seed(5)
    a = torch.randn(M, Kd, generator=g, device=DEV).to(torch.bfloat16)
    stride = (N // R) * Kd + 1024
    buf = torch.randn(R * stride, generator=g, device=DEV).to(torch.bfloat16)
    b = torch.cat([buf[r * stride : r * stride + (N // R) * Kd].view(N // R, Kd) for r in range(R)])
    ids = _ids(rows, N)
    out = [[torch.full((rows + 1,), 7.0, device=DEV) for _ in range(2)] for _ in range(2)]
    K.gemm_scores(a, b, ids, out[0][0][:rows], out[0][1][:rows], None, M, N, Kd, rows=rows)
    K.gemm_scores(a, buf[: (N // R) * Kd].view(N // R, Kd), ids, out[1][0][:rows], out[1][1][:rows], None, M, N, Kd, rows=rows, N_s=N // R,
                  b_shard_stride=stride)
    z = a.double() @ b.double().t()
    lp, ent, _, _ = scores_64(z[:rows], ids, 1)
    gemm = Kd * 2.0 ** -24 * float((a.double().abs() @ b.double().abs().t()).max())
    e = _eps(N, float(z.abs().max())) + 2 * gemm
    for lp_got, ent_got in out:
        _close(lp_got[:rows], lp, 2 * e)
        _close(ent_got[:rows], ent, (2 + ent) * e)
        assert lp_got[rows] == 7.0 and ent_got[rows] == 7.0       # rows behind the last one are left as they were
    with pytest.raises(K.KernelError):
        K.gemm_scores(a, b, ids, out[0][0], out[0][1], None, M, N, Kd, rows=M + 1)
    with pytest.raises(K.KernelError):
        K.gemm_scores(a, b, ids, out[0][0], out[0][1], None, M, N, Kd - 4, rows=rows)


@pytest.mark.parametrize("rows", [1, 5, 8, 9, 16, 17])
@pytest.mark.parametrize("V,d,cap", [(128, 64, None), (1000, 1024, 30.0), (20008, 520, None), (50304, 256, None)])
def test_head_scores_of_few_tokens(rows, V, d, cap):
    """Up to 16 tokens the product is formed with its operands exchanged."""
    head = _bf16_head(V, d, cap)
    w = head.weight.full()
    x = torch.randn(rows, d, generator=torch.Generator(device=DEV).manual_seed(3), device=DEV).to(torch.bfloat16)
    ids = torch.randint(0, V, (rows,), generator=torch.Generator(device=DEV).manual_seed(4), device=DEV)
    ids[0] = V - 1
    if rows > 4:
        ids[1], ids[2], ids[3], ids[4] = -100, V, 0, ids[0]
    z = x.double() @ w.double().t()
    gemm = d * 2.0 ** -24 * float((x.double().abs() @ w.double().abs().t()).max())
    lp, ent, _, _ = scores_64(z, ids, 1, 1.0, cap or 0.0)
    e = _eps(V, min(float(z.abs().max()), cap or math.inf), cap or 0.0) + 2 * gemm
    with torch.no_grad():
        out = head.token_log_probs(x, ids)
        again = head.token_log_probs(x, ids)
    _close(out.log_probs, lp, 2 * e)
    _close(out.entropy, ent, (2 + ent) * e)
    assert torch.equal(out.log_probs, again.log_probs) and torch.equal(out.entropy, again.entropy)
    leaf = x.clone().requires_grad_(True)                          # and the gradient, from the logits computed again
    got = head.token_log_probs(leaf, ids)
    gx, = torch.autograd.grad(got.log_probs.sum(), leaf)
    dz, _ = score_gradients_64(z, ids, torch.ones(rows, device=DEV), torch.zeros(rows, device=DEV), 1.0, cap or 0.0)
    want, size = dz @ w.double(), dz.abs() @ w.double().abs()
    _close(gx, want, (2.0 ** -8 + 2.0 ** -12 + 4 * e) * size + 2.0 ** -8 * want.abs() + 1e-12)


def test_certain_tokens_and_empty_batches():
    for cap in (None, 30.0):
        z = torch.full((64, 5000), -1000.0, device=DEV)
        z[:, 17] = torch.linspace(-20, 20, 64, device=DEV)
        out = F.token_log_probs(z, torch.full((64,), 17, device=DEV), logit_softcap=cap, temperature=0.25, top_k=2)
        assert torch.all(out.log_probs <= 0) and torch.all(out.top_log_probs <= 0) and torch.all(out.entropy >= 0)
    head = _bf16_head(64, 64)
    x = torch.zeros(0, 64, dtype=torch.bfloat16, device=DEV, requires_grad=True)
    ids = torch.zeros(0, dtype=torch.int64, device=DEV)
    out = head.token_log_probs(x, ids, top_k=3)
    loss = head.distillation_loss(x, ids.view(0, 1).expand(0, 4), torch.zeros(0, 4, device=DEV))
    z = torch.zeros(0, 10, device=DEV, requires_grad=True)
    kd = F.distillation_loss(z, ids.view(0, 1), torch.zeros(0, 1, device=DEV))
    gx, = torch.autograd.grad(out.log_probs.sum() + loss, x)
    assert out.top_ids.shape == (0, 3) and float(loss.detach()) == 0 and float(kd.detach()) == 0 and gx.shape == (0, 64)
    assert torch.autograd.grad(kd, z)[0].shape == (0, 10)


def test_distillation_of_more_classes_than_one_block_has_bits_for():
    rows, V = 400, 1_200_007
    z = torch.randn(rows, V, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV).to(torch.bfloat16)
    ids = torch.randint(0, V, (rows, 5), generator=torch.Generator(device=DEV).manual_seed(2), device=DEV)
    ids[:, 4] = ids[:, 0]
    t = torch.log(torch.tensor([0.4, 0.2, 0.1, 0.1, 0.7], device=DEV)).expand(rows, 5)
    loss = F.distillation_loss(z, ids, t, reduction="none")
    part = torch.arange(0, rows, 40, device=DEV)
    want, _ = distillation_64(z[part], ids[part], t[part], "rest", "none")
    _close(loss[part], want, 4 * _eps(V, 8.0) + 2.0 ** -23 * want.abs())


def test_head_scores_with_the_weights_still_to_be_gathered():
    """The epilogue's scores in a launch whose copy warps bring in the other shards (here from this GPU's memory)."""
    from olmax_b200.ops import _lib
    from olmax_b200.ops import kernels as K

    M, N, Kd, R = 264, 4096, 256, 4
    g = torch.Generator(device=DEV).manual_seed(6)
    a = torch.randn(M, Kd, generator=g, device=DEV).to(torch.bfloat16)
    b = torch.randn(N, Kd, generator=g, device=DEV).to(torch.bfloat16)
    per = N // R
    shards = [b[r * per : (r + 1) * per].clone() for r in range(R)]
    table = K.pointer_table([s.data_ptr() for s in shards], a.device)
    ids = _ids(M, N)
    want = [torch.empty(M, device=DEV) for _ in range(2)]
    K.gemm_scores(a, b, ids, *want, None, M, N, Kd, rows=M)
    for rank in (0, 2):
        buf = torch.zeros(R, per * Kd, dtype=torch.bfloat16, device=DEV)
        buf[rank] = shards[rank].view(-1)
        flags = torch.zeros(1024, dtype=torch.int32, device=DEV)
        got = [torch.empty(M, device=DEV) for _ in range(2)]
        K.gemm_scores(a, buf[0].view(per, Kd), ids, *got, None, M, N, Kd, rows=M, N_s=per, b_shard_stride=per * Kd, ag_src=table,
                      ag_flags=flags, ag_rank=rank)
        _lib.check_status()
        assert torch.equal(buf.view(N, Kd), b)
        for x, y in zip(got, want):
            _close(x, y, 4 * _eps(N, float((a.float() @ b.float().t()).abs().max())))


def test_extents_of_one_whatever_their_strides():
    z = _logits(5, 300)
    one = z[:, 7:8]                                                # one class: its stride says nothing
    odd = one.as_strided((5, 1), (300, 77))
    for t in (one, odd):
        out = F.token_log_probs(t, torch.zeros(5, dtype=torch.int64, device=DEV), top_k=1)
        assert torch.all(out.log_probs == 0) and torch.all(out.entropy == 0) and torch.all(out.top_ids == 0)
    ids, t = _teacher(5, 300, 1)
    for shape in ((5, 1), (1, 5)):                                 # one pair per row, one row
        zz = z if shape[0] == 5 else z[:1]
        i2, t2 = ids.view(shape), t.view(shape)
        i3 = torch.zeros(400, dtype=torch.int64, device=DEV).as_strided(shape, (13 if shape[0] > 1 else 50, 1 if shape[0] == 1 else 29)).copy_(i2)
        _check_distillation(zz, i3, t2, "rest")
        _check_scores(zz, ids.view(-1)[: zz.shape[0]], 3)
