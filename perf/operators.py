"""
Performance cases of the operators around the LM head's distribution: log probabilities of given tokens with entropy and
top alternatives, distillation from a teacher's top classes, and the same scores through the LM head.

A case is a dict of plain values; :func:`prepare` makes what a program has in hand before the call, :func:`run` makes one
pass (with ``own`` through the framework's operators, else in elementary torch operations in 32 bits), :func:`work` counts
what the pass cannot do without, :func:`exact` evaluates the definition in 64 bits.

``kind``:

* ``score``: ``token_log_probs`` without gradients: log p of given tokens and the entropy, with ``top`` > 0 also the most
  likely classes; ``given`` false asks for the entropy and the classes alone (a teacher's pass).
* ``train``: ``token_log_probs`` and the gradient of the logits for upstream gradients of both outputs.
* ``head``: the log probabilities and entropies of hidden states through an LM head.
* ``distill``: ``distillation_loss`` (mean) and the gradient of the logits.
"""

import math

import torch

own = False

_TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}


def listed():
    return [
        # One step of sampling from the 271M model: a single token's row, its log probability and five alternatives.
        dict(name="score-one", kind="score", rows=1, classes=50304, dtype="fp32", cap=0.0, temp=1.0, top=5, given=True, pad=0),
        # A decoding batch of 64 sequences at the Llama3 vocabulary: 20 alternatives each, bf16 logits.
        dict(name="score-batch", kind="score", rows=64, classes=128256, dtype="bf16", cap=0.0, temp=1.0, top=20, given=True, pad=0),
        # A scored prompt with an odd vocabulary (rows that start at every 4-byte offset), tempered and soft-capped.
        dict(name="score-odd", kind="score", rows=777, classes=50257, dtype="fp32", cap=30.0, temp=0.7, top=0, given=True, pad=0),
        # An evaluation batch at the OLMo2 vocabulary, whose padded classes are masked.
        dict(name="score-eval", kind="score", rows=4096, classes=100352, dtype="fp32", cap=0.0, temp=1.0, top=0, given=True, pad=74),
        # A teacher's pass: the 64 most likely classes of every token of a chunk.
        dict(name="teacher-top64", kind="score", rows=2048, classes=128256, dtype="fp32", cap=0.0, temp=1.0, top=64, given=False, pad=0),
        # A policy-gradient step with an entropy bonus over one chunk of the OLMo2 head.
        dict(name="policy-fp32", kind="train", rows=2048, classes=100352, dtype="fp32", cap=0.0, temp=1.0),
        # The same on bf16 logits, a ragged number of tokens, tempered and soft-capped.
        dict(name="policy-bf16", kind="train", rows=3001, classes=50304, dtype="bf16", cap=30.0, temp=0.8),
        # Scoring one prompt through the 271M model's head.
        dict(name="head-271M", kind="head", rows=328, classes=50304, width=1024, cap=0.0, temp=1.0),
        # An evaluation micro-batch through the OLMo2 7B head.
        dict(name="head-7B", kind="head", rows=4096, classes=100352, width=4096, cap=0.0, temp=1.0),
        # Unit-test sized distillation (the smoke model's vocabulary), renormalised top 8.
        dict(name="distill-small", kind="distill", rows=40, classes=4096, dtype="fp32", cap=0.0, temp=1.0, top=8, tail="renormalize"),
        # A chunk of an OLMo2 student against a stored top-64 teacher, the rest of the vocabulary as one class.
        dict(name="distill-rest", kind="distill", rows=2048, classes=100352, dtype="fp32", cap=0.0, temp=1.0, top=64, tail="rest"),
        # A Gemma2-like student: 256000 classes, bf16, soft-capped, at temperature 2, top 128, a ragged number of tokens.
        dict(name="distill-gemma", kind="distill", rows=1021, classes=256000, dtype="bf16", cap=30.0, temp=2.0, top=128, tail="rest"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        kind = rng.choice(["score", "score", "train", "head", "distill", "distill"])
        case = dict(kind=kind, rows=_log_int(rng, 1, 8192), cap=rng.choice([0.0, 0.0, 30.0]), temp=rng.choice([1.0, 1.0, 0.7, 2.0]))
        classes = _log_int(rng, 1000, 256000)
        if kind == "head":   # the head's GEMM takes whole 16-byte rows of both matrices
            case.update(classes=max(8, classes // 8 * 8), width=_log_int(rng, 64, 512) * 8)
        else:
            case.update(classes=classes, dtype=rng.choice(["fp32", "fp32", "bf16"]))
            if kind == "score":
                case.update(top=rng.choice([0, 0, 1, _log_int(rng, 2, 128)]), given=True, pad=rng.choice([0, 0, rng.randint(1, 100)]))
                if case["top"] and rng.random() < 0.3:
                    case["given"] = False
            if kind == "distill":
                case.update(top=_log_int(rng, 1, 128), tail=rng.choice(["rest", "rest", "renormalize"]))
        if _cost(case) <= most:
            return case


# ------------------------------------------------------------------------------------------------------------ the work
def work(case):
    rows, classes = case["rows"], case["classes"]
    if case["kind"] == "head":
        d = case["width"]
        return {"bytes": 2 * d * (rows + classes) + 16 * rows, "flops": 2 * rows * classes * d}
    size = 4 if case["dtype"] == "fp32" else 2
    if case["kind"] == "score":
        nbytes = size * rows * classes + rows * (4 + (12 if case["given"] else 0) + 12 * case["top"])
        return {"bytes": nbytes, "flops": 5 * rows * classes}
    nbytes = 2 * size * rows * classes   # the logits in, their gradient out
    if case["kind"] == "train":
        return {"bytes": nbytes + 24 * rows, "flops": 10 * rows * classes}
    return {"bytes": nbytes + 12 * rows * case["top"] + 4, "flops": 8 * rows * classes}


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 250)


# ---------------------------------------------------------------------------------------------------------- the inputs
def _logits(gen, dev, rows, classes, dtype, pad=0):
    """Logits as a language model gives them: frequent (low) classes ahead, a few peaks in every row, padding masked."""
    z = torch.randn(rows, classes, generator=gen, device=dev).mul_(2.0)
    z -= 0.6 * torch.arange(1, classes + 1, device=dev, dtype=torch.float32).log_()
    peaks = torch.randint(0, classes - pad, (rows, 6), generator=gen, device=dev)
    height = torch.rand(rows, 6, generator=gen, device=dev) * 12.0
    z.scatter_add_(1, peaks, height)
    if pad:
        z[:, classes - pad:] = -math.inf
    return z.to(_TYPES[dtype]), peaks


def _inputs(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=dev).manual_seed(seed)
    rows, classes = case["rows"], case["classes"]
    s = dict(case=case)
    if case["kind"] == "head":
        d = case["width"]
        s["x"] = torch.randn(rows, d, generator=gen, device=dev).to(torch.bfloat16)
        s["weight"] = (torch.randn(classes, d, generator=gen, device=dev) * (3.0 / math.sqrt(d))).to(torch.bfloat16)
        s["ids"] = torch.randint(0, classes, (rows,), generator=gen, device=dev)
    else:
        pad = case.get("pad", 0)
        s["logits"], peaks = _logits(gen, dev, rows, classes, case["dtype"], pad)
        anywhere = torch.randint(0, classes - pad, (rows,), generator=gen, device=dev)
        likely = torch.rand(rows, generator=gen, device=dev) < 0.7
        s["ids"] = torch.where(likely, peaks[:, 0], anywhere)
    if case["kind"] in ("head", "score", "train"):
        s["ids"][torch.rand(rows, generator=gen, device=dev) < 0.05] = -100   # prompt tokens that are not scored
    if case["kind"] == "train":
        s["g_log_probs"] = torch.randn(rows, generator=gen, device=dev) / rows
        s["g_entropy"] = torch.full((rows,), -0.01 / rows, device=dev)
    if case["kind"] == "distill":
        # a teacher that agrees with the student in part; rows of a prompt, and the ends of short lists, are padding
        k = min(case["top"], classes)
        teacher = s["logits"].float()
        teacher = teacher + torch.randn(rows, classes, generator=gen, device=dev)
        best, ids = teacher.topk(k, dim=-1)
        lse = torch.logsumexp(teacher / case["temp"], dim=-1, keepdim=True)
        del teacher
        s["teacher_log_probs"] = (best / case["temp"] - lse).contiguous()
        length = torch.where(torch.rand(rows, 1, generator=gen, device=dev) < 0.1,
                             torch.randint(0, k + 1, (rows, 1), generator=gen, device=dev), k)
        s["teacher_ids"] = ids.masked_fill(torch.arange(k, device=dev) >= length, -1)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own and case["kind"] == "head":
        from olmax_b200.nn import LMHead
        from olmax_b200.nn.module import build_module
        from olmax_b200.parallel import MeshResource

        s["head"] = build_module(lambda: LMHead(case["width"], case["classes"], logit_softcap=case["cap"] or None),
                                 mesh_resource=MeshResource.FSDP(1), device=s["x"].device)
        s["head"].store.load_full("proj.weight", s["weight"])
        s["head"].store.sync_shadow()
    if own and case["kind"] in ("train", "distill"):
        s["logits"].requires_grad_(True)
    return s


# -------------------------------------------------------------------------------------------------- with the operators
def _run_own(s):
    from olmax_b200.ops import functional as F

    case = s["case"]
    kind = case["kind"]
    if kind == "head":
        with torch.no_grad():
            out = s["head"].token_log_probs(s["x"], s["ids"], temperature=case["temp"])
        return out.log_probs, out.entropy
    if kind == "distill":
        loss = F.distillation_loss(s["logits"], s["teacher_ids"], s["teacher_log_probs"], temperature=case["temp"],
                                   tail=case["tail"], logit_softcap=case["cap"])
        return (loss.detach(), *torch.autograd.grad(loss, s["logits"]))
    options = dict(temperature=case["temp"], logit_softcap=case["cap"])
    if kind == "train":
        out = F.token_log_probs(s["logits"], s["ids"], **options)
        grad, = torch.autograd.grad((out.log_probs, out.entropy), s["logits"], (s["g_log_probs"], s["g_entropy"]))
        return out.log_probs.detach(), out.entropy.detach(), grad
    out = F.token_log_probs(s["logits"], s["ids"] if case["given"] else None, top_k=min(case["top"], case["classes"]), **options)
    return tuple(t for t in out if t is not None)


# ----------------------------------------------------------------------------------------------------------- plain form
def _distribution(logits, case):
    """(log p, p, d(scaled logit) / d(logit)) of rows of logits."""
    z = logits.float()
    slope = 1.0 / case["temp"]
    if case["cap"]:
        t = torch.tanh(z / case["cap"])
        z = case["cap"] * t
        slope = slope * (1.0 - t * t)
    z = z / case["temp"]
    z = z - z.amax(-1, keepdim=True)
    log_p = z - z.exp().sum(-1, keepdim=True).log()
    return log_p, log_p.exp(), slope


def _plain_scores(log_p, p, ids):
    entropy = -torch.where(p > 0, p * log_p, 0.0).sum(-1)
    known = (ids >= 0) & (ids < p.shape[-1])
    taken = log_p.gather(-1, ids.where(known, 0).unsqueeze(-1)).squeeze(-1)
    return torch.where(known, taken, 0.0), entropy, known


def _run_plain(s):
    case = s["case"]
    kind = case["kind"]
    if kind == "head":
        log_p, p, _ = _distribution(s["x"].float() @ s["weight"].float().t(), case)
        return _plain_scores(log_p, p, s["ids"])[:2]
    log_p, p, slope = _distribution(s["logits"], case)
    if kind == "score":
        log_probs, entropy, _ = _plain_scores(log_p, p, s["ids"])
        out = (log_probs, entropy) if case["given"] else (entropy,)
        if case["top"]:
            # largest logits first, equal ones by their class
            best = s["logits"].sort(dim=-1, descending=True, stable=True).indices[:, : case["top"]].contiguous()
            out += (log_p.gather(-1, best), best)
        return out
    if kind == "train":
        log_probs, entropy, known = _plain_scores(log_p, p, s["ids"])
        g = torch.where(known, s["g_log_probs"], 0.0).unsqueeze(-1)
        d = -p * (g + s["g_entropy"].unsqueeze(-1) * torch.where(p > 0, log_p + entropy.unsqueeze(-1), 0.0))
        d.scatter_add_(-1, s["ids"].where(known, 0).unsqueeze(-1), g)
        return log_probs, entropy, (d * slope).to(s["logits"].dtype)
    ids, t = s["teacher_ids"], s["teacher_log_probs"]
    rows, classes = log_p.shape
    given = ids >= 0
    some = given.any(-1, keepdim=True)
    q = torch.where(given, t.double().exp(), 0.0)   # 64 bits: what the listed classes leave of one can be little
    if case["tail"] == "renormalize":
        q = q / torch.where(some, q.sum(-1, keepdim=True), 1.0)
    mass = q.sum(-1, keepdim=True)
    listed_ = torch.zeros(rows, classes + 1, dtype=torch.bool, device=ids.device)
    listed_ = listed_.scatter_(1, ids.where(given, classes), True)[:, :classes]
    others = log_p.masked_fill(listed_, -math.inf)
    top = others.amax(-1, keepdim=True)
    rest_log_p = top + (others - top).exp().sum(-1, keepdim=True).log()
    rest = torch.where(some & rest_log_p.isfinite(), 1.0 - mass, 0.0).clamp(min=0.0)
    if case["tail"] == "renormalize":
        rest = torch.zeros_like(rest)
    total, rest, q = (mass + rest).float(), rest.float(), q.float()
    taken = log_p.gather(-1, ids.where(given, 0))
    loss = torch.where(q > 0, q * (q.log() - taken), 0.0).sum(-1, keepdim=True)
    loss = loss + torch.where(rest > 0, rest * (rest.log() - rest_log_p), 0.0)
    d = total * p - torch.where(rest > 0, rest * (others - rest_log_p).exp(), 0.0)
    d.scatter_add_(1, ids.where(given, 0), -q)
    count = some.sum().clamp(min=1)
    return loss.sum() / count, (d * slope / count).to(s["logits"].dtype)


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ------------------------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    """The definitions in 64 bits, a block of rows at a time; integers from repeated searches for the largest logit."""
    s = _inputs(case, seed)
    rows, classes = case["rows"], case["classes"]
    cap, temp, kind = case["cap"], case["temp"], case["kind"]
    block = max(1, 2 ** 25 // classes)
    parts = []
    scored = torch.tensor(0, device=s["ids"].device if "ids" in s else None)
    if kind == "distill":
        scored = (s["teacher_ids"] >= 0).any(1).sum().clamp(min=1).double()
    for r in range(0, rows, block):
        cut = slice(r, min(rows, r + block))
        raw = s["x"][cut].double() @ s["weight"].double().T if kind == "head" else s["logits"][cut].double()
        y = (torch.tanh(raw / cap) * cap if cap else raw) / temp
        dy = (1 - torch.tanh(raw / cap).square() if cap else torch.ones_like(raw)) / temp
        lse = torch.logsumexp(y, 1)
        prob = torch.softmax(y, 1)
        n = torch.arange(y.shape[0], device=y.device)
        if kind != "distill":
            ids = s["ids"][cut]
            ok = (0 <= ids) & (ids < classes)
            lp = torch.where(ok, y[n, ids.clamp(0, classes - 1)] - lse, 0)
            ent = -torch.special.xlogy(prob, prob).sum(1)
            one = (lp, ent) if case.get("given", True) else (ent,)
            if kind == "train":
                dlp = -prob
                dlp[n, ids.clamp(0, classes - 1)] += 1
                dent = -torch.special.xlogy(prob, prob) - prob * ent[:, None]
                one += ((dlp * (s["g_log_probs"][cut].double() * ok)[:, None]
                         + dent * s["g_entropy"][cut].double()[:, None]) * dy,)
            if kind == "score" and case["top"]:
                left, found = raw.clone(), []
                for _ in range(min(case["top"], classes)):
                    found.append(left.argmax(1))
                    left[n, found[-1]] = -math.inf
                found = torch.stack(found, 1)
                one += (y.gather(1, found) - lse[:, None], found)
            parts.append(one)
            continue
        ids, t = s["teacher_ids"][cut], s["teacher_log_probs"][cut].double()
        target = torch.zeros(y.shape[0], classes + 1, dtype=torch.float64, device=y.device)
        weight = torch.where(ids < 0, -math.inf, t)
        empty = (ids < 0).all(1)
        weight = torch.softmax(weight, 1).nan_to_num(0.0) if case["tail"] == "renormalize" else weight.exp()
        target.scatter_(1, ids.where(ids >= 0, classes), weight)
        target = target[:, :classes]
        named = torch.zeros(y.shape[0], classes + 1, dtype=torch.float64, device=y.device)
        named = named.scatter_(1, ids.where(ids >= 0, classes), 1.0)[:, :classes] > 0
        rest_q = (1 - target.sum(1)).clamp(min=0) * ~empty
        rest_q = rest_q * ~named.all(1) * (case["tail"] == "rest")
        lt = torch.logsumexp(torch.where(named, -math.inf, y), 1)
        log_p = y - lse[:, None]
        per_row = (torch.special.xlogy(target, target) - target * log_p).sum(1)
        per_row = per_row + torch.special.xlogy(rest_q, rest_q) - torch.where(rest_q > 0, rest_q * (lt - lse), 0)
        spread = torch.where(named, 0.0, (y - lt[:, None]).exp()) * rest_q[:, None]
        d = ((target.sum(1) + rest_q)[:, None] * prob - target - spread) * dy / scored
        parts.append((per_row, d))
    out = [torch.cat(p) for p in zip(*parts)]
    if kind == "distill":
        out[0] = out[0].sum() / scored
    return tuple(out)
