"""The measured operators of a training step beside the table path: what the
rows and the PLE block's weights are trained on, and the update of the weights.

Kinds of case (``kind``):

* ``logprobs``   -- log-probabilities of given tokens from logits
                    (``losses.token_logprobs``): the reference policy's scores;
* ``policy``     -- the clipped policy loss with its KL term, and the gradient
                    of the logits (``losses.policy_loss_grad``);
* ``preference`` -- the preference loss of paired log ratios, and the gradient
                    of the logits (``losses.preference_loss_grad``);
* ``muon``       -- one momentum step of matrices whose update is
                    orthogonalised by Newton-Schulz products (``muon.muon_step``).

Logits are those of a packed sequence's positions over the benchmark's
vocabulary of 151,936 (whose last ids are no tokens and masked), or an odd one;
a target below 0 leaves its row out.  Matrices are the PLE block's projections
(``n_embd`` 2560, four streams), or smaller ones.
"""
from __future__ import annotations

import math

import torch

own = False  # False: the plain form of every operator; True: the framework's kernels

DEV = "cuda"
VOCAB = 151_936
REAL_TOKENS = 151_669  # ids from here on are no tokens: their logits are -inf
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
CLIP = (0.2, 0.28)  # the ratio is held in [1 - 0.2, 1 + 0.28]
KL_COEF, BETA, SMOOTHING = 0.04, 0.1, 0.05
GRAD_SCALE = {"f32": 1.0, "bf16": 1.0, "f16": 4096.0}  # of the logits' gradients: fp16 ones are scaled, as they are trained with
MOMENTUM, LR, DECAY, EPS, STEPS = 0.95, 0.02, 0.01, 1e-7, 5
QUINTIC = (3.4445, -4.7750, 2.0315)


def listed() -> list[dict]:
    return [
        # one answer token scored at one position
        dict(name="logprobs_one_token", kind="logprobs", n=1, v=VOCAB, dtype="bf16", temperature=1.0, ignored=0.0),
        # the reference policy's scores of a packed sequence
        dict(name="logprobs_packed", kind="logprobs", n=2047, v=VOCAB, dtype="bf16", temperature=1.0, ignored=0.3),
        # a short sampled answer, fp32 logits as the descent's replica gives them
        dict(name="policy_answer_f32", kind="policy", n=37, v=VOCAB, dtype="f32", temperature=1.0, ignored=0.2, segments=1,
             reduction="token"),
        # a packed sequence of sampled answers
        dict(name="policy_packed", kind="policy", n=2047, v=VOCAB, dtype="bf16", temperature=1.0, ignored=0.3, segments=7,
             reduction="token"),
        # four packed sequences in one step, sampled at another temperature, each answer counted alike
        dict(name="policy_batch", kind="policy", n=8188, v=VOCAB, dtype="bf16", temperature=0.7, ignored=0.3, segments=29,
             reduction="sequence"),
        # one fact's two answers, fp32 logits
        dict(name="preference_fact_f32", kind="preference", n=46, v=VOCAB, dtype="f32", temperature=1.0, ignored=0.4, pairs=1),
        # a packed sequence of answer pairs
        dict(name="preference_packed", kind="preference", n=2047, v=VOCAB, dtype="bf16", temperature=1.0, ignored=0.3, pairs=6),
        # an odd vocabulary in fp16: rows start at odd addresses
        dict(name="preference_odd_f16", kind="preference", n=1531, v=50_257, dtype="f16", temperature=1.0, ignored=0.3, pairs=11),
        # many small matrices of one shape
        dict(name="muon_small", kind="muon", count=16, rows=64, cols=256, dtype="bf16"),
        # the block's value projection
        dict(name="muon_value_f32", kind="muon", count=1, rows=2560, cols=2560, dtype="f32"),
        # the block's whole key projection as one tall matrix, bf16 weights
        dict(name="muon_key_tall_bf16", kind="muon", count=1, rows=10_240, cols=2560, dtype="bf16"),
        # the value projection and the key projection's four streams, a matrix each
        dict(name="muon_block_f32", kind="muon", count=5, rows=2560, cols=2560, dtype="f32"),
    ]


def draw(rng) -> dict:
    def span(lo: int, hi: int) -> int:  # log-uniform, odd sizes among them
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    kind = rng.choice(["logprobs", "policy", "preference", "muon"])
    if kind == "muon":
        rows, cols = span(16, 4096), span(16, 4096)
        work = min(rows, cols) ** 2 * max(rows, cols)
        count = max(1, min(span(1, 24), 5 * 2560 ** 3 // work))
        return dict(kind=kind, count=count, rows=rows, cols=cols, dtype=rng.choice(["f32", "bf16", "f16"]))
    v = rng.choice([VOCAB, span(1000, 160_000), span(1000, 160_000)])
    n = min(span(1, 8188), 8188 * VOCAB // (2 * v))
    case = dict(kind=kind, n=n, v=v, dtype=rng.choice(["f32", "bf16", "bf16", "f16"]),
                temperature=rng.choice([1.0, 1.0, 0.7, 1.3]), ignored=rng.choice([0.0, 0.3, 0.7]))
    if kind == "policy":
        case.update(segments=span(1, 32), reduction=rng.choice(["token", "sequence"]))
    if kind == "preference":
        case.update(pairs=span(1, 16))
    return case


# ---- inputs -----------------------------------------------------------------------------------

def _gen(seed: int, salt: int) -> torch.Generator:
    return torch.Generator(device=DEV).manual_seed((seed * 1_000_003 + salt) % (1 << 62))


def _logits(case: dict, seed: int):
    """Logits about N(0, 2.5), the target's higher by 0 to 14; masked ids at -inf; a row that is left out holds NaN."""
    n, v, t = case["n"], case["v"], TYPES[case["dtype"]]
    g = _gen(seed, 1)
    real = REAL_TOKENS if v == VOCAB else v
    z = torch.empty((n, v), dtype=t, device=DEV)
    for i in range(0, n, 1024):  # bounds the fp32 numbers made at once
        z[i:i + 1024] = torch.randn((min(1024, n - i), v), generator=g, device=DEV) * 2.5
    targets = torch.randint(0, real, (n,), generator=g, device=DEV)
    z.scatter_add_(1, targets[:, None], (torch.rand((n, 1), generator=g, device=DEV) * 14.0).to(t))
    z[:, real:] = -math.inf
    out = torch.rand(n, generator=g, device=DEV) < case["ignored"]
    targets[out] = -100
    z[out & (torch.rand(n, generator=g, device=DEV) < 0.1), :7] = math.nan
    return z, targets


def _segments(n: int, count: int, g) -> torch.Tensor:
    """``count`` segments of uneven lengths over ``n`` positions in order, some empty where positions are few."""
    cuts = torch.sort(torch.randint(0, n + 1, (count - 1,), generator=g, device=DEV)).values
    return torch.searchsorted(cuts, torch.arange(n, device=DEV), right=True)


def _scores(z, targets, temperature):
    """What an earlier pass of the model gave: fp32 log-probabilities of the targets (0 where a row is left out)."""
    lp = torch.zeros(z.shape[0], dtype=torch.float32, device=DEV)
    for i in range(0, z.shape[0], 1024):
        y = z[i:i + 1024].float() / temperature
        t = targets[i:i + 1024]
        s = y.gather(1, t.clamp_min(0)[:, None])[:, 0] - torch.logsumexp(y, 1)
        lp[i:i + 1024] = torch.where(t >= 0, s, torch.zeros_like(s))
    return lp


def prepare(case: dict, seed: int) -> dict:
    g = _gen(seed, 2)
    if case["kind"] == "muon":
        t, shape = TYPES[case["dtype"]], (case["rows"], case["cols"])

        def some(size):
            return [torch.randn(shape, generator=g, device=DEV) * size for _ in range(case["count"])]

        # a gradient has a few strong directions over noise, the momentum both of earlier steps
        low = [torch.randn((shape[0], 4), generator=g, device=DEV) @ torch.randn((4, shape[1]), generator=g, device=DEV)
               for _ in range(case["count"])]
        return dict(case=case, params=[w.to(t) for w in some(0.02)],
                    grads=[((x + 0.3 * r) * 1e-3).to(t) for x, r in zip(some(1.0), low)],
                    momenta=[(x + 0.3 * r) * 4e-3 for x, r in zip(some(1.0), low)])
    z, targets = _logits(case, seed)
    s = dict(case=case, logits=z, targets=targets)
    n = case["n"]
    if case["kind"] == "policy":
        lp = _scores(z, targets, case["temperature"])
        s["segment_ids"] = _segments(n, case["segments"], g)
        s["advantages"] = torch.randn(n, generator=g, device=DEV)
        shift = torch.randn(n, generator=g, device=DEV) * 0.2  # the policy's log-ratio to the one that sampled
        for edge in (math.log(1 - CLIP[0]), math.log(1 + CLIP[1])):  # none within rounding of where it is clipped
            shift = torch.where((shift - edge).abs() < 2e-3, shift + 5e-3, shift)
        s["old_logprobs"] = lp - shift
        s["ref_logprobs"] = lp + torch.randn(n, generator=g, device=DEV) * 0.3
    if case["kind"] == "preference":
        count = 2 * case["pairs"]
        s["segment_ids"] = _segments(n, count, g)
        total = torch.zeros(count, device=DEV).index_add_(0, s["segment_ids"], _scores(z, targets, case["temperature"]))
        s["ref_logprobs"] = total + torch.randn(count, generator=g, device=DEV) * 8.0
    return s


# ---- one pass ---------------------------------------------------------------------------------

def run(s: dict):
    case = s["case"]
    if own:
        import __graft_entry__

        __graft_entry__.load_package()
        return _run_own(s, case)
    return {"logprobs": _plain_logprobs, "policy": _plain_policy, "preference": _plain_preference, "muon": _plain_muon}[case["kind"]](s, case)


def _run_own(s, case):
    kind = case["kind"]
    if kind == "muon":
        from engraft_ngram_amd import muon

        muon.muon_step(s["params"], s["grads"], s["momenta"], lr=LR, weight_decay=DECAY, momentum=MOMENTUM, nesterov=True,
                       steps=STEPS, coefficients=QUINTIC, eps=EPS)
        return dict(params=s["params"], momenta=s["momenta"])
    from engraft_ngram_amd import losses

    if kind == "logprobs":
        return losses.token_logprobs(s["logits"], s["targets"], temperature=case["temperature"])
    if kind == "policy":
        r, d = losses.policy_loss_grad(s["logits"], s["targets"], s["advantages"], s["old_logprobs"], ref_logprobs=s["ref_logprobs"],
                                       segment_ids=s["segment_ids"], n_segments=case["segments"], clip=CLIP, kl_coef=KL_COEF,
                                       temperature=case["temperature"], reduction=case["reduction"], grad_scale=GRAD_SCALE[case["dtype"]])
        return dict(loss=r.loss, kl=r.kl, clip_fraction=r.clip_fraction, logprobs=r.logprobs, d_logits=d)
    r, d = losses.preference_loss_grad(s["logits"], s["targets"], s["segment_ids"], s["ref_logprobs"], beta=BETA,
                                       label_smoothing=SMOOTHING, temperature=case["temperature"],
                                       grad_scale=GRAD_SCALE[case["dtype"]])
    return dict(loss=r.loss, margins=r.margins, sequence_logprobs=r.sequence_logprobs, logprobs=r.logprobs, d_logits=d)


def _softmax_stats(s, case):
    """exp(y - max), its sum, and the targets' log-probabilities, in fp32; rows left out count as zeros."""
    valid = s["targets"] >= 0
    y = torch.where(valid[:, None], s["logits"].float(), 0.0) / case["temperature"]
    top = y.amax(1, keepdim=True)
    e = (y - top).exp()
    total = e.sum(1, keepdim=True)
    lp = y.gather(1, s["targets"].clamp_min(0)[:, None]) - top - total.log()
    return valid, e, total, torch.where(valid, lp[:, 0], 0.0)


def _plain_logprobs(s, case):
    return _softmax_stats(s, case)[3]


def _d_logits(s, case, e, total, d_lp):
    """d_lp (onehot - softmax) / temperature, times the gradients' scale."""
    d = e * (-d_lp[:, None] / total)
    d.scatter_add_(1, s["targets"].clamp_min(0)[:, None], d_lp[:, None])
    return (d * (GRAD_SCALE[case["dtype"]] / case["temperature"])).to(s["logits"].dtype)


def _plain_policy(s, case):
    valid, e, total, lp = _softmax_stats(s, case)
    one = valid.float()
    if case["reduction"] == "token":
        w = one / one.sum().clamp_min(1.0)
    else:
        each = torch.zeros(case["segments"], device=DEV).index_add_(0, s["segment_ids"], one)
        w = one / (each.clamp_min(1.0) * (each > 0).sum().clamp_min(1))[s["segment_ids"]]
    ratio = (lp - s["old_logprobs"]).exp()
    a = s["advantages"]
    free, held = ratio * a, ratio.clamp(1 - CLIP[0], 1 + CLIP[1]) * a
    diff = s["ref_logprobs"] - lp
    kl = diff.exp() - diff - 1.0
    loss = (w * (KL_COEF * kl - torch.minimum(free, held))).sum()
    d_lp = w * (KL_COEF * (1.0 - diff.exp()) - torch.where(free <= held, free, 0.0))
    return dict(loss=loss, kl=(w * kl).sum(), clip_fraction=(w * (free > held).float()).sum(), logprobs=lp,
                d_logits=_d_logits(s, case, e, total, d_lp))


def _plain_preference(s, case):
    valid, e, total, lp = _softmax_stats(s, case)
    seqs = torch.zeros(2 * case["pairs"], device=DEV).index_add_(0, s["segment_ids"], lp)
    gain = (seqs - s["ref_logprobs"]).reshape(-1, 2)
    h = BETA * (gain[:, 0] - gain[:, 1])
    tail = (1.0 + (-h.abs()).exp()).log()
    loss = ((1 - SMOOTHING) * (tail + (-h).clamp_min(0.0)) + SMOOTHING * (tail + h.clamp_min(0.0))).mean()
    d_h = (SMOOTHING / (1.0 + (-h).exp()) - (1 - SMOOTHING) / (1.0 + h.exp())) / case["pairs"]
    d_seq = torch.stack([BETA * d_h, -BETA * d_h], 1).reshape(-1)
    d_lp = torch.where(valid, d_seq[s["segment_ids"]], 0.0)
    return dict(loss=loss, margins=h, sequence_logprobs=seqs, logprobs=lp, d_logits=_d_logits(s, case, e, total, d_lp))


def _plain_muon(s, case):
    a, b, c = QUINTIC
    tall = case["rows"] > case["cols"]
    g = torch.stack(s["grads"]).float()
    m = MOMENTUM * torch.stack(s["momenta"]) + g
    u = g + MOMENTUM * m
    x = u / (u.square().sum((1, 2), keepdim=True).sqrt() + EPS)
    x = x.mT.contiguous() if tall else x
    for _ in range(STEPS):
        gram = x @ x.mT.contiguous()
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    x = x.mT if tall else x
    w = torch.stack(s["params"]).float() * (1 - LR * DECAY) - LR * math.sqrt(max(1.0, case["rows"] / case["cols"])) * x
    for to, new in zip(s["params"] + s["momenta"], list(w) + list(m)):
        to.copy_(new)
    return dict(params=s["params"], momenta=s["momenta"])


# ---- bytes and operations ---------------------------------------------------------------------

def work(case: dict) -> dict:
    size = TYPES[case["dtype"]].itemsize
    if case["kind"] == "muon":
        m, n = sorted((case["rows"], case["cols"]))
        # per iteration: half of x x^T and of its square (both symmetric), and a whole product with x
        flops = case["count"] * STEPS * (m * m * n + m * m * m + 2 * m * m * n)
        return {"bytes": case["count"] * m * n * (3 * size + 8), "flops": flops}  # weight in and out, gradient, momentum in and out
    kept = case["n"] * case["v"] * (1 - case["ignored"])
    if case["kind"] == "logprobs":
        return {"bytes": kept * size + 12 * case["n"], "flops": 4 * kept}
    return {"bytes": (kept + case["n"] * case["v"]) * size + 40 * case["n"], "flops": 8 * kept}


# ---- the definition in 64 bits ----------------------------------------------------------------

def exact(case: dict, seed: int):
    s = prepare(case, seed)
    if case["kind"] == "muon":
        return _exact_muon(s, case)
    n, tau = case["n"], case["temperature"]
    tg = s["targets"]
    keep = torch.nonzero(tg >= 0)[:, 0]
    rows = 512  # positions at a time

    def scores(idx, z):
        return torch.log_softmax(z / tau, 1)[torch.arange(len(idx), device=DEV), tg[idx]]

    lp = torch.zeros(n, dtype=torch.float64, device=DEV)
    for idx in keep.split(rows):
        lp[idx] = scores(idx, s["logits"][idx].double())
    if case["kind"] == "logprobs":
        return lp
    leaf = lp.clone().requires_grad_()
    if case["kind"] == "policy":
        seg = s["segment_ids"]
        w = torch.zeros(n, dtype=torch.float64, device=DEV)
        if case["reduction"] == "token":
            w[keep] = 1.0 / max(1, len(keep))
        else:
            each = torch.bincount(seg[keep], minlength=case["segments"]).double()
            w[keep] = 1.0 / (each[seg[keep]] * float((each > 0).sum()))
        r = torch.exp(leaf - s["old_logprobs"].double())
        a = s["advantages"].double()
        free, held = r * a, torch.clamp(r, 1 - CLIP[0], 1 + CLIP[1]) * a
        log_q = s["ref_logprobs"].double() - leaf
        kl = torch.expm1(log_q) - log_q
        surrogate = torch.where(free <= held, free, held.detach())
        loss = (w[keep] * (KL_COEF * kl - surrogate)[keep]).sum()
        said = dict(loss=loss.detach(), kl=(w[keep] * kl.detach()[keep]).sum(), clip_fraction=w[(free > held) & (tg >= 0)].sum(), logprobs=lp)
    else:
        seqs = torch.stack([leaf[s["segment_ids"] == k].sum() for k in range(2 * case["pairs"])])
        gain = seqs - s["ref_logprobs"].double()
        h = BETA * (gain[0::2] - gain[1::2])
        loss = -((1 - SMOOTHING) * torch.nn.functional.logsigmoid(h) + SMOOTHING * torch.nn.functional.logsigmoid(-h)).mean()
        said = dict(loss=loss.detach(), margins=h.detach(), sequence_logprobs=seqs.detach(), logprobs=lp)
    (d_lp,) = torch.autograd.grad(loss, leaf)
    d = torch.zeros((n, case["v"]), dtype=torch.float64, device=DEV)
    for idx in keep.split(rows):
        z = s["logits"][idx].double().requires_grad_()
        (d[idx],) = torch.autograd.grad((scores(idx, z) * d_lp[idx]).sum() * GRAD_SCALE[case["dtype"]], z)
    return dict(said, d_logits=d)


def _exact_muon(s, case):
    a, b, c = QUINTIC
    params, momenta = [], []
    for w, grad, buf in zip(s["params"], s["grads"], s["momenta"]):
        m = MOMENTUM * buf.double() + grad.double()
        u = grad.double() + MOMENTUM * m
        x = u / (torch.linalg.matrix_norm(u) + EPS)
        eye = torch.eye(min(x.shape), dtype=torch.float64, device=DEV)
        for _ in range(STEPS):  # p(x) = (a + b x x^T + c (x x^T)^2) x, on whichever side is the smaller
            if x.shape[0] <= x.shape[1]:
                q = x @ x.T
                x = (a * eye + b * q + c * q @ q) @ x
            else:
                q = x.T @ x
                x = x @ (a * eye + b * q + c * q @ q)
        momenta.append(m)
        params.append((1 - LR * DECAY) * w.double() - LR * math.sqrt(max(1.0, w.shape[0] / w.shape[1])) * x)
    return dict(params=params, momenta=momenta)
