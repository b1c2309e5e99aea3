"""Values of the losses (``losses``) where they are hard to get: terms of no weight beside infinities, margins and
KL terms without end, losses that nearly cancel, gradients that overlap what they are made from.  The formulas are in
64 bits."""
from __future__ import annotations

import math

import pytest
import torch

from tests.test_gpu_losses import ALL, assert_within, lp_error, make, memory_returned, plain  # noqa: F401

pytestmark = pytest.mark.gpu


def test_overlapping_gradients_are_refused(cuda):
    """The gradient may lie in the logits' place or apart from them, also between their rows, but over none of them
    elsewhere, and over no other argument."""
    from engraft_ngram_amd import losses
    v, n = 100, 6
    buf = torch.randn(n + 1, 2 * v, device=cuda)
    t, a = torch.zeros(n, dtype=torch.int64, device=cuda), torch.zeros(n, device=cuda)
    z = buf[:n, :v]
    seg, ref = torch.arange(n, device=cuda), torch.zeros(n, device=cuda)
    wide = torch.zeros((n, v + n), device=cuda)
    kept = buf.clone()
    for out in (buf[1:, :v], buf[:n, 1:v + 1], buf[:n, v - 1:2 * v - 1], buf.view(-1)[:n * v].view(n, v),
                buf.view(-1)[v - 1:v - 1 + n * v].view(n, v)):
        for call in (lambda: losses.policy_loss_grad(z, t, a, out=out), lambda: losses.preference_loss_grad(z, t, seg, ref, out=out)):
            with pytest.raises(ValueError, match="overlap|row stride"):
                call()
    for call in (lambda: losses.policy_loss_grad(z, t, wide.view(-1)[:n], out=wide[:, :v]),
                 lambda: losses.policy_loss_grad(z, t, a, wide[0, 3:3 + n], out=wide[:, :v]),
                 lambda: losses.preference_loss_grad(z, t, seg, wide[0, 3:3 + n], out=wide[:, :v])):
        with pytest.raises(ValueError, match="overlap"):
            call()
    assert torch.equal(buf, kept)
    for call in (lambda **k: losses.policy_loss_grad(z, t, a + 1.0, **k), lambda **k: losses.preference_loss_grad(z, t, seg, ref, **k)):
        want = call()[1]
        assert torch.equal(call(out=buf[:n, v:])[1], want)
        assert torch.equal(call(out=buf[:n, v:v + v])[1], want) and torch.equal(z, kept[:n, :v])


# few rows in parts, few and some and many rows in one part each, held rows
SHAPES = [(5, 20_011), (37, 701), (300, 701), (600, 701), (520, 50_257)]


def masked_targets(n, v, dtype, seed):
    """make()'s rows, the target of the first rows with one at -inf."""
    z, t = make(n, v, dtype, seed, ignored=0.2 if n > 10 else 0.0)
    rows = torch.nonzero(t >= 0)[:3, 0]
    z[rows, t[rows]] = -math.inf
    return z, t, rows


@pytest.mark.parametrize("reduction", ["sum", "token", "sequence"])
@pytest.mark.parametrize("n,v", SHAPES)
def test_a_reference_without_a_kl_term(cuda, n, v, reduction):
    """kl_coef 0 with a reference (to report KL): loss and gradient are those without it, also where the policy gives a
    target no probability (KL is infinite there) or 1e-40 of the reference's."""
    from engraft_ngram_amd import losses
    z, t, rows = masked_targets(n, v, torch.float32, 1)
    far = torch.nonzero(t >= 0)[3, 0]
    z[far, t[far]] = -100.0
    a = torch.randn(n, generator=torch.Generator().manual_seed(2)).cuda()
    old, ref = torch.full((n,), -3.0, device=cuda), torch.full((n,), -2.5, device=cuda)
    seg = torch.arange(n, device=cuda) * 3 // n
    kw = dict(segment_ids=seg, n_segments=3, reduction=reduction)
    want, d_want = losses.policy_loss_grad(z, t, a, old, **kw)
    res, d = losses.policy_loss_grad(z, t, a, old, ref_logprobs=ref, **kw)
    assert want.loss.isfinite() and d_want.isfinite().all()
    assert torch.equal(res.loss, want.loss) and torch.equal(d, d_want)
    assert float(res.kl) == math.inf
    leaf = z.clone().requires_grad_()
    auto = losses.policy_loss(leaf, t, a, old, ref_logprobs=ref, **kw)
    auto.loss.backward()
    assert torch.equal(auto.loss.detach(), want.loss) and torch.equal(leaf.grad, d_want) and float(auto.kl) == math.inf
    # with a KL term the loss is as infinite as the term; rows without an infinite one keep their gradient
    res, d = losses.policy_loss_grad(z, t, a, old, ref_logprobs=ref, kl_coef=0.1, **kw)
    assert float(res.loss) == math.inf and float(res.kl) == math.inf
    rest = torch.ones(n, dtype=torch.bool, device=cuda)
    rest[rows] = rest[far] = False
    assert d[rest].isfinite().all()


@pytest.mark.parametrize("n,v", SHAPES)
def test_infinite_margins(cuda, n, v):
    """A masked token in the rejected answer: the pair is won beyond doubt, -log sigma(inf) = 0; in the chosen one: lost, an
    infinite loss.  With smoothing 1 the two change places; between, both are infinite.  The other pair stays as it is."""
    from engraft_ngram_amd import losses
    for which, eps, want in ((1, 0.0, 0.0), (0, 0.0, math.inf), (0, 1.0, 0.0), (1, 1.0, math.inf), (1, 0.1, math.inf),
                             (0, 0.1, math.inf)):
        z, t = make(n, v, torch.float32, 3, ignored=0.0)
        seg = torch.arange(n, device=cuda) * 4 // n
        ref = torch.zeros(4, device=cuda)
        row = int(torch.nonzero(seg == which)[0, 0])
        z[row, t[row]] = -math.inf
        lp = plain(z, t, 1.0)[0]
        h = 0.1 * (lp[seg == 2].sum() - lp[seg == 3].sum())
        other = -((1 - eps) * torch.nn.functional.logsigmoid(h) + eps * torch.nn.functional.logsigmoid(-h))
        res, d = losses.preference_loss_grad(z, t, seg, ref, label_smoothing=eps)
        assert float(res.margins[0]) == (math.inf if which == 1 else -math.inf)
        if want == 0.0:
            assert_within(res.loss, other / 2, 0.05 * n * lp_error(40.0) + 2.0 ** -23 * other)
            assert (d[seg < 2] == 0).all()
        else:
            assert float(res.loss) == want
        assert d.isfinite().all() and (d[seg >= 2] != 0).any()
        leaf = z.clone().requires_grad_()
        auto = losses.preference_loss(leaf, t, seg, ref, label_smoothing=eps)
        auto.loss.backward()
        assert torch.equal(auto.loss.detach(), res.loss) and torch.equal(leaf.grad, d)


def exact_rows(n, v, seed):
    """Logits of 0 and -inf: a row's sum is a whole number and its target's log-probability -log of it."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    some = torch.randint(2, v + 1, (n,), generator=g, device="cuda")
    z = torch.zeros((n, v), device="cuda").masked_fill_(torch.arange(v, device="cuda") >= some[:, None], -math.inf)
    return z, torch.zeros(n, dtype=torch.int64, device="cuda"), -some.double().log()


@pytest.mark.parametrize("reduction", ["sum", "token", "sequence"])
@pytest.mark.parametrize("n,v", [(6, 20_011), (64, 1003), (700, 1003)])
def test_losses_that_nearly_cancel(cuda, n, v, reduction):
    """Rows whose log-probabilities are exact: the loss and the KL term are off by the 64-bit terms' rounding (below 2^-44 of
    the terms' sizes, expm1 and log included) and fp32's of the result, however little the sums come to."""
    from engraft_ngram_amd import losses
    z, t, lp = exact_rows(n, v, 5)
    g = torch.Generator(device="cuda").manual_seed(6)
    seg = torch.arange(n, device=cuda) * 3 // n
    shift = torch.randn(n, generator=g, device=cuda).double() * 0.05
    old = (lp - shift).float()
    ref = (lp + torch.randn(n, generator=g, device=cuda).double() * 1e-3).float()
    ratio, diff = (lp - old.double()).exp(), ref.double() - lp
    w = torch.ones(n, dtype=torch.float64, device=cuda)
    if reduction == "token":
        w = w / n
    if reduction == "sequence":
        w = w / (3 * torch.bincount(seg, minlength=3)[seg])
    a = torch.randn(n, generator=g, device=cuda)
    kl = torch.expm1(diff) - diff
    a[-1] = 0.0  # the last row takes up the others' sum, but for its fp32 rounding
    a[-1] = (-(w * ratio * a.double()).sum() / (w[-1] * ratio[-1])).float()
    terms = w * ratio * a.double()
    kw = dict(ref_logprobs=ref, segment_ids=seg, n_segments=3, reduction=reduction, clip=(1.0, 1e6))
    for make_loss in (lambda: losses.policy_loss_grad(z, t, a, old, **kw)[0], lambda: losses.policy_loss(z, t, a, old, **kw)):
        res = make_loss()
        assert_within(res.loss, -terms.sum(), 2.0 ** -24 * terms.sum().abs() + 2.0 ** -44 * terms.abs().sum())
        assert_within(res.kl, (w * kl).sum(), 2.0 ** -24 * (w * kl).sum() + 2.0 ** -44 * (w * diff.abs()).sum())
        assert_within(res.logprobs, lp, 2.0 ** -23 * lp.abs())


@pytest.mark.parametrize("n,v", [(6, 20_011), (64, 1003), (300, 1003), (700, 1003)])
def test_margins_that_nearly_cancel(cuda, n, v):
    """Rows whose log-probabilities are exact, references within 1e-4 of the sums: margins and loss are off by the 64-bit
    sums' rounding and fp32's of the result."""
    from engraft_ngram_amd import losses
    z, t, lp = exact_rows(n, v, 7)
    seg = torch.arange(n, device=cuda) * 4 // n
    seqs = torch.stack([lp[seg == s].sum() for s in range(4)])
    ref = (seqs + torch.randn(4, generator=torch.Generator().manual_seed(1)).cuda().double() * 1e-4).float()
    gain = seqs - ref.double()
    h = 0.125 * (gain[0::2] - gain[1::2])
    want = -torch.nn.functional.logsigmoid(h).mean()
    for make_loss in (lambda: losses.preference_loss_grad(z, t, seg, ref, beta=0.125)[0],
                      lambda: losses.preference_loss(z, t, seg, ref, beta=0.125)):
        res = make_loss()
        assert_within(res.margins, h, 2.0 ** -24 * h.abs() + 2.0 ** -44 * seqs.abs().max())
        assert_within(res.loss, want, 2.0 ** -24 * want + 2.0 ** -44 * seqs.abs().max())
    assert_within(losses.token_logprobs(z, t), lp, 2.0 ** -23 * lp.abs())


@pytest.mark.parametrize("n,v,dtype", [(5, 151_936, torch.bfloat16), (600, 701, torch.float32), (520, 50_257, torch.float16),
                                       (520, 151_936, torch.bfloat16)])
def test_one_value_of_a_logprob(cuda, n, v, dtype):
    """Where rows are cut alike, the three calls give a row's log-probability the same bits: a policy's scores are the
    log-probabilities its loss then starts from."""
    from engraft_ngram_amd import losses
    z, t = make(n, v, dtype, 13)
    a, seg, ref = torch.ones(n, device=cuda), torch.arange(n, device=cuda) * 2 // n, torch.zeros(2, device=cuda)
    lp = losses.token_logprobs(z, t)
    for res in (losses.policy_loss_grad(z, t, a)[0], losses.policy_loss(z, t, a), losses.preference_loss_grad(z, t, seg, ref)[0],
                losses.preference_loss(z, t, seg, ref)):
        assert torch.equal(res.logprobs, lp)


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("n", [3, 70, 600])
def test_many_small_terms_beside_one(cuda, n, dtype):
    """A target at 0 among 151,935 logits of -17: each of their terms, 4.1e-8, is lost when it is added to the target's 1 alone.
    The sum (1.0063) is rounded where a thread adds a group of chunks (at most 10) and where threads and wavefronts
    are joined (at most 25 times in a row, 19 more over parts): 54 roundings of 2^-24."""
    from engraft_ngram_amd import losses
    v = 151_936
    z = torch.full((n, v), -17.0, dtype=dtype, device=cuda)
    t = torch.randint(0, v, (n,), generator=torch.Generator().manual_seed(n)).cuda()
    z[torch.arange(n, device=cuda), t] = 0.0
    want = -math.log1p((v - 1) * math.exp(-17.0))
    lp = losses.token_logprobs(z, t)
    assert float((lp.double() - want).abs().max()) <= 54 * 2.0 ** -24
    res, _ = losses.policy_loss_grad(z, t, torch.ones(n, device=cuda), out=z)
    assert float((res.logprobs.double() - want).abs().max()) <= 54 * 2.0 ** -24


@pytest.mark.parametrize("n,v", [(256, 20_011), (257, 20_011), (600, 701)])
def test_unordered_segments_have_no_sums(cuda, n, v):
    """Segments out of order: the sequences' sums are NaN like the margins, the same in every call; log-probabilities stay."""
    from engraft_ngram_amd import losses
    z, t = make(n, v, torch.bfloat16, n)
    lp = losses.preference_loss(z, t, torch.zeros_like(t), torch.zeros(2, device=cuda)).logprobs
    for seg in ((torch.arange(n, device=cuda) * 10 // n).flip(0), torch.arange(n, device=cuda) % 7):
        ref = torch.zeros(10, device=cuda)
        for res in (losses.preference_loss_grad(z, t, seg, ref)[0], losses.preference_loss(z, t, seg, ref)):
            assert res.sequence_logprobs.isnan().all() and res.margins.isnan().all() and res.loss.isnan()
            assert torch.equal(res.logprobs, lp)


@pytest.mark.parametrize("n", [1, 37, 256, 257])
@pytest.mark.parametrize("dtype", ALL)
def test_few_rows_against_autograd(cuda, n, dtype):
    """Few long rows: loss and gradient of the one call and of autograd have the same bits."""
    from engraft_ngram_amd import losses
    z, t = make(n, 20_011, dtype, n)
    gen = torch.Generator().manual_seed(n)
    a, old, ref = (torch.randn(n, generator=gen).cuda() for _ in range(3))
    seg = torch.arange(n, device=cuda) * 10 // n - 1  # -1 to 8, the last of no pair
    sums = torch.zeros(8, device=cuda)
    policy = dict(ref_logprobs=ref, segment_ids=seg.flip(0), n_segments=9, kl_coef=0.1, reduction="sequence")
    for grad, loss in ((lambda x: losses.policy_loss_grad(x, t, a, old, **policy), lambda x: losses.policy_loss(x, t, a, old, **policy)),
                       (lambda x: losses.preference_loss_grad(x, t, seg, sums), lambda x: losses.preference_loss(x, t, seg, sums))):
        res, d = grad(z)
        leaf = z.detach().requires_grad_()
        auto = loss(leaf)
        auto.loss.backward()
        assert torch.equal(leaf.grad, d) and not d.isnan().any()
        for x, y in zip(vars(res).values(), vars(auto).values()):
            assert torch.equal(x, y.detach())


@pytest.mark.parametrize("n,v,dtype", [(14_200, 151_936, torch.bfloat16), (43_000, 50_257, torch.float16),
                                       (540_000, 4001, torch.float16)])
def test_many_rows_past_32_bits(cuda, n, v, dtype):
    """More than 2^31 logits, in whole rows of every plan (held 20 and 8 chunks, not held): log-probabilities and the
    gradients of both losses of the last rows are those of the rows on their own."""
    from engraft_ngram_amd import losses
    tail = 40
    assert (n - tail) * v > 2 ** 31
    z = torch.zeros((n, v), dtype=dtype, device=cuda)
    t = torch.full((n,), -100, device=cuda)
    z[-tail:], t[-tail:] = make(tail, v, dtype, 3)
    a, seg = torch.randn(n, device=cuda), torch.zeros(n, dtype=torch.int64, device=cuda)
    seg[-tail // 2:] = 1
    few = z[-tail:].contiguous(), t[-tail:]
    assert_within(losses.token_logprobs(z, t)[-tail:], losses.token_logprobs(*few).double(), 2.0 ** -20)
    d = torch.empty_like(z)
    unit = {torch.bfloat16: 2.0 ** -7, torch.float16: 2.0 ** -10}[dtype]
    policy = dict(reduction="sum", grad_scale=1024.0)
    sums = torch.zeros(2, device=cuda)
    for all_rows, own in (
            (lambda: losses.policy_loss_grad(z, t, a, out=d, **policy), lambda: losses.policy_loss_grad(*few, a[-tail:], **policy)),
            (lambda: losses.preference_loss_grad(z, t, seg, sums, grad_scale=1024.0, out=d),
             lambda: losses.preference_loss_grad(*few, seg[-tail:], sums, grad_scale=1024.0))):
        d.fill_(7.0)
        all_rows()
        want = own()[1].double()
        # the rows' sums are taken in other orders: fp32's rounding of p, then the type's
        assert_within(d[-tail:], want, unit * want.abs() + 2.0 ** -23)
        assert not d[:-tail].any() and (want[few[1] >= 0].abs().amax(1) > 0).all()
