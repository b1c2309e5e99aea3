"""The losses of next-token logits (``losses``) against a plain float64
implementation: log-probabilities, loss terms and the gradient of the logits,
over types, odd vocabularies, row strides, masks and reductions; the gradient
against differences; autograd against the call that returns the gradient.

Tolerances.  With R the largest |z - max z| / temperature among the values that
count (p above 2^-30) or at the target, a log-probability's error is that of the
exponents' rounding (2^-23 R), of 2^x and ln (2^-22 each), and of a sum of
at most a few hundred fp32 terms a thread (random signs: below 2^-21): E = 2^-22
(8 + R) in all.  p_j has the relative error 2 E; the coefficient g adds its own
terms' (2 E relative to the terms without cancellation); the type adds half a
unit in the last place."""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def memory_returned():
    """What torch's allocator keeps of these tests' tensors goes back: other tests read its statistics."""
    yield
    import gc

    import torch
    gc.collect()
    torch.cuda.empty_cache()

EPS = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -24}
ALL = [torch.float32, torch.bfloat16, torch.float16]
SIZES = [(1, 1), (1, 7), (3, 8), (5, 1003), (4, 4096), (600, 129), (2, 50_257), (3, 151_936), (530, 40_001),
         (515, 50_257), (513, 163_841)]


def make(n, v, dtype, seed, pad=0, offset=0, ignored=0.3, int32=False):
    """Logits [n, v] in a wider buffer (row stride v + pad, first element at
    `offset`) whose every other value is NaN, and targets with rows left out."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    buf = torch.full((n * (v + pad) + offset,), math.nan, dtype=dtype, device="cuda")
    z = buf[offset:].view(n, v + pad)[:, :v]
    z.copy_(torch.randn((n, v), generator=g, device="cuda") * 3.0)
    t = torch.randint(0, v, (n,), generator=g, device="cuda")
    z[torch.arange(n, device="cuda"), t] += 4.0
    out = torch.rand(n, generator=g, device="cuda") < ignored
    t[out] = -100
    z[out] = math.nan  # never read
    return z, (t.int() if int32 else t)


def plain(z, t, temperature):
    """float64 log-probabilities, softmax and R of the rows with a target."""
    y = torch.where((t >= 0)[:, None], z.double(), 0.0) / temperature
    logp = torch.log_softmax(y, 1)
    lp = torch.where(t >= 0, logp.gather(1, t.long().clamp_min(0)[:, None])[:, 0], 0.0)
    top = y.amax(1, keepdim=True)
    r = torch.where(logp.exp() > 2.0 ** -30, top - y, 0.0).amax(1)
    r = torch.maximum(r, (top - y).gather(1, t.long().clamp_min(0)[:, None])[:, 0])
    return lp, logp.exp(), r


def lp_error(r):
    return 2.0 ** -22 * (8.0 + r)


def assert_within(got, want, tol):
    bad = ~((got.double() - want).abs() <= tol)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off; largest {float((got.double() - want).abs().max())}"


def check_gradient(d, t, p, r, g, g_size, temperature, scale=1.0):
    """d against scale * g ([j == t] - p) / temperature; g_size: g's terms without cancellation."""
    one = torch.zeros_like(p)
    valid = t >= 0
    one[valid, t[valid].long()] = 1.0
    k = (scale / temperature) * torch.where(valid, g, 0.0)[:, None]
    size = (scale / temperature) * torch.where(valid, g_size, 0.0)[:, None]
    want = k * (one - p)
    e = 2.0 * lp_error(r)[:, None]
    tol = size * e * (p + one) * 2.0 + EPS[d.dtype] * want.abs() + TINY[d.dtype]
    assert_within(d, want, tol)
    assert (d[~valid] == 0).all()


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("n,v", SIZES)
def test_token_logprobs(cuda, n, v, dtype):
    from engraft_ngram_amd import losses
    for temperature, pad, offset, int32 in ((1.0, 0, 0, False), (0.6, 3, 1, True)):
        z, t = make(n, v, dtype, n + v, pad, offset, int32=int32)
        lp = losses.token_logprobs(z, t, temperature=temperature)
        want, _, r = plain(z, t, temperature)
        assert lp.dtype == torch.float32 and lp.shape == (n,)
        assert_within(lp, want, lp_error(r))
        assert torch.equal(lp, losses.token_logprobs(z, t, temperature=temperature))


def policy_inputs(n, lp, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    a = torch.randn(n, generator=g, device="cuda")
    shift = torch.randn(n, generator=g, device="cuda") * 0.3
    for edge in (math.log(0.8), math.log(1.3)):  # not within rounding of an edge
        shift = torch.where((shift - edge).abs() < 1e-3, shift + 2e-3, shift)
    return a, (lp - shift).float(), (lp + torch.randn(n, generator=g, device="cuda") * 0.4).float()


@pytest.mark.parametrize("reduction", ["sum", "token", "sequence"])
@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("n,v", SIZES)
def test_policy_loss(cuda, n, v, dtype, reduction):
    from engraft_ngram_amd import losses
    temperature, pad, offset = ((1.0, 0, 0), (0.7, 5, 3))[(n + v) % 2]
    z, t = make(n, v, dtype, 3 * n + v, pad, offset, int32=n % 2 == 1)
    lp, p, r = plain(z, t, temperature)
    a, old, ref = policy_inputs(n, lp, n)
    seg = torch.randint(-1, 6, (n,), generator=torch.Generator().manual_seed(n)).cuda()  # any order, some of none
    beta, scale = 0.1, 8.0
    valid = t >= 0
    w = valid.double()
    if reduction == "token":
        w = w / max(1, int(valid.sum()))
    if reduction == "sequence":
        w = w * ((seg >= 0) & (seg < 5))
        each = torch.stack([w[seg == s].sum() for s in range(5)])
        w = w / (each.clamp_min(1.0) * max(1, int((each > 0).sum())))[seg.clamp(0, 4)]
    ratio = (lp - old.double()).exp()
    free, held = ratio * a, ratio.clamp(0.8, 1.3) * a
    diff = ref.double() - lp
    kl = torch.expm1(diff) - diff
    terms = w * (beta * kl - torch.minimum(free, held))
    g = w * (-torch.where(free <= held, free, 0.0) - beta * torch.expm1(diff))
    size = w * (ratio * a.abs() + beta * (1.0 + diff.exp()))
    e = lp_error(r)
    res, d = losses.policy_loss_grad(z, t, a, old, ref_logprobs=ref, segment_ids=seg, n_segments=5, clip=(0.2, 0.3),
                                     kl_coef=beta, temperature=temperature, reduction=reduction, grad_scale=scale)
    assert_within(res.logprobs, lp, e)
    assert_within(res.loss, terms.sum(), 2 ** -23 * terms.sum().abs() + (2.0 * e * (size + w)).sum())
    assert_within(res.kl, (w * kl).sum(), 2 ** -22 * (w * kl).sum() + (2.0 * e * w * (1.0 + diff.exp())).sum())
    assert_within(res.clip_fraction, (w * (free > held)).sum(), 1e-6 * (1.0 + (w * (free > held)).sum()))
    check_gradient(d, t, p, r, g, size, temperature, scale)
    # autograd: the same loss, the same gradient at the same scale
    leaf = z.detach().requires_grad_()
    auto = losses.policy_loss(leaf, t, a, old, ref_logprobs=ref, segment_ids=seg, n_segments=5, clip=(0.2, 0.3),
                              kl_coef=beta, temperature=temperature, reduction=reduction)
    (auto.loss * scale).backward()
    assert torch.equal(auto.loss.detach(), res.loss) and torch.equal(leaf.grad, d)
    # in place of the logits
    same = torch.empty_strided(z.shape, (v + pad, 1), dtype=dtype, device="cuda").copy_(z)
    res2, d2 = losses.policy_loss_grad(same, t, a, old, ref_logprobs=ref, segment_ids=seg, n_segments=5,
                                       clip=(0.2, 0.3), kl_coef=beta, temperature=temperature, reduction=reduction,
                                       grad_scale=scale, out=same)
    assert d2 is same and torch.equal(d2, d) and torch.equal(res2.loss, res.loss)


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("n,v", SIZES)
def test_preference_loss(cuda, n, v, dtype):
    from engraft_ngram_amd import losses
    pairs, beta, eps, scale = 1 + n // 200, 0.3, 0.1, 16.0
    temperature, pad, offset = ((0.8, 0, 0), (1.0, 1, 1))[v % 2]
    z, t = make(n, v, dtype, 5 * n + v, pad, offset)
    lp, p, r = plain(z, t, temperature)
    gen = torch.Generator().manual_seed(n)
    seg = torch.sort(torch.randint(0, 2 * pairs + 1, (n,), generator=gen)).values.cuda()  # the last id: of no pair
    seg = seg.int() if n % 2 else seg
    seqs = torch.stack([lp[seg == s].sum() for s in range(2 * pairs)])
    ref = (seqs.cpu() + torch.randn(2 * pairs, generator=gen, dtype=torch.float64) * 3.0).float().cuda()
    gain = seqs - ref.double()
    h = beta * (gain[0::2] - gain[1::2])
    want = -((1 - eps) * torch.nn.functional.logsigmoid(h) + eps * torch.nn.functional.logsigmoid(-h)).mean()
    g_h = (eps * torch.sigmoid(h) - (1 - eps) * torch.sigmoid(-h)) / pairs
    g_seq = torch.stack([beta * g_h, -beta * g_h], 1).reshape(-1)
    inside = (seg >= 0) & (seg < 2 * pairs) & (t >= 0)
    g = torch.where(inside, g_seq[seg.long().clamp(0, 2 * pairs - 1)], 0.0)
    e = lp_error(r)
    e_seq = torch.stack([e[seg == s].sum() for s in range(2 * pairs)])
    e_h = beta * (e_seq[0::2] + e_seq[1::2])
    res, d = losses.preference_loss_grad(z, t, seg, ref, beta=beta, label_smoothing=eps, temperature=temperature,
                                         grad_scale=scale)
    assert_within(res.logprobs, lp, e)
    assert_within(res.sequence_logprobs, seqs, e_seq + 2 ** -23 * seqs.abs())
    assert_within(res.margins, h, e_h + 2 ** -23 * h.abs())
    assert_within(res.loss, want, e_h.mean() + 2 ** -23 * want)
    # g carries the margin's error (|dg / dh| <= beta / (4 pairs)) besides a row's own
    err = beta / (4 * pairs) * e_h.max() + 2 ** -22 * g.abs()
    check_gradient(d, t, p, r, g, g.abs() + err / lp_error(r), temperature, scale)
    leaf = z.detach().requires_grad_()
    auto = losses.preference_loss(leaf, t, seg, ref, beta=beta, label_smoothing=eps, temperature=temperature)
    (auto.loss * scale).backward()
    assert torch.equal(auto.loss.detach(), res.loss) and torch.equal(leaf.grad, d)
    assert torch.equal(auto.margins, res.margins)


def test_masked_vocabulary_and_extreme_rows(cuda):
    """-inf columns get exact zeros; a row at the type's lowest value is uniform;
    an overwhelming logit gives 0 and 1; a row of -inf alone, a NaN and a target out of
    range give NaN in their own row only."""
    from engraft_ngram_amd import losses
    for dtype in ALL:
        v = 1001
        z, t = make(7, v, dtype, 1, ignored=0.0)
        z[:, 900:] = -math.inf
        t.clamp_max_(899)
        z[1] = torch.finfo(dtype).min
        z[2] = -1.0
        z[2, 5] = 300.0
        t[2] = 5
        z[3] = -math.inf
        z[4, 17] = math.nan
        t[5] = v
        a = torch.ones(7, device="cuda")
        res, d = losses.policy_loss_grad(z, t, a, reduction="sum")
        assert_within(res.logprobs[:1], plain(z[:1], t[:1], 1.0)[0], 2.0 ** -17)
        assert (d[0, 900:] == 0).all() and (d[6, 900:] == 0).all() and d[0, :900].isfinite().all()
        assert abs(float(res.logprobs[1]) + math.log(v)) < 1e-5
        assert float(res.logprobs[2]) == 0.0 and (d[2] == 0).all()
        for i in (3, 4, 5):
            assert math.isnan(float(res.logprobs[i])) and d[i].isnan().all()
        assert d[6].isfinite().all() and math.isnan(float(res.loss))


def test_nothing_to_learn_from(cuda):
    """No row with a target: a loss of 0 (log 2 for a pair), all-zero gradients, no NaN; no rows at all."""
    from engraft_ngram_amd import losses
    z = torch.full((4, 33), math.nan, device="cuda", dtype=torch.bfloat16)
    t = torch.full((4,), -100, device="cuda")
    zero, seg = torch.zeros(4, device="cuda"), torch.zeros(4, dtype=torch.int64, device="cuda")
    for reduction in ("sum", "token", "sequence"):
        res, d = losses.policy_loss_grad(z, t, zero, zero, ref_logprobs=zero, kl_coef=0.1, segment_ids=seg,
                                         n_segments=3, reduction=reduction)
        assert float(res.loss) == 0.0 and float(res.kl) == 0.0 and (d == 0).all() and (res.logprobs == 0).all()
    res, d = losses.preference_loss_grad(z, t, seg, torch.zeros(2, device="cuda"))
    assert abs(float(res.loss) - math.log(2.0)) < 1e-6 and (d == 0).all() and (res.sequence_logprobs == 0).all()
    none = z[:0]
    empty, no = torch.zeros(0, device="cuda"), torch.zeros(0, dtype=torch.int64, device="cuda")
    res, d = losses.policy_loss_grad(none, no, empty)
    assert float(res.loss) == 0.0 and d.shape == (0, 33) and losses.token_logprobs(none, no).numel() == 0
    res, d = losses.preference_loss_grad(none, no, no, torch.zeros(4, device="cuda"))
    assert abs(float(res.loss) - math.log(2.0)) < 1e-6 and (res.margins == 0).all()


def test_optional_terms(cuda):
    """Without old log-probabilities the ratio is 1 and its gradient stays; without a reference there is no KL
    term, also where the target's logit is -inf."""
    from engraft_ngram_amd import losses
    z, t = make(9, 77, torch.float32, 4, ignored=0.2)
    a = torch.randn(9, device="cuda")
    lp, p, r = plain(z, t, 1.0)
    res, d = losses.policy_loss_grad(z, t, a, reduction="sum")
    valid = (t >= 0).double()
    assert_within(res.loss, -(valid * a).sum(), 1e-6)
    assert float(res.kl) == 0.0 and float(res.clip_fraction) == 0.0
    check_gradient(d, t, p, r, -valid * a.double(), valid * a.abs().double(), 1.0)
    z[t >= 0, t[t >= 0]] = -math.inf
    res, d = losses.policy_loss_grad(z, t, a, torch.full((9,), -3.0, device="cuda"), reduction="sum")
    assert float(res.kl) == 0.0 and not d.isnan().any()


@pytest.mark.parametrize("which", ["policy", "preference"])
def test_gradient_against_differences(cuda, which):
    """Along random directions u: (L(z + h u) - L(z - h u)) / 2h against <d, u>.  The losses' third derivatives
    along u (|u_j| about 1, 13 rows) stay below 100; with h = 2^-6 the remainder is below h^2 100 / 6 = 4e-3 of it,
    and fp32's rounding of L (about 20) adds 2^-23 20 / h = 1.5e-4."""
    from engraft_ngram_amd import losses
    z, t = make(13, 19, torch.float32, 11)
    z = torch.where((t >= 0)[:, None], z, 0.0)
    lp = plain(z, t, 1.0)[0]
    a, old, ref = policy_inputs(13, lp, 5)
    seg = torch.arange(13, device="cuda") // 3

    def value(x):
        if which == "policy":
            return losses.policy_loss_grad(x, t, a, old, ref_logprobs=ref, kl_coef=0.2, clip=(0.9, 9.0), reduction="sum")
        return losses.preference_loss_grad(x, t, seg, torch.zeros(4, device="cuda"), beta=0.2, label_smoothing=0.1)

    d = value(z)[1].double()
    g = torch.Generator(device="cuda").manual_seed(3)
    h = 2.0 ** -6
    for _ in range(5):
        u = torch.randn(z.shape, generator=g, device="cuda")
        slope = (float(value(z + h * u)[0].loss) - float(value(z - h * u)[0].loss)) / (2 * h)
        assert abs(slope - float((d * u).sum())) < 4e-3 + 2e-4


def test_unordered_segments_give_nan(cuda):
    from engraft_ngram_amd import losses
    z, t = make(6, 50, torch.float32, 2, ignored=0.0)
    seg = torch.tensor([0, 0, 1, 0, 1, 1], device="cuda")
    res, d = losses.preference_loss_grad(z, t, seg, torch.zeros(2, device="cuda"))
    assert math.isnan(float(res.loss)) and d.isnan().all() and res.margins.isnan().all()


def test_other_stream_and_repeats(cuda):
    """The call runs on the current stream, gives the same bits again, and keeps nothing between calls."""
    from engraft_ngram_amd import losses
    z, t = make(300, 5003, torch.bfloat16, 8)
    seg = torch.arange(300, device="cuda") // 60
    ref = torch.zeros(4, device="cuda")
    first, d = losses.preference_loss_grad(z, t, seg, ref)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other, d2 = losses.preference_loss_grad(z, t, seg, ref)
        z2 = z + 1.0
        third, d3 = losses.preference_loss_grad(z2, t, seg, ref)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(first.loss, other.loss) and torch.equal(d, d2) and torch.equal(first.logprobs, other.logprobs)
    assert not torch.equal(d2, d3)


def test_in_a_graph(cuda):
    """A captured call replays on the values its inputs then hold."""
    from engraft_ngram_amd import losses
    z, t = make(40, 3001, torch.bfloat16, 9)
    a = torch.randn(40, device="cuda")
    lp = losses.token_logprobs(z, t)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        losses.policy_loss_grad(z, t, a, lp, ref_logprobs=lp, kl_coef=0.1)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res, d = losses.policy_loss_grad(z, t, a, lp, ref_logprobs=lp, kl_coef=0.1)
    for k in range(4):
        z.copy_(make(40, 3001, torch.bfloat16, 20 + k)[0].nan_to_num(0.0))
        want, dw = losses.policy_loss_grad(z, t, a, lp, ref_logprobs=lp, kl_coef=0.1)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(res.loss, want.loss) and torch.equal(d, dw) and torch.equal(res.logprobs, want.logprobs)


@pytest.mark.parametrize("n,v", [(12, 700), (40, 151_936), (600, 3001)])
def test_preference_in_place(cuda, n, v):
    """The gradient over the logits: the bits of the gradient beside them, in parts and whole rows."""
    from engraft_ngram_amd import losses
    z, t = make(n, v, torch.bfloat16, n)
    seg = torch.arange(n, device="cuda") * 4 // n
    ref = torch.zeros(4, device="cuda")
    res, d = losses.preference_loss_grad(z, t, seg, ref)
    version = z._version
    res2, d2 = losses.preference_loss_grad(z, t, seg, ref, out=z)
    assert d2 is z and torch.equal(d2, d) and torch.equal(res2.loss, res.loss) and z._version > version


def test_offsets_past_32_bits(cuda):
    """More than 2^31 logits: the last rows as on their own, in every kernel that many rows take."""
    from engraft_ngram_amd import losses
    n, v, tail = 14_200, 151_936, 40
    assert (n - tail) * v > 2 ** 31
    z = torch.zeros((n, v), dtype=torch.bfloat16, device="cuda")
    t = torch.full((n,), -100, device="cuda")
    z[-tail:], t[-tail:] = make(tail, v, torch.bfloat16, 3)
    a = torch.randn(n, device="cuda")
    lp = losses.token_logprobs(z, t)
    want = losses.token_logprobs(z[-tail:].contiguous(), t[-tail:])
    assert_within(lp[-tail:], want.double(), 2.0 ** -20)
    assert (lp[:-tail] == 0).all()
    d = torch.full_like(z, 7.0)
    res, _ = losses.policy_loss_grad(z, t, a, reduction="sum", out=d)
    few, d_few = losses.policy_loss_grad(z[-tail:].contiguous(), t[-tail:], a[-tail:], reduction="sum")
    # the two take their rows' sums in other orders: fp32's rounding of p, then bf16's
    assert_within(d[-tail:], d_few.double(), 2.0 ** -7 * d_few.double().abs() + 2.0 ** -60)
    assert (d[:-tail] == 0).all()
    d.fill_(7.0)
    seg = torch.zeros(n, dtype=torch.int64, device="cuda")
    seg[-tail // 2:] = 1
    losses.preference_loss_grad(z, t, seg, torch.zeros(2, device="cuda"), out=d)
    assert (d[:-tail] == 0).all() and (d[-tail:][t[-tail:] >= 0].abs().sum(1) > 0).all()


@pytest.mark.parametrize("n", [1, 2, 37, 256, 257])
@pytest.mark.parametrize("dtype", ALL)
def test_few_rows_against_in_place(cuda, n, dtype):
    """Few long rows find what they need of the loss in the gradient's launch, unless the gradient replaces
    the logits: the same bits either way, and autograd's."""
    from engraft_ngram_amd import losses
    v = 20_011
    z, t = make(n, v, dtype, n)
    gen = torch.Generator().manual_seed(n)
    a, old, ref = (torch.randn(n, generator=gen).cuda() for _ in range(3))
    seg = torch.arange(n, device="cuda") * 10 // n - 1  # -1 to 8, the last of no pair
    unordered = seg.flip(0) if n > 2 else seg

    def policy(z, count, **kw):
        return losses.policy_loss_grad(z, t, a, old, ref_logprobs=ref, segment_ids=unordered, n_segments=count,
                                       kl_coef=0.1, reduction="sequence", **kw)

    def preference(z, ids, **kw):
        return losses.preference_loss_grad(z, t, ids, torch.zeros(8, device="cuda"), **kw)

    for f, arg in ((policy, 9), (policy, 3000), (preference, seg), (preference, unordered)):
        res, d = f(z, arg)
        same = z.clone()
        res2, d2 = f(same, arg, out=same)
        assert torch.equal(d.isnan(), d2.isnan()) and torch.equal(d.nan_to_num(), d2.nan_to_num())
        for x, y in zip(vars(res).values(), vars(res2).values()):
            assert torch.equal(x.isnan(), y.isnan()) and torch.equal(x.nan_to_num(), y.nan_to_num())
        if n > 2 and arg is unordered:
            rows = (unordered >= 0) & (unordered < 8) & (t >= 0)
            assert res.loss.isnan() and d[rows].isnan().all() and not d[~rows].any()
