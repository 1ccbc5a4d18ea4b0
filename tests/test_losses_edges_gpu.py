"""Calls of the objectives over logits at the edges of what they accept, each
against its definition in 64 bits."""
import ctypes as C
import math

import pytest
import torch

from dop import losses
from dop._lib import DOP_BF16, DOP_F32, DopError, check as ok, lib
from test_losses_gpu import (BF16, F32, IDS, TYPES, U, UNEVEN, check, check_preference, demo, gen, last,
                             make_logits, onehot, preference_reference, teacher, tokens_of,
                             uneven_rows)

pytestmark = pytest.mark.gpu


# --------------------------------------------------------- no pairs at all
@pytest.mark.parametrize("rows,off", [(5, [2]), (1, [0]), (300, [300]), (0, [0])])
@pytest.mark.parametrize("grad", [True, False])
def test_preference_without_pairs(cuda, rows, off, grad):
    """0 pairs: the loss is 0 (here written over 7), and so is every row's
    part, whose logits are not read."""
    V = 33
    z = torch.full((rows, V), float("nan"), device="cuda")
    tokens = tokens_of(rows, V, 1)
    loss = torch.full((), 7.0, device="cuda")
    logp, lse, dlogp = (torch.full((rows,), 7.0, device="cuda") for _ in range(3))
    dz = torch.full((rows, V), 7.0, device="cuda")
    ok(lib().dop_preference_loss_grad(
        rows, V, DOP_F32, z.data_ptr(), V, tokens.data_ptr(), 0, (C.c_int64 * 1)(*off), None, None,
        1.0, 0.1, 0.0, 0, 1.0, loss.data_ptr(), None, None, logp.data_ptr(), lse.data_ptr(),
        dlogp.data_ptr(), DOP_F32, dz.data_ptr() if grad else None, V,
        torch.cuda.current_stream().cuda_stream))
    assert float(loss) == 0.0
    for t in (logp, lse, dlogp):
        assert (t == 0).all()
    assert (dz == (0.0 if grad else 7.0)).all()
    r = losses.preference_loss(z, tokens, off, grad=grad)
    assert float(r.loss) == 0.0 and r.pair_loss.shape == (0,)


# --------------------------------------------- the model's get and put, streams
def pool_of(t):
    """The stream that the allocator has t's memory for."""
    for s in torch.cuda.memory_snapshot():
        if s["address"] <= t.data_ptr() < s["address"] + s["total_size"]:
            return s["stream"]
    raise AssertionError("not the allocator's")


@pytest.mark.parametrize("precision", [DOP_F32, DOP_BF16], ids=["f32", "bf16"])
def test_model_on_another_stream(cuda, precision):
    """The get and the put on a stream that is not current, given or entered:
    the same bytes, in memory of that stream."""
    c, m, P, tokens, targets = demo(precision)
    want = m.forward(P, tokens)
    g = losses.token_logp_backward(want, targets, losses.token_logp(want, targets)[1],
                                   torch.ones(tokens.numel(), device="cuda"))
    grad = m.backward(P, tokens, g)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    z = m.forward(P, tokens, stream=side)
    d = m.backward(P, tokens, g, stream=side)
    with torch.cuda.stream(side):
        z2 = m.forward(P, tokens.view(2, -1))
        d2 = m.backward(P, tokens.view(2, -1), g)
    torch.cuda.synchronize()
    for a, b in ((z, want), (z2, want), (d, grad), (d2, grad)):
        assert torch.equal(a, b)
    assert [pool_of(t) for t in (z, d, z2, d2)] == [side.cuda_stream] * 4
    assert pool_of(want) == pool_of(grad) == torch.cuda.current_stream().cuda_stream
    m.close()


def test_model_operands(cuda):
    """Outputs and inputs of another type, size, layout or device are refused
    (tests/test_model_operands_cpu.py has each of them)."""
    c, m, P, tokens, targets = demo(DOP_F32)
    z = m.forward(P, tokens)
    for bad in (z.bfloat16(), z[:-1].clone(), z.cpu(), z.t()):
        with pytest.raises(DopError):
            m.forward(P, tokens, logits=bad)
        with pytest.raises(DopError):
            m.backward(P, tokens, bad)
    for bad in (P[:-1], P.bfloat16(), P.cpu()):
        with pytest.raises(DopError):
            m.backward(P, tokens, z, grad=bad)
        with pytest.raises(DopError):
            m.forward(bad, tokens)
    with pytest.raises(DopError):
        m.forward(P, tokens.int())
    assert m.forward(P, tokens, logits=z) is z
    m.close()


# ------------------------------------- rows whose maximum is large or far
# Elements of a row count by their distance from its maximum, which fp32 holds
# to 2^-24 of itself; one more than 150 ln 2 / below it has probability 0.
# With |t| <= 150 the power of two's argument c (z - m) is off by 2 u |t| (c
# rounded, and the product), so a probability's relative error is at most
#     150 * 2 ln 2 u + 8 u + (V / 128 + 64) u
# whatever the size of m (the last two as in test_losses_gpu).
def rel_near(vocab):
    return (150 * 2 * math.log(2) + 8 + vocab / 128 + 64) * U


LOG2E = 1.4426950408889634  # as a temperature: the power of two's factor is 1, |c m| is |m|
LARGE = [(3e6, LOG2E), (1.6e7, LOG2E), (2e7, LOG2E), (1.3e8, LOG2E), (3e8, LOG2E), (1e9, 1.0),
         (1e9, 0.1), (3e9, LOG2E), (6e9, 1.0), (1e10, 1.0), (1e12, 0.5), (1e15, 2.0), (1e20, 1.0),
         (1e30, 3.0), (1e38, 1.0), (1e38, 0.05), (1e5, 2.0 ** -16), (1e15, 2.0 ** 16)]


def large_rows(vocab, dtype, base, seed):
    """Rows around +-base: one value throughout, whole steps of the type below
    it, ordinary values with one entry there, and rows that are masked by it
    but for a few entries a little above it."""
    _, z = make_logits(6, vocab, dtype, 1, 0, seed=seed)
    b = float(torch.tensor(base).to(dtype))
    step = b * torch.finfo(dtype).eps
    k = torch.randint(0, 6, (2, vocab), generator=gen(seed + 1), device="cuda").double()
    z[0] = -b
    z[1] = (b - step * k[0]).to(dtype)
    z[2] = (-b - step * k[1]).to(dtype)
    z[3, vocab * 2 // 3] = b
    z[4] = -b
    z[4, vocab - 2] = -b / 2
    z[5] = b
    # a token of the largest value in every row
    tokens = z.double().argmax(1)
    return z, tokens


def from_maximum(z, tau):
    """x less its maximum, the maximum, log sum exp of the first, and p."""
    m = z.double().amax(1)
    t = (z.double() - m[:, None]) / tau
    l = torch.logsumexp(t, 1)
    return t, m / tau, l, torch.exp(t - l[:, None])




@pytest.mark.parametrize("vocab", [300, 9001, 300001])
@pytest.mark.parametrize("base,tau", LARGE)
@pytest.mark.parametrize("dtype,grad", TYPES, ids=IDS)
def test_large_rows(cuda, vocab, base, tau, dtype, grad):
    z, tokens = large_rows(vocab, dtype, base, 401)
    t, m, l, p = from_maximum(z, tau)
    rel, n = rel_near(vocab), z.shape[0]
    hot = onehot(tokens, vocab, torch.ones(n, dtype=torch.bool, device="cuda"))
    want = t.gather(1, tokens[:, None])[:, 0] - l
    logp, lse = losses.token_logp(z, tokens, temperature=tau)
    check("logp", logp, want, rel + last(want, F32))
    # c, rounded, stands for the temperature where the maximum is not far
    check("lse", lse, (m + l).float(), rel + 2 * last(m + l, F32))

    old, adv = (want - 0.1).float(), torch.tensor([1.0, -0.5, 0.7, 1.3, 2.0, -1.0], device="cuda")
    d = -adv.double() * torch.exp(want - old.double())
    r = losses.policy_loss(z, tokens, old, adv, temperature=tau, scale=0.5, clip_high=0.5, grad_dtype=grad)
    check("row_loss", r.row_loss, d, d.abs() * (rel + 8 * U) + last(d, F32))
    ref = 0.5 / tau * d[:, None] * (hot - p)
    tol = 0.5 / tau * d.abs()[:, None] * (2 * rel + 8 * U) * (p + hot)
    check("policy dlogits", r.dlogits, ref, tol + last(ref, grad))


@pytest.mark.parametrize("vocab", [300, 9001, 300001])
@pytest.mark.parametrize("base,tau", LARGE)
@pytest.mark.parametrize("dtype,grad", TYPES, ids=IDS)
@pytest.mark.parametrize("tail", [False, True], ids=["top", "tail"])
def test_distill_large_rows(cuda, vocab, base, tau, dtype, grad, tail):
    """The lists hold some of the entries that have a probability; in row 3
    an ordinary entry too, and in the last two rows one that the student has
    at -base and the teacher at probability 0."""
    z, tokens = large_rows(vocab, dtype, base, 411)
    z = torch.cat([z, z[3:5]])
    g = gen(412)
    z[6:] = torch.randn(2, vocab, generator=g, device="cuda").to(dtype)
    tokens = torch.cat([tokens, torch.tensor([3, 4], device="cuda")])
    low = torch.tensor([5, vocab - 1], device="cuda")
    z[6:].scatter_(1, low[:, None], -base)
    t, m, l, p = from_maximum(z, tau)
    n, K = z.shape[0], 6
    # up to four entries of probability, the row's first largest among them
    order = torch.topk(t - torch.rand(n, vocab, generator=g, device="cuda") * 1e-3, K, 1).indices
    order[:, 0] = tokens
    for i in range(1, K):  # an entry stands once
        order[:, i] = torch.where((order[:, :i] == order[:, i:i + 1]).any(1), torch.full_like(tokens, -1), order[:, i])
    order[6:, K - 1] = low
    top = torch.randn(n, K, generator=g, device="cuda") * tau
    at = order.clamp(min=0)
    here = order >= 0
    # what the student has not got, the teacher has not got either
    none = ~here | (t.gather(1, at) < -60.0)
    top = torch.where(none, torch.full_like(top, -math.inf), top)
    y = top.double() / tau
    tl = None
    if tail:
        tl = torch.logsumexp(y, 1).float() + 0.2
        # nothing but the listed entries has probability: none is left for the rest
        alone = torch.zeros(n, vocab, dtype=torch.bool, device="cuda").scatter_(1, at, here)
        rest = torch.logsumexp((t - l[:, None]).masked_fill(alone, -math.inf), 1)
        tl = torch.where(rest < -60.0, tl - 0.21, tl)
    lq = y - (torch.logsumexp(y, 1) if tl is None else tl.double())[:, None]
    q = torch.where(none, torch.zeros_like(lq), torch.exp(lq))
    lp = (t - l[:, None]).gather(1, at)
    zero = torch.zeros_like(lq)
    row = torch.where(none, zero, q * (torch.where(none, zero, lq) - torch.where(none, zero, lp))).sum(1)
    size = torch.where(none, zero, q * (1 + lq.abs().nan_to_num(0, 0, 0) + torch.where(none, zero, lp).abs())).sum(1)
    Q, share = q.sum(1), torch.zeros(n, dtype=torch.float64, device="cuda")
    if tail:
        qr = torch.clamp(1 - Q, min=0.0)
        some = qr > 0
        qr_ = torch.where(some, qr, torch.ones_like(qr))
        rest_ = torch.where(some, rest, torch.zeros_like(rest))
        row = row + torch.where(some, qr * (torch.log(qr_) - rest_), torch.zeros_like(qr))
        size = size + 1 + torch.where(some, rest_.abs(), torch.zeros_like(qr))
        share = torch.where(some, qr / torch.exp(rest_), share)
        Q = Q + qr
    member = torch.zeros(n, vocab, dtype=torch.bool, device="cuda").scatter_(1, at, here)
    ref = Q[:, None] * p - share[:, None] * torch.where(member, torch.zeros_like(p), p)
    qv = torch.zeros_like(p).scatter_add_(1, at, torch.where(here, q, zero))
    ref = tau * (ref - qv)
    rel = rel_near(vocab)
    r = losses.distill_loss(z, order.int().contiguous(), top, teacher_lse=tl, temperature=tau, scale=1.0,
                            grad_dtype=grad)
    check("row_loss", r.row_loss, tau * tau * row, tau * tau * size * (rel + 8 * U) + last(tau * tau * row, F32))
    tol = tau * (p * (2 * rel + 8 * U) * (Q[:, None] + share[:, None] * ~member) + 8 * U * qv)
    check("dlogits", r.dlogits, ref, tol + last(ref, grad))


@pytest.mark.parametrize("tail", [False, True], ids=["top", "tail"])
@pytest.mark.parametrize("whole", [0.0, 1.0, 2.0, 6.0])
def test_distill_between_the_forms(cuda, whole, tail):
    """Maxima of the listed entries and of the others on both sides of 2^24
    and a few steps apart."""
    V, B = 500, 2.0 ** 24
    _, z = make_logits(4, V, F32, seed=421)
    k = torch.randint(0, 8, (4, V), generator=gen(422), device="cuda").float()
    z[:] = (B - 4.0 + whole) - k
    index = torch.arange(4, dtype=torch.int32, device="cuda").repeat(4, 1).contiguous()
    z[0, :4] = B + 2.0
    z[1, :4] = B - 8.0
    z[2] *= -1.0
    z[3] = -z[3]
    z[3, :4] = -B + 6.0
    tau = LOG2E
    t, m, l, p = from_maximum(z, tau)
    top = torch.randn(4, 4, generator=gen(423), device="cuda")
    y = top.double() / tau
    tl = torch.logsumexp(y, 1).float() + 0.2 if tail else None
    lq = y - (torch.logsumexp(y, 1) if tl is None else tl.double())[:, None]
    q, lp = torch.exp(lq), (t - l[:, None])
    row, size = (q * (lq - lp[:, :4])).sum(1), (q * (1 + lq.abs() + lp[:, :4].abs())).sum(1)
    ref = p.clone()
    share = torch.zeros(4, 1, dtype=torch.float64, device="cuda")
    if tail:
        qr, rest = 1 - q.sum(1), torch.logsumexp(lp[:, 4:], 1)
        row, size = row + qr * (torch.log(qr) - rest), size + 1 + rest.abs()
        share = (qr / torch.exp(rest))[:, None]
        ref[:, 4:] -= share * p[:, 4:]
    ref[:, :4] -= q
    rel = rel_near(V)
    r = losses.distill_loss(z, index, top, teacher_lse=tl, temperature=tau, scale=1.0)
    check("row_loss", r.row_loss, tau * tau * row, tau * tau * size * (rel + 8 * U) + last(tau * tau * row, F32))
    tol = p * (2 * rel + 8 * U) * (1 + share) + 8 * U
    check("dlogits", r.dlogits, tau * ref, tau * tol + last(tau * ref, F32))


def test_far_rows_among_ordinary_ones_on_several_ctas(cuda):
    """Masks of -1e9, -1e10 and the lowest value over most of a row, over
    whole CTAs' shares and over the start, and a row masked altogether."""
    for dtype in (F32, BF16):
        for vocab in (1003, 40007, 300001):
            for low in (-1e9, -1e10, torch.finfo(dtype).min):
                _, z = make_logits(4, vocab, dtype, 1, 0, seed=431)
                z[0, : vocab // 2] = low
                z[1, vocab // 100:] = low
                z[2, ::2] = low
                z[3] = low
                tokens = torch.tensor([vocab - 1, 0, 1, vocab // 3], device="cuda")
                t, m, l, p = from_maximum(z, 1.0)
                want = t.gather(1, tokens[:, None])[:, 0] - l
                rel = rel_near(vocab)
                logp, lse = losses.token_logp(z, tokens)
                check("logp", logp, want, rel + last(want, F32))
                one = torch.ones(4, device="cuda")
                r = losses.policy_loss(z, tokens, want.float(), one, scale=1.0)
                hot = onehot(tokens, vocab, one > 0)
                ref = -torch.exp(want - want.float().double())[:, None] * (hot - p)
                check("dlogits", r.dlogits, ref, (2 * rel + 8 * U) * (p + hot) + last(ref, dtype))


# ------------------------------ adjoints where fp32 does not hold the row's lse
@pytest.mark.parametrize("vocab", [300, 9001, 300001])
@pytest.mark.parametrize("base,tau", [(5e3, 1.0), (1e5, 1.0), (50.0, 1e-3)] + LARGE)
@pytest.mark.parametrize("dtype,grad", TYPES, ids=IDS)
def test_logp_backward_large_rows(cuda, vocab, base, tau, dtype, grad):
    """p is the row's softmax whatever its lse: where that is above 4096 it
    does not come from the fp32 lse, of which 2^-24 would be an error of its
    own in p.  A far row with entries of -inf is among them."""
    z, tokens = large_rows(vocab, dtype, base, 441)
    z[2, 1::3] = -math.inf
    z[4, 3] = -math.inf
    tokens = z.double().argmax(1)
    t, m, l, p = from_maximum(z, tau)
    rel, n = rel_near(vocab), z.shape[0]
    logp, lse = losses.token_logp(z, tokens, temperature=tau)
    g = torch.tensor([1.0, -0.5, 0.7, 1.3, -2.0, 0.25], device="cuda")
    hot = onehot(tokens, vocab, g != 0)
    ref = (g.double() / tau)[:, None] * (hot - p)
    held = (m + l).abs() <= 4096
    tol = (g.double().abs() / tau)[:, None] * (
        (rel + U * torch.where(held, (m + l).abs(), torch.zeros_like(m)))[:, None] * p + 4 * U * (p + hot))
    # c stands for the temperature in p = 2^(c z - lse / ln 2) too: the lse is c's
    dz = losses.token_logp_backward(z, tokens, lse, g, temperature=tau, grad_dtype=grad)
    check("dlogits", dz, ref, tol + last(ref, grad))
    if grad is dtype:  # in the logits' own memory
        own = torch.empty(z.shape[0] * z.stride(0), dtype=dtype, device="cuda")
        own = own.view(z.shape[0], z.stride(0))[:, :vocab].copy_(z)
        losses.token_logp_backward(own, tokens, lse, g, temperature=tau, dlogits=own)
        assert torch.equal(own, dz)


@pytest.mark.parametrize("vocab", [300, 9001, 300001])
@pytest.mark.parametrize("base,tau", [(5e3, 1.0), (1e9, 1.0), (1e20, 1.0), (1e38, 0.05)])
@pytest.mark.parametrize("dtype,grad", TYPES, ids=IDS)
def test_preference_large_rows(cuda, vocab, base, tau, dtype, grad):
    z, tokens = large_rows(vocab, dtype, base, 451)
    t, m, l, p = from_maximum(z, tau)
    rel = rel_near(vocab)
    off, beta = [0, 2, 3, 4, 6], 0.3
    logp = t.gather(1, tokens[:, None])[:, 0] - l
    ref_logp = (logp + torch.randn(6, generator=gen(452), device="cuda")).float()
    dif = logp - ref_logp.double()
    margin = beta * torch.stack([dif[0:2].sum() - dif[2], dif[3] - dif[4:6].sum()])
    dm = -torch.sigmoid(-margin)
    d = beta * torch.stack([dm[0], dm[0], -dm[0], dm[1], -dm[1], -dm[1]])
    r = losses.preference_loss(z, tokens, off, ref_logp=ref_logp, temperature=tau, beta=beta, scale=1.0,
                               grad_dtype=grad)
    tol_m = beta * 3 * rel
    check("margin", r.margin, margin, tol_m + last(margin, F32))
    check("dlogp", r.dlogp, d, beta * (tol_m / 4 + 4 * U) + last(d, F32))
    hot = onehot(tokens, vocab, d != 0)
    ref = (d / tau)[:, None] * (hot - p)
    held = (m + l).abs() <= 4096
    tol = (beta * (tol_m / 4 + 4 * U) / tau) * (hot + p) + (d.abs() / tau)[:, None] * (
        (rel + U * torch.where(held, (m + l).abs(), torch.zeros_like(m)))[:, None] * p + 4 * U * (p + hot))
    check("dlogits", r.dlogits, ref, tol + last(ref, grad))


def test_logp_backward_rows_without_a_finite_logit(cuda):
    """They give NaN, and skipped ones 0, as in the forward."""
    z = torch.zeros(4, 50, device="cuda")
    z[0] = -math.inf
    z[1, 7] = math.inf
    z[2, 9] = math.nan
    tokens = torch.tensor([1, 7, 3, 4], device="cuda")
    logp, lse = losses.token_logp(z, tokens)
    assert torch.isnan(logp[:3]).all()
    dz = losses.token_logp_backward(z, tokens, lse, torch.tensor([1.0, 1.0, 1.0, 0.0], device="cuda"))
    assert torch.isnan(dz[:3]).all() and (dz[3] == 0).all()


# ------------------------------------------------- a policy row's scalars
@pytest.mark.parametrize("gap", [1e-4, 1e-3, 1e-2, 0.0])
@pytest.mark.parametrize("vocab", [97, 40007])
def test_policy_kl_of_small_gaps(cuda, gap, vocab):
    """KL alone (advantage 0): exp(gap) - gap - 1 is about gap^2 / 2, and
    moves by |expm1(gap)| times the log-probability's error e, and by e^2."""
    n, kl = 6, 0.25
    _, z = make_logits(n, vocab, F32, seed=501)
    tokens = tokens_of(n, vocab, 502)
    t, m, l, p = from_maximum(z, 1.0)
    lp = t.gather(1, tokens[:, None])[:, 0] - l
    # (beside the gap, what the fp32 ref_logp leaves: it is an input)
    sign = torch.tensor([1.0, -1.0, 1.0, -1.0, 0.5, -0.5], device="cuda")
    ref = (lp + gap * sign).float()
    g = ref.double() - lp
    want, d = kl * (torch.expm1(g) - g), -kl * torch.expm1(g)
    zero = torch.zeros(n, device="cuda")
    r = losses.policy_loss(z, tokens, lp.float(), zero, ref_logp=ref, kl_coef=kl, scale=1.0)
    # the log-probability's error, as in test_losses_gpu
    e = (float(z.abs().max()) * 2 + 8 + vocab / 128 + 64) * U
    check("row_loss", r.row_loss, want, kl * (torch.expm1(g).abs() * e + e * e) + last(want, F32))
    hot = onehot(tokens, vocab, zero == 0)
    check("dlogits", r.dlogits, d[:, None] * (hot - p),
          (kl * e + 8 * U * d.abs())[:, None] * (hot + p) + (d.abs() * 2 * e)[:, None] * p + last(d[:, None] * p, F32))


def test_policy_large_ratios(cuda):
    """A ratio beyond fp32 beside an advantage of 0, or under the clip, and a
    KL term whose exponential fp32 does not hold."""
    V = 40
    _, z = make_logits(4, V, F32, seed=511)
    tokens = tokens_of(4, V, 512)
    t, m, l, p = from_maximum(z, 1.0)
    lp = t.gather(1, tokens[:, None])[:, 0] - l
    old = (lp - torch.tensor([100.0, 200.0, 0.0, 95.0], device="cuda")).float()
    adv = torch.tensor([0.0, 2.0, 0.0, -1e-4], device="cuda")
    ref = (lp + torch.tensor([0.0, 0.0, 91.0, 0.0], device="cuda")).float()
    kl = 1e-3
    ratio, gap = torch.exp(lp - old.double()), ref.double() - lp
    inside = torch.tensor([1.0, 0.0, 1.0, 1.0], device="cuda")
    A = adv.double()
    want = -torch.where(inside > 0, ratio * A, 1.2 * A) + kl * (torch.expm1(gap) - gap)
    d = -A * ratio * inside - kl * torch.expm1(gap)
    r = losses.policy_loss(z, tokens, old, adv, ref_logp=ref, kl_coef=kl, scale=1.0)
    e = (float(z.abs().max()) * 2 + 8 + 64 + 1) * U
    small = kl * (torch.expm1(gap).abs() * e + e * e)
    check("row_loss", r.row_loss, want, (ratio * A).abs() * inside * (e + 4 * U) + small + last(want, F32) + 4 * U * A.abs())
    hot = onehot(tokens, V, inside >= 0)
    check("dlogits", r.dlogits, d[:, None] * (hot - p),
          (d.abs() * (3 * e + 8 * U) + kl * e)[:, None] * (hot + p) + last(d[:, None] * p, F32))


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("vocab", [64, 32768])
def test_policy_scalars_are_of_64_bits(cuda, dtype, vocab):
    """Rows of zeros, 2^k of them: every power and their sum are exact, so the
    log-probability -k ln 2 has 64 bits, and a row's loss is off by its own
    rounding to fp32 alone (2^-40 of the parts is far below that)."""
    gap = torch.tensor([1e-5, -1e-4, 1e-3, -1e-2, 0.3, -7.0, 1e-6, 0.0], device="cuda")
    n, kl = gap.numel(), 0.375
    z = torch.zeros(n, vocab, dtype=dtype, device="cuda")
    lp = -math.log(vocab)
    ref, old = lp + gap, lp - gap
    g, step = ref.double() - lp, lp - old.double()
    adv = torch.tensor([0.0, 0.0, 0.0, 0.0, 0.0, 0.0, 1.5, -0.75], device="cuda")
    r = losses.policy_loss(z, tokens_of(n, vocab, 521), old, adv, ref_logp=ref, kl_coef=kl, scale=1.0)
    A, ratio = adv.double(), torch.exp(step)
    want = -ratio * A + kl * (torch.expm1(g) - g)
    check("row_loss", r.row_loss, want, last(want, F32) + 2.0 ** -40 * (ratio * A).abs())
    d = -ratio * A - kl * torch.expm1(g)
    hot = (d * (1 - 1 / vocab)).float().double()
    got = r.dlogits.gather(1, tokens_of(n, vocab, 521)[:, None])[:, 0]
    # the coefficient and its product with p are rounded to fp32, and the sum
    # of the two at the token, each once; then to the type
    check("dlogits", got, hot, d.abs() * 4 * U + last(hot, dtype))


# ------------------------------------------------ masked entries of a teacher
@pytest.mark.parametrize("tail", [False, True], ids=["top", "tail"])
@pytest.mark.parametrize("tau", [0.25, 0.5, 1.0, 2.0])
@pytest.mark.parametrize("low", [torch.finfo(torch.float32).min, -1e30, -1e9, -1e4])
def test_distill_masked_teacher(cuda, tail, tau, low):
    """A teacher's logit at the type's lowest value, or otherwise masked, is
    one of probability 0: the same loss and adjoint as with -inf, and those
    bytes."""
    _, z = make_logits(5, 777, F32, seed=601)
    index, top, tlse = teacher(z, 12, tau, 602, tail)
    top[:, 4:9] = low
    top[4, :11] = low
    if tail:
        tlse = torch.logsumexp(top / tau, 1) + 0.1
    inf = torch.where(top == low, torch.full_like(top, -math.inf), top)
    a = losses.distill_loss(z, index, top, teacher_lse=tlse, temperature=tau)
    b = losses.distill_loss(z, index, inf, teacher_lse=tlse, temperature=tau)
    assert torch.isfinite(b.row_loss).all() and torch.isfinite(b.dlogits).all()
    for x, y in zip(a, b):
        assert torch.equal(x, y)


# ------------------------------------------- dlogits between the logits' rows
@pytest.mark.parametrize("dtype,grad", TYPES, ids=IDS)
@pytest.mark.parametrize("vocab,gap", [(7, 0), (1001, 3), (40007, 1)])
def test_dlogits_between_the_rows(cuda, dtype, grad, vocab, gap):
    """Logits and dlogits side by side in rows of one buffer, either first:
    nothing of one is written by the other."""
    rows = 4
    size, gsize = torch.finfo(dtype).bits // 8, torch.finfo(grad).bits // 8
    _, z = make_logits(rows, vocab, dtype, seed=701)
    tokens, f = tokens_of(rows, vocab, 702), torch.ones(rows, device="cuda")
    first = (vocab * size + gap * 4 + 3) // 4 * 4
    for a, b in ((0, first), ((vocab * gsize + gap * 4 + 3) // 4 * 4, 0)):
        width = (max(a + vocab * size, b + vocab * gsize) + gap + 3) // 4 * 4
        buf = torch.full((rows * width,), 0x5a, dtype=torch.uint8, device="cuda")
        zin = torch.as_strided(buf.view(dtype), (rows, vocab), (width // size, 1), a // size).copy_(z)
        out = torch.as_strided(buf.view(grad), (rows, vocab), (width // gsize, 1), b // gsize)
        r = losses.policy_loss(zin, tokens, f, f, scale=1.0, dlogits=out)
        assert torch.equal(zin, z)
        want = torch.empty(rows * (width // size), dtype=dtype, device="cuda")
        same = torch.as_strided(want, (rows, vocab), (width // size, 1), 0)  # rows at the same alignment
        if a % 16 == 0:
            same.copy_(z)
            assert torch.equal(losses.policy_loss(same, tokens, f, f, scale=1.0, grad_dtype=grad).dlogits, out)
        else:
            x = losses.policy_loss(z, tokens, f, f, scale=1.0, grad_dtype=grad).dlogits
            check("dlogits", out, x, x.double().abs() * (torch.finfo(grad).eps + 400 * U))
        rest = torch.as_strided(buf, (rows, width), (width, 1)).clone()
        rest[:, a:a + vocab * size] = 0x5a
        rest[:, b:b + vocab * gsize] = 0x5a
        assert (rest == 0x5a).all()


def test_one_row_in_place_under_two_strides(cuda):
    _, z = make_logits(3, 50, F32, 2, 0, seed=711)
    row, flat = z[1:2], z[1].unsqueeze(0)
    tokens, f = tokens_of(1, 50, 712), torch.ones(1, device="cuda")
    want = losses.policy_loss(row, tokens, f, f).dlogits
    losses.policy_loss(row, tokens, f, f, dlogits=torch.as_strided(flat, (1, 50), (50, 1)))
    check("dlogits", row, want, want.double().abs() * 400 * U)


# ------------------------- what the far rows' tests above do not put together
@pytest.mark.parametrize("vocab", UNEVEN)
@pytest.mark.parametrize("dtype,grad", TYPES, ids=IDS)
def test_preference_uneven_rows(cuda, vocab, dtype, grad):
    z = uneven_rows(vocab, dtype, 801)
    n = z.shape[0]
    tokens, off = tokens_of(n, vocab, 802), [0, 4, 9, 13, n]
    ref = -5.0 + torch.randn(n, generator=gen(803), device="cuda")
    e = preference_reference(z, tokens, off, ref, None, 1.0, 0.05, 0.1, False, 0.5)
    r = losses.preference_loss(z, tokens, off, ref_logp=ref, beta=0.05, label_smoothing=0.1, scale=0.5,
                               grad_dtype=grad)
    check_preference(r, e, 0.5, grad)


@pytest.mark.parametrize("low", [-1e10, -1e9, -3e7])
@pytest.mark.parametrize("vocab", [500, 40007, 300001])
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_distill_with_everything_outside_the_list_masked(cuda, low, vocab, dtype):
    """The student has its mass on the listed entries, at the start, in the
    middle and at the end; the others are masked to one far value, so a rest
    that the teacher holds there costs it their distance."""
    n, K = 4, 6
    _, z = make_logits(n, vocab, dtype, 1, 0, seed=811)
    index = torch.tensor([0, 1, vocab // 2, vocab // 2 + 1, vocab - 2, vocab - 1], device="cuda").repeat(n, 1)
    keep = z.gather(1, index)
    z[:] = low
    z.scatter_(1, index, keep)
    top = torch.randn(n, K, generator=gen(812), device="cuda")
    # a rest of 0 in the first two rows, of 0.2 in the others
    share = torch.tensor([0.0, 0.0, 0.2, 0.2], device="cuda")
    tl = torch.logsumexp(top, 1) - torch.log1p(-share) - 1e-3 * (share == 0)
    t, m, l, p = from_maximum(z, 1.0)
    lp, lq = (t - l[:, None]).gather(1, index), top.double() - tl.double()[:, None]
    q = torch.exp(lq)
    qr = torch.clamp(1 - q.sum(1), min=0.0)
    rest = t[:, 2] - l + math.log(vocab - K)
    row = (q * (lq - lp)).sum(1) + torch.where(qr > 0, qr * (torch.log(qr) - rest), torch.zeros_like(qr))
    size = (q * (1 + lq.abs() + lp.abs())).sum(1) + (qr > 0) * (1 + rest.abs())
    Q = q.sum(1) + qr
    ref = Q[:, None] * p - (qr / (vocab - K))[:, None]
    ref.scatter_(1, index, Q[:, None] * p.gather(1, index) - q)
    rel = rel_near(vocab)
    r = losses.distill_loss(z, index.int().contiguous(), top, teacher_lse=tl, scale=1.0)
    check("row_loss", r.row_loss, row, size * (rel + 8 * U) + last(row, F32))
    # the rest's q is 1 less a sum of q rounded to fp32
    tol = 2 * rel * Q[:, None] * p + ((qr * (2 * rel) + 8 * U) / (vocab - K))[:, None] + 8 * U * (ref.abs() + p)
    tol.scatter_add_(1, index, 8 * U * q)
    check("dlogits", r.dlogits, ref, tol + last(ref, dtype))


@pytest.mark.parametrize("dtype,grad,vocab", [(F32, F32, 851965), (F32, BF16, 851965), (BF16, BF16, 1703929)],
                         ids=IDS)
@pytest.mark.parametrize("base", [2e7, 1e10, -1e10])
def test_far_rows_of_the_largest_vocabulary(cuda, dtype, grad, vocab, base):
    _, z = make_logits(2, vocab, dtype, 2, 1, seed=821)
    b = float(torch.tensor(base).to(dtype))
    z[0] = b
    z[1, vocab // 3:] = b
    z[1, : vocab // 3] = b - abs(b) / 4
    tokens = torch.tensor([5, vocab - 1], device="cuda")
    t, m, l, p = from_maximum(z, 1.0)
    want, rel = t.gather(1, tokens[:, None])[:, 0] - l, rel_near(vocab)
    logp, lse = losses.token_logp(z, tokens)
    check("logp", logp, want, rel + last(want, F32))
    one = torch.ones(2, device="cuda")
    hot = onehot(tokens, vocab, one > 0)
    ratio = torch.exp(want - want.float().double())
    r = losses.policy_loss(z, tokens, want.float(), one, scale=1.0, grad_dtype=grad)
    ref = -ratio[:, None] * (hot - p)
    check("policy dlogits", r.dlogits, ref, (2 * rel + 8 * U) * (p + hot) + last(ref, grad))
    d = losses.token_logp_backward(z, tokens, lse, -one, grad_dtype=grad)
    check("dlogits", d, p - hot, (rel + 8 * U) * (p + hot) + last(p - hot, grad))
    # all of the teacher's mass on two entries of probability, and a third of it elsewhere
    index = torch.stack([tokens - 3, tokens], 1).int()
    for share in (0.0, 1 / 3):
        tl = torch.full((2,), math.log(2.0) - math.log1p(-share) - 1e-3 * (share == 0), device="cuda")
        r = losses.distill_loss(z, index, torch.zeros(2, 2, device="cuda"), teacher_lse=tl, scale=1.0, grad_dtype=grad)
        q = torch.exp(-tl.double())
        qr = torch.clamp(1 - 2 * q, min=0.0)
        rest = torch.log(1 - 2 * p.gather(1, tokens[:, None])[:, 0])
        row = 2 * q * (-tl.double() - want) + torch.where(qr > 0, qr * (torch.log(qr) - rest), torch.zeros_like(qr))
        check("row_loss", r.row_loss, row, (3 + 2 * want.abs()) * (rel + 8 * U) + last(row, F32))
