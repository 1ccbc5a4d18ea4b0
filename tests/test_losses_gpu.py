"""The objectives over logits (dop.losses) against their definitions in 64
bits on the same inputs, at the sizes, strides and masks where they can go
wrong, and together with the model lens.

Error bounds, elementwise, from the arithmetic the kernels document.  With
u = 2^-24 (half a step of fp32) and X the largest |c z| of the row (c =
log2(e) / tau), a probability 2^(c z - b) / s has relative error at most

    rel = X (2 ln 2) u   the rounded c, and the rounding of c z - b
        + 8 u            2^x (2^-22) and its counterpart in s
        + (V / 128 + 64) u   the fp32 sum: a thread adds at most V / 128
                             terms (128 threads or more share a row), the
                             rest is a tree and its rescalings
and log p has that absolute error, plus u |log p| where it is stored in
fp32.  The bounds below carry rel through each formula, and the last
rounding of an output is finfo.eps / 2 of its type."""
import math

import pytest
import torch

from dop import losses
from dop._lib import DOP_BF16, DOP_F32, DopError, lib

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F32, BF16 = torch.float32, torch.bfloat16
TYPES = [(F32, F32), (F32, BF16), (BF16, BF16)]
IDS = ["f32", "f32-bf16", "bf16"]


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def make_logits(rows, vocab, dtype, pad=0, shift=0, seed=0, std=2.5):
    """[rows, vocab] inside a buffer filled with NaN: `pad` elements between
    the rows and `shift` ahead of the first."""
    ld = vocab + pad
    buf = torch.full((shift + rows * ld + 8,), float("nan"), dtype=dtype, device="cuda")
    z = buf[shift: shift + rows * ld].view(rows, ld)[:, :vocab]
    z.copy_((torch.randn(rows, vocab, generator=gen(seed), device="cuda") * std).to(dtype))
    return buf, z


def rel_of(z, tau):
    x = z.double().abs()
    x = torch.where(torch.isfinite(x) & (x < 1e30), x, torch.zeros_like(x)).amax(1) if z.numel() else x.sum(1)
    return x / tau / math.log(2) * 2 * math.log(2) * U + (8 + z.shape[1] / 128 + 64) * U


def check(name, got, ref, tol):
    got, ref = got.double(), ref.double()
    tol = torch.as_tensor(tol, dtype=torch.float64, device=ref.device).expand_as(ref)
    same = (got == ref) | (torch.isnan(got) & torch.isnan(ref))
    off = torch.where(same, torch.zeros_like(ref), (got - ref).abs())
    bad = ~(off <= tol + 1e-37)
    assert not bad.any(), (name, int(bad.sum()), off[bad][:4].tolist(), tol[bad][:4].tolist(),
                           bad.nonzero()[:4].tolist())


def last(ref, dtype):
    return ref.double().abs() * torch.finfo(dtype).eps / 2


def softmax64(z, tau, live):
    """(x, lse, p) in 64 bits, rows that are not live replaced by zeros."""
    x = torch.where(live[:, None], z.double() / tau, torch.zeros((), dtype=torch.float64, device="cuda"))
    return x, torch.logsumexp(x, 1), torch.softmax(x, 1)


def logp64(x, tokens):
    """log softmax(x) at the tokens: the maximum leaves first, so that a row
    of the type's lowest value keeps its digits."""
    return torch.log_softmax(x, 1).gather(1, tokens[:, None])[:, 0]


def live_rows(tokens, weight, vocab):
    live = (tokens >= 0) & (tokens < vocab)
    return live if weight is None else live & (weight != 0)


def onehot(tokens, vocab, live):
    h = torch.zeros(tokens.numel(), vocab, dtype=torch.float64, device="cuda")
    rows = live.nonzero()[:, 0]
    h[rows, tokens[rows]] = 1.0
    return h


# ------------------------------------------------------------------ inputs
SHAPES = [(1, 1), (3, 2), (5, 7), (1, 31), (4, 32), (2, 255), (3, 1000), (7, 4097), (2, 32000),
          (1, 50001), (3, 131073), (500, 17), (450, 9001), (450, 20011), (446, 33003), (1, 700001)]
LAYOUT = [(0, 0), (3, 1), (16, 0)]


def tokens_of(rows, vocab, seed):
    return torch.randint(0, vocab, (rows,), generator=gen(seed), device="cuda")


def weights_of(rows, seed):
    w = torch.rand(rows, generator=gen(seed), device="cuda") + 0.5
    w[1::3] = 0.0
    return w


def check_logp(z, tokens, weight, tau, logp, lse):
    live = live_rows(tokens, weight, z.shape[1])
    x, l, _ = softmax64(z, tau, live)
    rel = rel_of(torch.where(live[:, None], z.double(), torch.zeros_like(x)), tau)
    t = torch.where(live, tokens, torch.zeros_like(tokens))
    ref = logp64(x, t)
    zero = torch.zeros_like(ref)
    ref, l = torch.where(live, ref, zero), torch.where(live, l, zero)
    check("logp", logp, ref, torch.where(live, rel + last(ref, F32), zero))
    check("lse", lse, l, torch.where(live, rel + last(l, F32), zero))
    return ref, l


# ------------------------------------------------------ log-probabilities
@pytest.mark.parametrize("rows,vocab", SHAPES)
@pytest.mark.parametrize("pad,shift", LAYOUT)
@pytest.mark.parametrize("dtype,grad", TYPES, ids=IDS)
def test_token_logp(cuda, rows, vocab, pad, shift, dtype, grad):
    buf, z = make_logits(rows, vocab, dtype, pad, shift, seed=vocab)
    tokens, weight, tau = tokens_of(rows, vocab, 1), weights_of(rows, 2), 0.7
    for w in (None, weight):
        logp, lse = losses.token_logp(z, tokens, weight=w, temperature=tau)
        check_logp(z, tokens, w, tau, logp, lse)
    dlogp = torch.randn(rows, generator=gen(3), device="cuda")
    dlogp[::4] = 0.0
    logp, lse = losses.token_logp(z, tokens, temperature=tau)
    # dlogits inside a buffer of its own layout: what lies between stays
    out = torch.full((rows, vocab + 5), 7.0, dtype=grad, device="cuda")
    dz = losses.token_logp_backward(z, tokens, lse, dlogp, temperature=tau, dlogits=out[:, :vocab])
    live = live_rows(tokens, dlogp, vocab)
    x, l64, p = softmax64(z, tau, live)
    hot = onehot(tokens, vocab, live)
    g = (dlogp.double() / tau)[:, None]
    ref = torch.where(live[:, None], g * (hot - p), torch.zeros_like(p))
    # p from the stored lse: u |lse| more
    tol = g.abs() * ((rel_of(z, tau) + U * l64.abs())[:, None] * p + 4 * U * (p + hot))
    check("dlogits", dz, ref, tol + last(ref, grad))
    assert bool((out[:, vocab:] == 7.0).all())


def test_extreme_rows(cuda):
    """-inf entries, the type's lowest value, far maxima, and rows without a
    finite logit."""
    V, inf = 1003, float("inf")
    for dtype in (F32, BF16):
        _, z = make_logits(8, V, dtype, seed=5)
        z[0, 1:] = -inf                      # one entry left
        z[1, ::2] = -inf
        z[2, 10:] = torch.finfo(dtype).min   # a mask of the lowest value
        z[3] = 300.0                         # equal entries
        z[4, 7] = 30000.0                    # one far above the rest
        z[5] = torch.finfo(dtype).min
        z[6] = -inf
        z[7, 3] = float("nan")
        tokens = torch.tensor([0, 1, 3, 5, 7, 9, 0, 3], device="cuda")
        logp, lse = losses.token_logp(z, tokens)
        check_logp(z[:6], tokens[:6], None, 1.0, logp[:6], lse[:6])
        assert torch.isnan(logp[6:]).all()
        dz = losses.token_logp_backward(z[:6], tokens[:6], lse[:6].contiguous(),
                                        torch.ones(6, device="cuda"))
        live = torch.ones(6, dtype=torch.bool, device="cuda")
        _, l64, p = softmax64(z[:6], 1.0, live)
        ref = onehot(tokens[:6], V, live) - p
        tol = (rel_of(z[:6], 1.0) + U * torch.where(l64.abs() < 1e30, l64.abs(), 0.0))[:, None] * p + 8 * U
        check("dlogits", dz[:5], ref[:5], (tol + last(ref, dtype))[:5])
        # skipped rows are not read: NaN, +inf and -inf there change nothing
        w = torch.ones(8, device="cuda")
        w[6:] = 0.0
        z[6, 0] = inf
        logp, lse = losses.token_logp(z, tokens, weight=w)
        assert (logp[6:] == 0).all() and (lse[6:] == 0).all()


def test_tokens_outside_the_vocabulary(cuda):
    _, z = make_logits(4, 100, F32, seed=9)
    z[1:] = float("nan")
    tokens = torch.tensor([5, -1, 100, -(1 << 40)], device="cuda")
    logp, lse = losses.token_logp(z, tokens)
    assert logp[0] != 0 and (logp[1:] == 0).all() and (lse[1:] == 0).all()
    one = torch.ones(4, device="cuda")
    dz = losses.token_logp_backward(z, tokens, lse, one)
    assert (dz[1:] == 0).all() and (dz[0] != 0).any()
    r = losses.policy_loss(z, tokens, logp, one)
    assert (r.row_loss[1:] == 0).all() and (r.dlogits[1:] == 0).all()
    assert torch.isfinite(r.loss)


# ------------------------------------------------------------------ policy
def policy_reference(z, tokens, old, adv, ref_logp, weight, tau, lo, hi, kl, scale):
    V = z.shape[1]
    live = live_rows(tokens, weight, V)
    x, l, p = softmax64(z, tau, live)
    t = torch.where(live, tokens, torch.zeros_like(tokens))
    logp = logp64(x, t)
    w = (torch.ones_like(logp) if weight is None else weight.double()) * live
    zero = torch.zeros_like(logp)
    A, lp = adv.double(), logp.clone().requires_grad_()
    ratio = torch.exp(lp - old.double())
    loss = -torch.min(ratio * A, torch.clamp(ratio, 1 - lo, 1 + hi) * A)
    size = (ratio * A).abs() + A.abs()
    if kl:
        gap = ref_logp.double() - lp
        loss = loss + kl * (torch.exp(gap) - gap - 1)
        size = size + kl * (torch.exp(gap) + 1 + gap.abs())
    (d,) = torch.autograd.grad(loss.sum(), lp)
    size, loss = size.detach(), loss.detach()
    g = scale * w * d / tau
    dz = torch.where(live[:, None], g[:, None] * (onehot(tokens, V, live) - p), torch.zeros_like(p))
    rel = rel_of(torch.where(live[:, None], z.double(), torch.zeros_like(x)), tau)
    err_l = w * size * (rel + 4 * U)
    tol = (scale * w * size / tau * (2 * rel + 8 * U))[:, None] * (p + onehot(tokens, V, live))
    return dict(row_loss=torch.where(live, w * loss, zero), logp=torch.where(live, logp, zero),
                dlogits=dz, tol_row=err_l, tol_logp=rel * live, tol_dz=tol)


def check_policy(r, e, scale, grad):
    check("row_loss", r.row_loss, e["row_loss"], e["tol_row"] + last(e["row_loss"], F32))
    check("logp", r.logp, e["logp"], e["tol_logp"] + last(e["logp"], F32))
    total = scale * e["row_loss"].sum()
    check("loss", r.loss, total, scale * (e["tol_row"] + last(e["row_loss"], F32)).sum() + last(total, F32))
    if grad is not None:
        check("dlogits", r.dlogits, e["dlogits"], e["tol_dz"] + last(e["dlogits"], grad))


def policy_inputs(z, tokens, tau, seed, lo, hi):
    rows = z.shape[0]
    x = torch.nan_to_num(z.double()) / tau
    logp = (x.gather(1, tokens[:, None])[:, 0] - torch.logsumexp(x, 1)).float()
    moved = 0.3 * torch.randn(rows, generator=gen(seed), device="cuda")
    for border in (math.log(1 - lo), math.log(1 + hi)):  # away from the branch
        moved = torch.where((moved - border).abs() < 1e-3, moved + 4e-3, moved)
    adv = torch.randn(rows, generator=gen(seed + 1), device="cuda")
    ref = logp + 0.4 * torch.randn(rows, generator=gen(seed + 2), device="cuda")
    return logp - moved, adv, ref


@pytest.mark.parametrize("rows,vocab", [(1, 1)] + SHAPES[2:])
@pytest.mark.parametrize("pad,shift", LAYOUT)
@pytest.mark.parametrize("dtype,grad", TYPES, ids=IDS)
def test_policy_loss(cuda, rows, vocab, pad, shift, dtype, grad):
    _, z = make_logits(rows, vocab, dtype, pad, shift, seed=vocab + 1)
    tokens, tau, lo, hi, kl, scale = tokens_of(rows, vocab, 4), 0.9, 0.15, 0.3, 0.07, 0.37
    old, adv, ref = policy_inputs(z, tokens, tau, 11, lo, hi)
    for w, k in ((None, 0.0), (weights_of(rows, 6), kl)):
        e = policy_reference(z, tokens, old, adv, ref, w, tau, lo, hi, k, scale)
        r = losses.policy_loss(z, tokens, old, adv, ref_logp=ref if k else None, weight=w,
                               temperature=tau, clip_low=lo, clip_high=hi, kl_coef=k, scale=scale,
                               grad_dtype=grad)
        assert r.dlogits.dtype is grad
        check_policy(r, e, scale, grad)
        only = losses.policy_loss(z, tokens, old, adv, ref_logp=ref, weight=w, temperature=tau,
                                  clip_low=lo, clip_high=hi, kl_coef=k, scale=scale, grad=False)
        assert only.dlogits is None and torch.equal(only.loss, r.loss)
        assert torch.equal(only.row_loss, r.row_loss)


def test_policy_branches(cuda):
    """Both signs of the advantage on both sides of the clip, and exactly on
    its border, where the ratio counts as inside."""
    V = 50
    _, z = make_logits(6, V, F32, seed=21)
    tokens = tokens_of(6, V, 22)
    logp, _ = losses.token_logp(z, tokens)
    step = torch.tensor([0.5, 0.5, -0.5, -0.5, 0.0, 0.0], device="cuda")
    adv = torch.tensor([1.0, -1.0, 1.0, -1.0, 2.0, 0.0], device="cuda")
    e = policy_reference(z, tokens, logp - step, adv, None, None, 1.0, 0.2, 0.2, 0.0, 1.0)
    r = losses.policy_loss(z, tokens, logp - step, adv, scale=1.0)
    check_policy(r, e, 1.0, F32)
    zero = (r.dlogits == 0).all(1).tolist()
    assert zero == [True, False, False, True, False, True]
    # clip 0: a ratio within rounding of 1; nothing is NaN and the loss is -A
    r = losses.policy_loss(z, tokens, logp, adv, clip_low=0.0, clip_high=0.0, scale=1.0)
    check("row_loss", r.row_loss, -adv, adv.abs().double() * 40 * U)


FAR = [(2, 300), (1, 40007), (1, 300001)]  # a row on one CTA, and on several


def far_rows(vocab, dtype, seed):
    """Rows whose sums cannot be taken relative to their first elements: far
    smaller ones ahead of a late maximum, all of the type's lowest value but
    a few equal ones a little above it, all far, and a late entry near the
    type's largest value."""
    _, z = make_logits(5, vocab, dtype, 1, 0, seed=seed)
    low, high = torch.finfo(dtype).min, torch.finfo(dtype).max
    z[0] -= 300.0
    z[0, -3] = 150.0
    z[1] = low
    z[1, vocab // 2::7] = low * 0.75
    z[2] = low
    z[3, -2] = high * 0.5
    z[4, :-5] = low
    return z


@pytest.mark.parametrize("rows,vocab", FAR)
@pytest.mark.parametrize("dtype,grad", TYPES, ids=IDS)
def test_policy_far_rows(cuda, rows, vocab, dtype, grad):
    z = far_rows(vocab, dtype, 23)
    tokens = torch.tensor([vocab - 3, vocab // 2, 5, vocab - 2, vocab - 4], device="cuda")
    x = torch.log_softmax(z.double(), 1)
    logp = x.gather(1, tokens[:, None])[:, 0].float()
    adv = torch.tensor([1.0, -0.5, 0.7, 1.3, 2.0], device="cuda")
    ref = logp + 0.1
    e = policy_reference(z, tokens, logp, adv, ref, None, 1.0, 0.2, 0.2, 0.1, 0.5)
    # rel_of() counts the far logits as 0: their powers are exact
    r = losses.policy_loss(z, tokens, logp, adv, ref_logp=ref, kl_coef=0.1, scale=0.5, grad_dtype=grad)
    check_policy(r, e, 0.5, grad)
    # the log-probability and the sum alone agree with it
    got, lse = losses.token_logp(z, tokens)
    check("logp", got, e["logp"], e["tol_logp"] + last(e["logp"], F32))


GAPS = [30.0, 43.0, 46.0, 60.0, 86.0, 88.0, 91.0, 97.0, 104.0]


def uneven_rows(vocab, dtype, seed):
    """Rows of which a third of the 16-byte pieces (in the first three fifths)
    lie GAPS below the rest, so that what a thread meets first says little of
    what it meets later, and below nothing of what another meets."""
    _, z = make_logits(2 * len(GAPS), vocab, dtype, seed=seed, std=1.0)
    i = torch.arange(vocab, device="cuda")
    low = (i // (16 // z.element_size()) % 3 == 0) & (i < vocab * 3 // 5)
    gap = torch.tensor(GAPS, device="cuda")
    z[:len(GAPS)] -= (low * gap[:, None]).to(dtype)
    z[len(GAPS):, vocab * 9 // 10] += gap.to(dtype)
    return z


UNEVEN = [300, 9001, 33003, 300001]


@pytest.mark.parametrize("vocab", UNEVEN)
@pytest.mark.parametrize("dtype,grad", TYPES, ids=IDS)
def test_policy_uneven_rows(cuda, vocab, dtype, grad):
    z = uneven_rows(vocab, dtype, 27)
    tokens = tokens_of(z.shape[0], vocab, 28)
    check_logp(z, tokens, None, 1.0, *losses.token_logp(z, tokens))
    old, adv, ref = policy_inputs(z, tokens, 1.0, 29, 0.2, 0.2)
    e = policy_reference(z, tokens, old, adv, ref, None, 1.0, 0.2, 0.2, 0.1, 0.5)
    # of probabilities below 2^-62 fp32 need hold nothing
    e["tol_dz"] = e["tol_dz"] + e["dlogits"].abs().amax(1, keepdim=True) * 2.0 ** -60
    r = losses.policy_loss(z, tokens, old, adv, ref_logp=ref, kl_coef=0.1, scale=0.5, grad_dtype=grad)
    check_policy(r, e, 0.5, grad)


# -------------------------------------------------------------- preference
def preference_reference(z, tokens, off, ref_logp, weight, tau, beta, eps, norm, scale):
    rows, V = z.shape
    inside = torch.zeros(rows, dtype=torch.bool, device="cuda")
    inside[off[0]:off[-1]] = True
    live = live_rows(tokens, weight, V) & inside
    x, l, p = softmax64(z, tau, live)
    t = torch.where(live, tokens, torch.zeros_like(tokens))
    logp = torch.where(live, logp64(x, t), torch.zeros_like(l))
    w = (torch.ones_like(logp) if weight is None else weight.double()) * live
    rel = rel_of(torch.where(live[:, None], z.double(), torch.zeros_like(x)), tau) * live
    lp = logp.clone().requires_grad_()
    dif = w * (lp - (0.0 if ref_logp is None else ref_logp.double()))
    each = w * (rel + U * logp.abs())
    margins, tols = [], []
    for i in range(len(off) // 2):
        s, e = [], 0.0
        for q in (0, 1):
            a, b = off[2 * i + q], off[2 * i + q + 1]
            n = w[a:b].sum() if norm else torch.tensor(1.0, device="cuda").double()
            n = torch.where(n == 0, torch.ones_like(n), n)
            s.append(dif[a:b].sum() / n)
            e = e + each[a:b].sum() / n
        margins.append(beta * (s[0] - s[1]))
        tols.append(beta * e)
    m = torch.stack(margins) if margins else dif[:0]
    tol_m = torch.stack([torch.as_tensor(v, device="cuda").double() for v in tols]) if tols else dif[:0].detach()
    ls = torch.nn.functional.logsigmoid
    pair = -(1 - eps) * ls(m) - eps * ls(-m)
    loss = scale * pair.sum()
    (d,) = torch.autograd.grad(loss, lp) if margins else (torch.zeros_like(logp),)
    # the adjoint of a row moves by at most beta scale w / n / 4 times its margin's error
    tol_d = torch.zeros_like(logp)
    for i in range(len(off) // 2):
        for q in (0, 1):
            a, b = off[2 * i + q], off[2 * i + q + 1]
            n = w[a:b].sum() if norm else torch.tensor(1.0, device="cuda").double()
            n = torch.where(n == 0, torch.ones_like(n), n)
            tol_d[a:b] = abs(beta) * scale * w[a:b] / n * (tol_m[i] / 4 + 4 * U)
    hot = onehot(tokens, V, live)
    dz = (d / tau)[:, None] * (hot - p)
    lse = torch.where(live, l, torch.zeros_like(l))
    tol_z = (tol_d / tau)[:, None] * (hot + p) + (d.abs() / tau)[:, None] * (
        (rel + U * lse.abs())[:, None] * p + 4 * U * (p + hot))
    return dict(logp=logp, lse=lse, margin=m.detach(), pair=pair.detach(), loss=loss.detach(),
                dlogp=d.detach(), dlogits=dz.detach(), rel=rel, tol_m=tol_m, tol_d=tol_d, tol_z=tol_z)


def check_preference(r, e, scale, grad):
    check("logp", r.logp, e["logp"], e["rel"] + last(e["logp"], F32))
    check("lse", r.lse, e["lse"], e["rel"] + last(e["lse"], F32))
    check("margin", r.margin, e["margin"], e["tol_m"] + last(e["margin"], F32))
    check("pair_loss", r.pair_loss, e["pair"], e["tol_m"] + last(e["pair"], F32))
    check("loss", r.loss, e["loss"], scale * (e["tol_m"] + last(e["pair"], F32)).sum() + last(e["loss"], F32))
    check("dlogp", r.dlogp, e["dlogp"], e["tol_d"] + last(e["dlogp"], F32))
    if grad is not None:
        check("dlogits", r.dlogits, e["dlogits"], e["tol_z"] + last(e["dlogits"], grad))


@pytest.mark.parametrize("rows,vocab,off", [
    (2, 7, [0, 1, 2]), (9, 33, [0, 3, 9]), (10, 1000, [1, 1, 4, 4, 4]), (5, 100, [2, 2, 2]),
    (40, 4097, [0, 7, 19, 20, 33]), (12, 32000, [0, 4, 6, 6, 11]), (3, 50001, [0, 2, 3])])
@pytest.mark.parametrize("dtype,grad", TYPES, ids=IDS)
@pytest.mark.parametrize("norm", [False, True])
def test_preference_loss(cuda, rows, vocab, off, dtype, grad, norm):
    """Ragged and empty sequences, rows ahead of the first and behind the last."""
    _, z = make_logits(rows, vocab, dtype, 1, 0, seed=vocab + 7)
    tokens = tokens_of(rows, vocab, 8)
    weight = weights_of(rows, 9)
    z[weight == 0] = float("nan")
    ref = -5.0 + torch.randn(rows, generator=gen(10), device="cuda")
    z[:off[0]] = float("nan")
    z[off[-1]:] = float("nan")
    scale = 0.7
    e = preference_reference(z, tokens, off, ref, weight, 1.3, 0.2, 0.1, norm, scale)
    r = losses.preference_loss(z, tokens, off, ref_logp=ref, weight=weight, temperature=1.3, beta=0.2,
                               label_smoothing=0.1, length_normalize=norm, scale=scale, grad_dtype=grad)
    check_preference(r, e, scale, grad)


def test_preference_large_margins_and_many_pairs(cuda):
    """More pairs than one launch takes; margins of both signs far from 0."""
    pairs, V = 300, 64
    off = [0]
    for i in range(2 * pairs):
        off.append(off[-1] + (i * 7) % 4)
    rows = off[-1]
    _, z = make_logits(rows, V, F32, seed=31, std=6.0)
    tokens = tokens_of(rows, V, 32)
    e = preference_reference(z, tokens, off, None, None, 1.0, 5.0, 0.0, False, 1.0 / pairs)
    r = losses.preference_loss(z, tokens, torch.tensor(off), beta=5.0)
    check_preference(r, e, 1.0 / pairs, F32)
    assert float(r.margin.max()) > 40 and float(r.margin.min()) < -40


# ------------------------------------------------------------ distillation
def distill_reference(z, index, top, tlse, weight, tau, scale):
    rows, V = z.shape
    live = torch.ones(rows, dtype=torch.bool, device="cuda") if weight is None else weight != 0
    w = (torch.ones(rows, device="cuda") if weight is None else weight).double()
    x = torch.where(live[:, None], z.double() / tau, torch.zeros((), dtype=torch.float64, device="cuda"))
    x.requires_grad_()
    lp = torch.log_softmax(x, 1)
    here = (index >= 0) & (index < V)
    at = torch.where(here, index, torch.zeros_like(index)).long()
    y = torch.where(here, top.double() / tau, torch.full_like(top, -math.inf).double())
    any_ = (y > -math.inf).any(1, keepdim=True)
    base = torch.logsumexp(y, 1, keepdim=True) if tlse is None else tlse.double()[:, None]
    lq = torch.where(y > -math.inf, y - torch.where(any_ | torch.tensor(tlse is not None, device="cuda"), base, torch.zeros_like(base)), y)
    q = torch.exp(lq)
    g = lp.gather(1, at)
    zero = torch.zeros_like(g)
    terms = torch.where(q > 0, q * (torch.where(q > 0, lq, zero) - torch.where(q > 0, g, zero)), zero)
    l = terms.sum(1)
    # how far the terms' parts reach before they cancel
    size = torch.where(q > 0, q * (1 + lq.nan_to_num(0, 0, 0).abs() + g.abs()), zero).sum(1)
    ratio = torch.zeros(rows, 1, dtype=torch.float64, device="cuda")
    member = torch.zeros(rows, V, dtype=torch.int32, device="cuda").scatter_add_(1, at, here.int()) > 0
    qr = torch.zeros(rows, dtype=torch.float64, device="cuda")
    if tlse is not None:
        qr = torch.clamp(1 - q.sum(1), min=0) * ~member.all(1)
        lr = torch.logsumexp(lp.masked_fill(member, -math.inf), 1)
        some = qr > 0
        lr_ = torch.where(some, lr, torch.zeros_like(lr))
        l = l + torch.where(some, qr * (torch.log(torch.where(some, qr, torch.ones_like(qr))) - lr_), torch.zeros_like(l))
        # 1 - sum q loses what the fp32 lse of the teacher does not have: none, it is exact here
        size = size + torch.where(some, qr * (1 + lr_.abs()) + 1 + lr_.abs() , torch.zeros_like(l))
        ratio = torch.where(some, qr / torch.exp(lr_), torch.zeros_like(qr))[:, None]
    k = tau * tau * w * live
    (d,) = torch.autograd.grad((scale / tau * k * l).sum(), x)
    p = torch.exp(lp.detach())
    qv = torch.zeros_like(p).scatter_add_(1, at, q * here)
    rel = rel_of(torch.where(live[:, None], z.double(), torch.zeros_like(p)), tau)
    G = (scale * tau * w * live)[:, None]
    tol = G * (p * (2 * rel[:, None] + 8 * U) * (1 + ratio * ~member) + 8 * U * qv)
    return dict(row=(k * l).detach(), dlogits=d, size=size.detach(), rel=rel, k=k, tol=tol)


def check_distill(r, e, scale, grad):
    tol = e["k"] * e["size"].detach() * (e["rel"] + 8 * U) + last(e["row"], F32)
    check("row_loss", r.row_loss, e["row"], tol)
    total = scale * e["row"].sum()
    check("loss", r.loss, total, scale * tol.sum() + last(total, F32))
    if grad is not None:
        check("dlogits", r.dlogits, e["dlogits"], e["tol"] + last(e["dlogits"], grad))


def teacher(z, k, tau, seed, tail):
    rows, V = z.shape
    index = torch.argsort(torch.rand(rows, V, generator=gen(seed), device="cuda"), 1)[:, :k].int().contiguous()
    top = 3.0 * torch.randn(rows, index.shape[1], generator=gen(seed + 1), device="cuda")
    tlse = None
    if tail:
        tlse = torch.logsumexp(top / tau, 1) + 0.3 * torch.rand(rows, generator=gen(seed + 2), device="cuda") + 0.02
    return index, top, tlse


@pytest.mark.parametrize("rows,vocab,k", [(1, 1, 1), (3, 2, 1), (5, 7, 3), (4, 32, 32), (2, 255, 100),
                                          (3, 1000, 1), (7, 4097, 64), (2, 32000, 128), (1, 50001, 1000),
                                          (3, 131073, 17), (500, 17, 4), (450, 9001, 20), (450, 20011, 33),
                                          (446, 33003, 64), (1, 700001, 50)])
@pytest.mark.parametrize("pad,shift", LAYOUT)
@pytest.mark.parametrize("dtype,grad", TYPES, ids=IDS)
@pytest.mark.parametrize("tail", [False, True], ids=["top", "tail"])
def test_distill_loss(cuda, rows, vocab, k, pad, shift, dtype, grad, tail):
    _, z = make_logits(rows, vocab, dtype, pad, shift, seed=vocab + 2)
    tau, scale = 2.0, 0.3
    index, top, tlse = teacher(z, k, tau, 41, tail)
    for w in (None, weights_of(rows, 42)):
        e = distill_reference(z, index, top, tlse, w, tau, scale)
        r = losses.distill_loss(z, index, top, teacher_lse=tlse, weight=w, temperature=tau,
                                scale=scale, grad_dtype=grad)
        check_distill(r, e, scale, grad)
        only = losses.distill_loss(z, index, top, teacher_lse=tlse, weight=w, temperature=tau,
                                   scale=scale, grad=False)
        assert only.dlogits is None and torch.equal(only.row_loss, r.row_loss)


@pytest.mark.parametrize("tail", [False, True], ids=["top", "tail"])
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_distill_odd_lists(cuda, tail, dtype):
    """Absent entries, entries named twice or three times, probability 0, a
    list without entries, and more places than vocabulary."""
    V, K = 301, 12
    _, z = make_logits(6, V, dtype, 2, 1, seed=51)
    index, top, _ = teacher(z, K, 1.0, 52, False)
    index[0, 3] = -1
    index[0, 4] = V
    index[0, 5] = 2 ** 31 - 1
    index[1, :6] = index[1, 0]
    index[2, 2] = index[2, 9]
    index[2, 4] = index[2, 9]
    top[3, 1:] = -math.inf
    index[4] = -1
    index[5, 0] = 0
    index[5, 1] = V - 1
    live_top = torch.where((index >= 0) & (index < V), top, torch.full_like(top, -math.inf))
    tlse = torch.logsumexp(live_top, 1).clamp(min=-20) + 0.25 if tail else None
    e = distill_reference(z, index, top, tlse, None, 1.0, 1.0)
    r = losses.distill_loss(z, index, top, teacher_lse=tlse, scale=1.0)
    check_distill(r, e, 1.0, dtype)
    if not tail:
        assert r.row_loss[4] == 0 and (r.dlogits[4] == 0).all()
    _, small = make_logits(2, 3, dtype, seed=53)
    index = torch.tensor([[0, 1, 2, 0, -1], [2, 2, 2, 2, 2]], dtype=torch.int32, device="cuda")
    top = torch.randn(2, 5, generator=gen(54), device="cuda")
    tl = torch.logsumexp(top, 1) + 0.5 if tail else None
    if tail:  # the first list is the whole vocabulary: no class is left for the rest
        tl[0] = torch.logsumexp(torch.tensor([top[0, 0], top[0, 1], top[0, 2], top[0, 3]]), 0).cuda()
    e = distill_reference(small, index, top, tl, None, 1.0, 1.0)
    r = losses.distill_loss(small, index, top, teacher_lse=tl, scale=1.0)
    check_distill(r, e, 1.0, dtype)


def test_distill_extreme_rows(cuda):
    """Student entries of -inf (listed: an infinite loss; outside: nothing),
    and a student whose mass outside the list is below fp32's range."""
    V = 500
    _, z = make_logits(4, V, F32, seed=61)
    index, top, tlse = teacher(z, 8, 1.0, 62, True)
    z[0, 100:] = -math.inf
    index[0] = torch.arange(8, dtype=torch.int32, device="cuda")
    z[1, index[1, 0].long()] = -math.inf
    z[2, index[2].long()] += 200.0
    z[3, index[3].long()] -= 200.0
    e = distill_reference(z, index, top, tlse, None, 1.0, 1.0)
    r = losses.distill_loss(z, index, top, teacher_lse=tlse, scale=1.0)
    assert math.isinf(r.row_loss[1]) and math.isinf(e["row"][1])
    keep = [0, 2, 3]
    check("row_loss", r.row_loss[keep], e["row"][keep], (e["size"] * (e["rel"] + 8 * U) + last(e["row"], F32))[keep])
    check("dlogits", r.dlogits[keep], e["dlogits"][keep], (e["tol"] + last(e["dlogits"], F32))[keep])


@pytest.mark.parametrize("rows,vocab", FAR)
@pytest.mark.parametrize("dtype,grad", TYPES, ids=IDS)
@pytest.mark.parametrize("tail", [False, True], ids=["top", "tail"])
def test_distill_far_rows(cuda, rows, vocab, dtype, grad, tail):
    z = far_rows(vocab, dtype, 63)
    index, top, tlse = teacher(z, 40, 1.0, 64, tail)
    index[0, 0] = vocab - 3
    index[1] = vocab // 2 + 7 * torch.arange(40, dtype=torch.int32, device="cuda") % (vocab // 2)
    index[3, 0] = vocab - 2
    keep = [0, 2] if tail else [0, 1, 2, 3]
    for row in keep:  # (a far listed maximum leaves the others nothing: an infinite loss)
        lp = torch.log_softmax(z[row].double(), 0)[index[row].long()]
        top[row] = torch.where(lp > -80, top[row], torch.full_like(top[row], -math.inf))
    if tail:
        here = torch.logsumexp(top, 1)
        tlse = torch.where(here > -50, here, torch.zeros_like(here)) + 0.2
    rows_ = [r for r in keep if bool((top[r] > -math.inf).any())]
    zz, ii, tt = z[rows_].clone(), index[rows_].contiguous(), top[rows_].contiguous()
    tl = tlse[rows_].contiguous() if tail else None
    e = distill_reference(zz, ii, tt, tl, None, 1.0, 1.0)
    r = losses.distill_loss(zz, ii, tt, teacher_lse=tl, scale=1.0, grad_dtype=grad)
    fine = torch.isfinite(e["row"])
    check("row_loss", r.row_loss[fine], e["row"][fine], (e["size"] * (e["rel"] + 8 * U) + last(e["row"], F32))[fine])
    check("dlogits", r.dlogits[fine], e["dlogits"][fine], (e["tol"] + last(e["dlogits"], grad))[fine])


@pytest.mark.parametrize("vocab", UNEVEN)
@pytest.mark.parametrize("dtype,grad", TYPES, ids=IDS)
@pytest.mark.parametrize("tail", [False, True], ids=["top", "tail"])
def test_distill_uneven_rows(cuda, vocab, dtype, grad, tail):
    z = uneven_rows(vocab, dtype, 67)
    index, top, tlse = teacher(z, 30, 1.0, 68, tail)
    e = distill_reference(z, index, top, tlse, None, 1.0, 1.0)
    # of probabilities below 2^-62 fp32 need hold nothing
    e["tol"] = e["tol"] + e["dlogits"].abs().amax(1, keepdim=True) * 2.0 ** -60
    check_distill(losses.distill_loss(z, index, top, teacher_lse=tlse, scale=1.0, grad_dtype=grad), e, 1.0, grad)


@pytest.mark.parametrize("dtype,grad,vocab", [(F32, F32, 851965), (F32, BF16, 851965), (BF16, BF16, 1703929)],
                         ids=IDS)
@pytest.mark.parametrize("shift", [0, 1, 3])
def test_largest_vocabulary(cuda, dtype, grad, vocab, shift):
    """The longest rows there may be, from addresses that make them touch the
    most 16-byte pieces, with the longest list."""
    _, z = make_logits(2, vocab, dtype, 2, shift, seed=71)
    tokens = torch.tensor([vocab - 1, 0], device="cuda")
    check_logp(z, tokens, None, 1.0, *losses.token_logp(z, tokens))
    old, adv, ref = policy_inputs(z, tokens, 1.0, 72, 0.2, 0.2)
    e = policy_reference(z, tokens, old, adv, ref, None, 1.0, 0.2, 0.2, 0.1, 0.5)
    check_policy(losses.policy_loss(z, tokens, old, adv, ref_logp=ref, kl_coef=0.1, scale=0.5, grad_dtype=grad),
                 e, 0.5, grad)
    for tail in (False, True):
        index, top, tlse = teacher(z, 1024, 1.0, 73, tail)
        e = distill_reference(z, index, top, tlse, None, 1.0, 1.0)
        check_distill(losses.distill_loss(z, index, top, teacher_lse=tlse, scale=1.0, grad_dtype=grad), e, 1.0, grad)


# -------------------------------------------------- gradient by differences
@pytest.mark.parametrize("which", ["logp", "policy", "preference", "distill", "distill_tail"])
def test_gradient_against_differences(cuda, which):
    """<dlogits, u> against the central difference of the 64-bit loss along u,
    step 2^-10: its truncation is below h^2 times the third derivative, itself
    at most (2 max|u| / tau)^3 times the rows' factors, and what rounds in 64
    bits is far below that."""
    rows, V, tau, h = 6, 97, 1.5, 2.0 ** -10
    _, z = make_logits(rows, V, F32, seed=71)
    tokens = tokens_of(rows, V, 72)
    old, adv, ref = policy_inputs(z, tokens, tau, 73, 0.2, 0.2)
    off = [0, 2, 3, 4, 6]
    index, top, tlse = teacher(z, 9, tau, 74, which == "distill_tail")
    if which == "logp":
        g = torch.randn(rows, generator=gen(75), device="cuda")
        _, lse = losses.token_logp(z, tokens, temperature=tau)
        dz = losses.token_logp_backward(z, tokens, lse, g, temperature=tau)

        def loss(x):
            return (g.double() * torch.log_softmax(x / tau, 1).gather(1, tokens[:, None])[:, 0]).sum()
    elif which == "policy":
        dz = losses.policy_loss(z, tokens, old, adv, ref_logp=ref, temperature=tau, kl_coef=0.1,
                                scale=1.0).dlogits

        def loss(x):
            return policy_reference(x, tokens, old, adv, ref, None, tau, 0.2, 0.2, 0.1, 1.0)["row_loss"].sum()
    elif which == "preference":
        dz = losses.preference_loss(z, tokens, off, ref_logp=ref, temperature=tau, beta=0.5,
                                    label_smoothing=0.1, scale=1.0).dlogits

        def loss(x):
            return preference_reference(x, tokens, off, ref, None, tau, 0.5, 0.1, False, 1.0)["loss"]
    else:
        dz = losses.distill_loss(z, index, top, teacher_lse=tlse, temperature=tau, scale=1.0).dlogits

        def loss(x):
            return distill_reference(x, index, top, tlse, None, tau, 1.0)["row"].sum()
    for k in range(3):
        u = torch.rand(rows, V, generator=gen(80 + k), device="cuda").double() * 2 - 1
        diff = (loss(z.double() + h * u) - loss(z.double() - h * u)) / (2 * h)
        got = (dz.double() * u).sum()
        bound = rows * 8 * (2 / tau) ** 3 * h * h + 64 * U * (dz.double().abs() * u.abs()).sum() * 8
        assert abs(float(diff - got)) <= float(bound), (which, float(diff), float(got), float(bound))


# ------------------------------------- in place, streams, graphs, no memory
def every(z, tokens, old, adv, ref, index, top, tlse, off, dlogits=None, stream=None):
    """One call of each objective that writes dlogits; with "own", into fresh
    copies of z in z's own layout (a row's alignment sets its sum's order)."""
    def c():
        if dlogits != "own":
            return z
        x = torch.empty(z.shape[0] * z.stride(0), dtype=z.dtype, device="cuda")
        x = x.view(z.shape[0], z.stride(0))[:, :z.shape[1]]
        return x.copy_(z)

    def d(x):
        return x if dlogits == "own" else None
    out = []
    x = c()
    out += list(losses.policy_loss(x, tokens, old, adv, ref_logp=ref, kl_coef=0.1, dlogits=d(x), stream=stream))
    x = c()
    out += list(losses.preference_loss(x, tokens, off, ref_logp=ref, dlogits=d(x), stream=stream))
    x = c()
    out += list(losses.distill_loss(x, index, top, dlogits=d(x), stream=stream))
    x = c()
    out += list(losses.distill_loss(x, index, top, teacher_lse=tlse, dlogits=d(x), stream=stream))
    x = c()
    logp, lse = losses.token_logp(x, tokens, stream=stream)
    out += [logp, lse, losses.token_logp_backward(x, tokens, lse, adv, dlogits=d(x), stream=stream)]
    return out


def every_inputs(rows, vocab, dtype, seed):
    _, z = make_logits(rows, vocab, dtype, 3, 0, seed=seed)
    tokens = tokens_of(rows, vocab, seed + 1)
    old, adv, ref = policy_inputs(z, tokens, 1.0, seed + 2, 0.2, 0.2)
    index, top, tlse = teacher(z, min(16, vocab), 1.0, seed + 5, True)
    off = [0, rows // 3, rows - 1]
    return z, tokens, old, adv, ref, index, top, tlse, off


@pytest.mark.parametrize("rows,vocab", [(3, 77), (5, 32000), (2, 131073)])
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_in_place_and_repeated(cuda, rows, vocab, dtype):
    """dlogits in the logits' memory, and a second run, give the same bytes."""
    inp = every_inputs(rows, vocab, dtype, 91)
    first, again, own = every(*inp), every(*inp), every(*inp, dlogits="own")
    for a, b, c in zip(first, again, own):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_other_streams_and_two_at_once(cuda):
    """Calls on two streams at once, given or current, equal those alone."""
    sets = [every_inputs(4, 32000, BF16, s) for s in (101, 202)]
    alone = [every(*i) for i in sets]
    torch.cuda.synchronize()
    one, two = torch.cuda.Stream(), torch.cuda.Stream()
    got = [[], []]
    for _ in range(4):
        got[0].append(every(*sets[0], stream=one))
        with torch.cuda.stream(two):
            got[1].append(every(*sets[1]))
    torch.cuda.synchronize()
    for a, runs in zip(alone, got):
        for r in runs:
            assert all(torch.equal(x, y) for x, y in zip(a, r))


def test_rows_of_every_shape_at_once(cuda):
    """Rows kept in shared memory, in tensor memory and over clusters of CTAs,
    on four streams at once."""
    sets = []
    for rows, vocab, dtype in ((600, 20011, BF16), (300, 33003, F32), (200, 131073, F32), (20, 700001, BF16)):
        _, z = make_logits(rows, vocab, dtype, seed=vocab + 9)
        sets.append((z, teacher(z, 16, 1.0, 110, True)))
    call = lambda z, t: losses.distill_loss(z, t[0], t[1], teacher_lse=t[2])
    alone = [call(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[] for _ in sets]
    for _ in range(3):
        for s, stream, g in zip(sets, streams, got):
            with torch.cuda.stream(stream):
                g.append(call(*s))
    torch.cuda.synchronize()
    for a, runs in zip(alone, got):
        for r in runs:
            assert all(torch.equal(x, y) for x, y in zip(a, r))


def test_captured_and_replayed(cuda):
    """Every objective in one graph, without a call ahead of the capture on
    its stream, replayed on new values in the same memory."""
    inp = list(every_inputs(6, 4097, F32, 301))
    new = every_inputs(6, 4097, F32, 302)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = every(*inp)
    for values in (new, every_inputs(6, 4097, F32, 303)):
        want = every(*values[:8], inp[8])
        for t, v in zip(inp[:8], values[:8]):
            t.copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_no_rows(cuda):
    z = torch.empty(0, 100, device="cuda")
    i64, f = torch.empty(0, dtype=torch.int64, device="cuda"), torch.empty(0, device="cuda")
    logp, lse = losses.token_logp(z, i64)
    assert logp.shape == (0,) and lse.shape == (0,)
    assert losses.token_logp_backward(z, i64, lse, f).shape == (0, 100)
    assert losses.policy_loss(z, i64, f, f).loss == 0
    assert losses.preference_loss(z, i64, [0]).loss == 0
    r = losses.preference_loss(z, i64, [0, 0, 0], scale=1.0)
    check("pair of nothing", r.pair_loss, torch.full((1,), math.log(2.0), device="cuda"), 2 * U)
    assert losses.distill_loss(z, torch.empty(0, 3, dtype=torch.int32, device="cuda"),
                               torch.empty(0, 3, device="cuda")).loss == 0


def test_refusals_of_tensors(cuda):
    _, z = make_logits(4, 10, F32, seed=1)
    tok, f = tokens_of(4, 10, 1), torch.zeros(4, device="cuda")
    for bad in (lambda: losses.token_logp(z.half(), tok),
                lambda: losses.token_logp(z.t(), tok),
                lambda: losses.token_logp(z[:1].expand(4, 10), tok),
                lambda: losses.token_logp(z, tok.int()),
                lambda: losses.token_logp(z, tok[:3]),
                lambda: losses.token_logp(z, tok.cpu()),
                lambda: losses.token_logp(z, tok, weight=f.double()),
                lambda: losses.token_logp(z, tok, weight=torch.zeros(8, device="cuda")[::2]),
                lambda: losses.token_logp_backward(z.bfloat16(), tok, f, f, grad_dtype=F32),
                lambda: losses.token_logp_backward(z, tok, f, f, dlogits=z[:, :9]),
                lambda: losses.token_logp_backward(z, tok, f, f, dlogits=z.half()),
                lambda: losses.policy_loss(z, tok, f, f, grad=False, dlogits=z),
                lambda: losses.policy_loss(z, tok, f, f, kl_coef=0.1),
                lambda: losses.preference_loss(z, tok, [0, 2]),
                lambda: losses.preference_loss(z, tok, [0, 2, 5]),
                lambda: losses.preference_loss(z, tok, torch.zeros(3, dtype=torch.int64, device="cuda")),
                lambda: losses.distill_loss(z, tok, f),
                lambda: losses.distill_loss(z, tok[:, None], f[:, None]),
                lambda: losses.distill_loss(z, tok.int()[:, None], f[:, None], temperature=0.0),
                lambda: losses.distill_loss(z, tok.int()[:, None][:, :0], f[:, None][:, :0])):
        with pytest.raises(DopError):
            bad()


def test_far_offsets(cuda):
    """Rows whose elements lie more than 2^32 bytes and 2^31 elements into the
    logits."""
    V, ld = 1000, (1 << 31) // 2 + 8
    buf = torch.empty(2 * ld + V, dtype=BF16, device="cuda")
    z = torch.as_strided(buf, (3, V), (ld, 1))
    z.copy_((torch.randn(3, V, generator=gen(5), device="cuda") * 2).bfloat16())
    tokens = tokens_of(3, V, 6)
    small = torch.empty(3, V, dtype=BF16, device="cuda").copy_(z)  # rows 16-byte aligned, as z's
    inp = (torch.zeros(3, device="cuda"), torch.ones(3, device="cuda"))
    a = losses.policy_loss(small, tokens, *inp)
    b = losses.policy_loss(z, tokens, *inp, dlogits=z)
    assert torch.equal(a.loss, b.loss) and torch.equal(a.dlogits, b.dlogits.clone())


# ------------------------------------------------------------- with the model
def demo(precision):
    from dop.mixtral import MixtralConfig, Model, demo_batch, init_params, init_router
    c = MixtralConfig.demo()
    if precision == DOP_BF16:  # the bf16 lens takes whole 32-column tiles
        c = MixtralConfig(32, 64, 2, 4, 2, 16, 96, 4, 2, 1e-5, 1_000_000.0, 24)
    p = init_params(c)
    init_router(c, p)
    batch, seq, tokens, targets = demo_batch(c)
    P = torch.from_numpy(p).cuda()
    P = P + 0.01 * torch.randn(P.shape, generator=gen(1), device="cuda")
    if precision == DOP_BF16:
        P = P.bfloat16()
    return (c, Model(c, batch, seq, precision), P.contiguous(),
            torch.tensor(tokens, device="cuda"), torch.tensor(targets, device="cuda"))


@pytest.mark.parametrize("precision", [DOP_F32, DOP_BF16], ids=["f32", "bf16"])
def test_model_trained_on_the_objectives(cuda, precision):
    """Cross-entropy written as each objective gives the model's own
    forward_backward: distillation from one teacher entry, the policy loss at
    ratio 1 and advantage 1, and the log-probability's adjoint -1 / n."""
    c, m, P, tokens, targets = demo(precision)
    n = tokens.numel()
    want = m.forward_backward(P, tokens, targets)
    logits = m.forward(P, tokens)
    assert torch.equal(logits, want.logits)
    logp, lse = losses.token_logp(logits, targets)
    # fp32 adjoints through the model: the three differ from the model's own
    # by the rounding of p (rel of it) where V = 32; a bf16 cotangent rounds
    # to 2^-8 first, in the model's own path too, and what lies near a
    # rounding border may fall to the other side: 2^-7 of the largest
    tol = 2.0 ** -7 if precision == DOP_BF16 else 1e-4
    kinds = [F32] if precision == DOP_F32 else [F32, BF16]
    top = torch.zeros(n, 1, device="cuda")
    for kind in kinds:
        outs = [losses.distill_loss(logits, targets.int()[:, None].contiguous(), top, grad_dtype=kind),
                losses.policy_loss(logits, targets, logp, torch.ones(n, device="cuda"), grad_dtype=kind)]
        assert abs(float(outs[0].loss - want.loss)) < 1e-5 * float(want.loss)
        grads = [o.dlogits for o in outs]
        grads.append(losses.token_logp_backward(logits, targets, lse, torch.full((n,), -1.0 / n, device="cuda"),
                                                grad_dtype=kind))
        for d in grads:
            m.forward(P, tokens)
            got = m.backward(P, tokens, d)
            assert float((got - want.grad).abs().max()) <= tol * float(want.grad.abs().max())
    m.close()


def test_model_preference_step_lowers_nothing_else(cuda):
    """A run as a user makes it: reference log-probabilities, then for each
    objective the get, the objective in the logits' memory, and the put.  The
    put is linear in dlogits: doubled, it doubles the adjoint bit for bit."""
    c, m, P, tokens, targets = demo(DOP_F32)
    logits = m.forward(P, tokens)
    ref, _ = losses.token_logp(logits, targets)
    n = tokens.numel()
    P2 = P + 0.02 * torch.randn(P.shape, generator=gen(2), device="cuda")
    adv = torch.randn(n, generator=gen(3), device="cuda")
    index, top, tlse = teacher(logits, 8, 1.0, 4, True)
    runs = [lambda z, s: losses.policy_loss(z, targets, ref, adv, ref_logp=ref, kl_coef=0.1, scale=s, dlogits=z),
            lambda z, s: losses.preference_loss(z, targets, [0, 5, 8, 12, n], ref_logp=ref, scale=s, dlogits=z),
            lambda z, s: losses.distill_loss(z, index, top, teacher_lse=tlse, scale=s, dlogits=z)]
    for f in runs:
        grads = []
        for s in (0.25, 0.5):
            z = m.forward(P2, tokens)
            r = f(z, s)
            assert torch.isfinite(r.loss) and r.dlogits.data_ptr() == z.data_ptr()
            grads.append(m.backward(P2, tokens, z))
        assert torch.equal(2 * grads[0], grads[1]) and float(grads[0].abs().max()) > 0
        # differences of the loss along one direction of the parameters
        u = torch.randn(P.shape, generator=gen(5), device="cuda")
        h = 2.0 ** -9 / float(u.norm()) * 4
        vals = [float(f(m.forward(P2 + t * h * u, tokens), 0.5).loss.double()) for t in (1, -1)]
        slope = (grads[1].double() * u.double()).sum().item()
        # fp32 logits of this model carry about 2^-20 of their size into a
        # loss of order 1, over 2h; the rest is h^2
        bound = 2.0 ** -19 / (2 * h) * 4 + 0.02 * abs(slope)
        assert abs((vals[0] - vals[1]) / (2 * h) - slope) <= bound
    m.close()


def test_model_state_and_refusals(cuda):
    c, m, P, tokens, targets = demo(DOP_F32)
    d = torch.zeros(tokens.numel(), c.vocab, device="cuda")
    with pytest.raises(DopError) as e:
        m.backward(P, tokens, d)  # before any forward
    assert e.value.code == -5
    m.forward(P, tokens)
    for bad in (d[:, :-1], d.double(), d.bfloat16(), d.t()):
        with pytest.raises(DopError):
            m.backward(P, tokens, bad)
    assert lib().dop_model_forward(m._h, P.data_ptr(), tokens.data_ptr(), d.data_ptr() + 4, None) == -1
    m.close()
