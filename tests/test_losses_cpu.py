"""Refusals of the objectives over logits (dop_token_logp ... in
include/dop.h), through the C ABI and through dop.losses.  Every refused call
returns before any device work, so these run without a GPU."""
import ctypes as C

import pytest
import torch

from dop import losses
from dop._lib import DOP_BF16, DOP_F32, DopError, lib

P = 1 << 20  # an aligned address that no refused call dereferences
FAR = 1 << 40
INF, NAN = float("inf"), float("nan")


def call(name, **over):
    """The named entry point with valid arguments but for those in `over`."""
    off = over.pop("seq_off", [0, 1, 2])
    a = dict(rows=4, vocab=10, prec=DOP_F32, z=P, ld=10, tokens=P, weight=None, tau=1.0, logp=P,
             lse=P, dlogp=P, gprec=DOP_F32, dz=FAR, ldd=10, old=P, adv=P, ref=P, lo=0.2, hi=0.2,
             kl=0.1, scale=1.0, loss=P, row_loss=P, pairs=1, beta=0.1, smooth=0.0, norm=0,
             pair_loss=P, margin=P, k=2, idx=P, top=P, tlse=None)
    assert set(over) <= set(a)
    a.update(over)
    g = lambda *ks: [a[k] for k in ks]  # noqa: E731
    args = {
        "dop_token_logp": lambda: g("rows", "vocab", "prec", "z", "ld", "tokens", "weight", "tau",
                                    "logp", "lse"),
        "dop_token_logp_backward": lambda: g("rows", "vocab", "prec", "z", "ld", "tokens", "lse",
                                             "dlogp", "tau", "gprec", "dz", "ldd"),
        "dop_policy_loss_grad": lambda: g("rows", "vocab", "prec", "z", "ld", "tokens", "old",
                                          "adv", "ref", "weight", "tau", "lo", "hi", "kl", "scale",
                                          "loss", "row_loss", "logp", "gprec", "dz", "ldd"),
        "dop_preference_loss_grad": lambda: g("rows", "vocab", "prec", "z", "ld", "tokens",
                                              "pairs") + [
            None if off is None else (C.c_int64 * len(off))(*off)] + g(
            "ref", "weight", "tau", "beta", "smooth", "norm", "scale", "loss", "pair_loss",
            "margin", "logp", "lse", "dlogp", "gprec", "dz", "ldd"),
        "dop_distill_loss_grad": lambda: g("rows", "vocab", "prec", "z", "ld", "k", "idx", "top",
                                           "tlse", "weight", "tau", "scale", "loss", "row_loss",
                                           "gprec", "dz", "ldd"),
    }[name]()
    return getattr(lib(), name)(*args, None)


EVERY = ["dop_token_logp", "dop_token_logp_backward", "dop_policy_loss_grad",
         "dop_preference_loss_grad", "dop_distill_loss_grad"]
GRAD = EVERY[1:]


def refused(name, code=-1, **over):
    assert call(name, **over) == code
    assert lib().dop_last_error().decode() != ""


@pytest.mark.parametrize("name", EVERY)
@pytest.mark.parametrize("over", [
    dict(rows=-1), dict(rows=1 << 31), dict(vocab=0), dict(vocab=1 << 31, ld=1 << 31),
    dict(prec=2), dict(prec=-1), dict(z=None), dict(z=P + 2), dict(ld=9), dict(ld=0),
    dict(tau=0.0), dict(tau=-1.0), dict(tau=INF), dict(tau=NAN)], ids=str)
def test_shared_refusals(name, over):
    if "vocab" in over:
        over = {**over, "ldd": max(10, over["vocab"])}
    refused(name, **over)


@pytest.mark.parametrize("name", GRAD)
@pytest.mark.parametrize("over", [
    dict(gprec=3), dict(prec=DOP_BF16, gprec=DOP_F32), dict(ldd=9), dict(dz=FAR + 2),
    dict(dz=P, gprec=DOP_BF16),              # the logits' memory in another type
    dict(dz=P, ldd=11),                      # in another stride
    dict(dz=P + 4), dict(dz=P + 156), dict(z=P + 4, dz=P),  # partly on the logits
], ids=str)
def test_gradient_refusals(name, over):
    refused(name, **over)


@pytest.mark.parametrize("name,over", [
    ("dop_token_logp", dict(tokens=None)), ("dop_token_logp", dict(logp=None)),
    ("dop_token_logp", dict(lse=None)),
    ("dop_token_logp_backward", dict(tokens=None)), ("dop_token_logp_backward", dict(lse=None)),
    ("dop_token_logp_backward", dict(dlogp=None)), ("dop_token_logp_backward", dict(dz=None)),
    ("dop_policy_loss_grad", dict(tokens=None)), ("dop_policy_loss_grad", dict(old=None)),
    ("dop_policy_loss_grad", dict(adv=None)), ("dop_policy_loss_grad", dict(loss=None)),
    ("dop_policy_loss_grad", dict(row_loss=None)), ("dop_policy_loss_grad", dict(logp=None)),
    ("dop_policy_loss_grad", dict(ref=None)),
    ("dop_policy_loss_grad", dict(lo=-0.1)), ("dop_policy_loss_grad", dict(lo=1.1)),
    ("dop_policy_loss_grad", dict(hi=-0.1)), ("dop_policy_loss_grad", dict(hi=INF)),
    ("dop_policy_loss_grad", dict(lo=NAN)), ("dop_policy_loss_grad", dict(kl=NAN)),
    ("dop_policy_loss_grad", dict(scale=INF)),
    ("dop_preference_loss_grad", dict(seq_off=None)),
    ("dop_preference_loss_grad", dict(seq_off=[0, 2, 1])),
    ("dop_preference_loss_grad", dict(seq_off=[-1, 1, 2])),
    ("dop_preference_loss_grad", dict(seq_off=[0, 1, 5])),
    ("dop_preference_loss_grad", dict(pairs=-1)), ("dop_preference_loss_grad", dict(beta=NAN)),
    ("dop_preference_loss_grad", dict(smooth=-0.1)), ("dop_preference_loss_grad", dict(smooth=1.1)),
    ("dop_preference_loss_grad", dict(scale=NAN)), ("dop_preference_loss_grad", dict(margin=None)),
    ("dop_preference_loss_grad", dict(pair_loss=None)),
    ("dop_preference_loss_grad", dict(dlogp=None)), ("dop_preference_loss_grad", dict(lse=None)),
    ("dop_distill_loss_grad", dict(idx=None)), ("dop_distill_loss_grad", dict(top=None)),
    ("dop_distill_loss_grad", dict(k=0)), ("dop_distill_loss_grad", dict(k=-1)),
    ("dop_distill_loss_grad", dict(scale=INF)), ("dop_distill_loss_grad", dict(loss=None)),
], ids=str)
def test_own_refusals(name, over):
    refused(name, **over)


def test_unsupported_sizes():
    refused("dop_distill_loss_grad", code=-4, k=1025)
    for name in EVERY:
        for prec, most in ((DOP_F32, 851_965), (DOP_BF16, 1_703_929)):
            refused(name, code=-4, prec=prec, gprec=prec, vocab=most + 1, ld=most + 1, ldd=most + 1)


def test_model_refusals():
    L = lib()
    assert L.dop_model_forward(None, P, P, P, None) == -1
    assert L.dop_model_backward(None, P, P, DOP_F32, P, P, None) == -1


def test_python_refusals():
    """dop.losses checks what a pointer cannot show before the call."""
    host = torch.zeros(4, 10)
    tok = torch.zeros(4, dtype=torch.int64)
    for bad in (host, host[0], host.double(), None):
        with pytest.raises(DopError):
            losses.token_logp(bad, tok)
        with pytest.raises(DopError):
            losses.distill_loss(bad, tok, tok)
