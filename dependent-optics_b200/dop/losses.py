"""Objectives over a model's logits, each with its adjoint.

What the model lens is trained on after next-token cross-entropy
(src/mixtral.rs:966-991; these have no counterpart in the crate): token
log-probabilities and their adjoint, the clipped policy loss with a KL term,
the preference loss over pairs of sequences, and distillation from a teacher's
top logits.  include/dop.h defines each of them.

`logits` is a torch CUDA tensor [rows, vocab], float32 or bfloat16, whose rows
may lie apart (stride(1) == 1, stride(0) >= vocab).  The adjoint `dlogits` is
written into the tensor given as `dlogits` (which may be `logits` itself) or
into a new one of `grad_dtype` (default: the logits' type; bfloat16 for float32
logits is what a bf16 `Model.backward` takes without a conversion).  Tokens are
int64, indices int32, everything else float32, contiguous, on the logits'
device.  `weight` [rows] masks and scales rows; a row of weight 0, or whose
token lies outside [0, vocab), is skipped and its logits are not read.

Work goes to `stream`, or to the device's current stream when it is None; the
call does not wait for it.  A stream given is the caller's to order behind what
wrote the tensors, which stay in use until it has done the work.  Arguments that
do not fit raise DopError.

    logits = model.forward(params, tokens)
    r = losses.policy_loss(logits, actions, old_logp, advantage, dlogits=logits)
    grad = model.backward(params, tokens, r.dlogits)
"""
from __future__ import annotations

import contextlib
import ctypes as C
from typing import Any, NamedTuple

import torch

from ._lib import DOP_BF16, DOP_F32, DopError, check, lib

_PRECISION = {torch.float32: DOP_F32, torch.bfloat16: DOP_BF16}


class PolicyLoss(NamedTuple):
    loss: Any      # scalar tensor
    row_loss: Any  # [rows]
    logp: Any      # [rows]
    dlogits: Any   # [rows, vocab] or None


class PreferenceLoss(NamedTuple):
    loss: Any
    pair_loss: Any  # [pairs]
    margin: Any     # [pairs]
    logp: Any       # [rows]
    lse: Any        # [rows]
    dlogp: Any      # [rows]: the loss's adjoint with respect to logp
    dlogits: Any


class DistillLoss(NamedTuple):
    loss: Any
    row_loss: Any
    dlogits: Any


def _refuse(msg):
    raise DopError(-1, f"invalid argument: {msg}")


def _matrix(t, name):
    """(rows, vocab, precision, row stride) of a matrix of logits."""
    if not isinstance(t, torch.Tensor) or t.dim() != 2 or not t.is_cuda:
        _refuse(f"{name} must be a CUDA tensor [rows, vocab]")
    prec = _PRECISION.get(t.dtype)
    if prec is None:
        _refuse(f"{name} must be float32 or bfloat16, not {t.dtype}")
    rows, vocab = t.shape
    ld, one = t.stride()
    if one != 1 and vocab > 1:
        _refuse(f"the elements of a row of {name} must be contiguous")
    return rows, vocab, prec, ld if rows > 1 else max(ld, vocab)


def _vector(t, name, dtype, shape, device):
    """Device pointer of a contiguous tensor of that type and shape (None: NULL)."""
    if t is None:
        return None
    if not isinstance(t, torch.Tensor) or t.dtype is not dtype or t.shape != shape:
        _refuse(f"{name} must be a {dtype} tensor of shape {shape}")
    if t.device != device or not t.is_contiguous():
        _refuse(f"{name} must be contiguous and on the logits' device")
    return t.data_ptr()


_HERE = contextlib.nullcontext()


def _on(logits, stream):
    """A context in which the logits' device and the call's stream are current
    (what the call allocates then belongs to that stream)."""
    if stream is not None:
        if stream.device != logits.device:
            _refuse("the stream belongs to another device than the logits")
        return torch.cuda.stream(stream)
    if logits.get_device() != torch.cuda.current_device():
        return torch.cuda.device(logits.device)
    return _HERE


def _current(device):
    """The current stream's handle (without a Stream object: a microsecond of
    a small call's time)."""
    return torch._C._cuda_getCurrentRawStream(device.index)


def _gradient(logits, dlogits, grad_dtype, grad):
    """dlogits (given, new, or None), its pointer, precision and row stride."""
    if not grad:
        if dlogits is not None:
            _refuse("dlogits given although grad is False")
        return None, None, DOP_F32, logits.shape[1]
    if dlogits is None:
        dlogits = torch.empty(logits.shape, dtype=grad_dtype or logits.dtype, device=logits.device)
    elif dlogits.shape != logits.shape or dlogits.device != logits.device:
        _refuse("dlogits must have the logits' shape and device")
    elif grad_dtype is not None and dlogits.dtype is not grad_dtype:
        _refuse("dlogits is not of grad_dtype")
    _, _, prec, ld = _matrix(dlogits, "dlogits")
    return dlogits, dlogits.data_ptr(), prec, ld


def token_logp(logits, tokens, *, weight=None, temperature=1.0, stream=None):
    """(logp, lse), both float32 [rows]: the log-probability of tokens[r] under
    softmax(logits[r] / temperature), and the row's log-sum-exp."""
    rows, vocab, prec, ld = _matrix(logits, "logits")
    dev = logits.device
    tok = _vector(tokens, "tokens", torch.int64, (rows,), dev)
    w = _vector(weight, "weight", torch.float32, (rows,), dev)
    with _on(logits, stream):
        logp = torch.empty(rows, dtype=torch.float32, device=dev)
        lse = torch.empty_like(logp)
        check(lib().dop_token_logp(rows, vocab, prec, logits.data_ptr(), ld, tok, w, temperature,
                                   logp.data_ptr(), lse.data_ptr(), _current(dev)))
    return logp, lse


def token_logp_backward(logits, tokens, lse, dlogp, *, temperature=1.0, dlogits=None,
                        grad_dtype=None, stream=None):
    """dlogits from dlogp [rows], the adjoint of `token_logp`'s logp, and the
    lse it returned.  Rows with dlogp 0 get a row of zeros; those that the
    forward skipped by their weight need a dlogp of 0."""
    rows, vocab, prec, ld = _matrix(logits, "logits")
    dev = logits.device
    tok = _vector(tokens, "tokens", torch.int64, (rows,), dev)
    l = _vector(lse, "lse", torch.float32, (rows,), dev)
    g = _vector(dlogp, "dlogp", torch.float32, (rows,), dev)
    with _on(logits, stream):
        dlogits, dz, gprec, ldd = _gradient(logits, dlogits, grad_dtype, True)
        check(lib().dop_token_logp_backward(rows, vocab, prec, logits.data_ptr(), ld, tok, l, g,
                                            temperature, gprec, dz, ldd, _current(dev)))
    return dlogits


def policy_loss(logits, tokens, old_logp, advantage, *, ref_logp=None, weight=None,
                temperature=1.0, clip_low=0.2, clip_high=0.2, kl_coef=0.0, scale=None,
                dlogits=None, grad_dtype=None, grad=True, stream=None) -> PolicyLoss:
    """The clipped policy loss with a KL term towards ref_logp; `scale`
    defaults to 1 / rows."""
    rows, vocab, prec, ld = _matrix(logits, "logits")
    dev, f32, one = logits.device, torch.float32, (rows,)
    tok = _vector(tokens, "tokens", torch.int64, one, dev)
    old = _vector(old_logp, "old_logp", f32, one, dev)
    adv = _vector(advantage, "advantage", f32, one, dev)
    ref = _vector(ref_logp, "ref_logp", f32, one, dev)
    w = _vector(weight, "weight", f32, one, dev)
    if scale is None:
        scale = 1.0 / max(rows, 1)
    with _on(logits, stream):
        loss = torch.empty((), dtype=f32, device=dev)
        row_loss = torch.empty(rows, dtype=f32, device=dev)
        logp = torch.empty_like(row_loss)
        dlogits, dz, gprec, ldd = _gradient(logits, dlogits, grad_dtype, grad)
        check(lib().dop_policy_loss_grad(rows, vocab, prec, logits.data_ptr(), ld, tok, old, adv,
                                         ref, w, temperature, clip_low, clip_high, kl_coef, scale,
                                         loss.data_ptr(), row_loss.data_ptr(), logp.data_ptr(),
                                         gprec, dz, ldd, _current(dev)))
    return PolicyLoss(loss, row_loss, logp, dlogits)


def preference_loss(logits, tokens, seq_off, *, ref_logp=None, weight=None, temperature=1.0,
                    beta=0.1, label_smoothing=0.0, length_normalize=False, scale=None,
                    dlogits=None, grad_dtype=None, grad=True, stream=None) -> PreferenceLoss:
    """The preference loss over pairs of packed sequences.  `seq_off` (a
    sequence of ints or a CPU int64 tensor, 2 * pairs + 1 of them) gives the
    row offsets: pair i's chosen sequence is rows seq_off[2i] .. seq_off[2i+1],
    its rejected one seq_off[2i+1] .. seq_off[2i+2].  `scale` defaults to
    1 / pairs."""
    rows, vocab, prec, ld = _matrix(logits, "logits")
    dev, f32, one = logits.device, torch.float32, (rows,)
    if isinstance(seq_off, torch.Tensor):
        if seq_off.is_cuda or seq_off.dtype is not torch.int64 or seq_off.dim() != 1:
            _refuse("seq_off must be integers on the host")
        seq_off = seq_off.tolist()
    n = len(seq_off)
    if n % 2 != 1:
        _refuse("seq_off must hold 2 * pairs + 1 offsets")
    pairs = n // 2
    off = (C.c_int64 * n)(*seq_off)
    tok = _vector(tokens, "tokens", torch.int64, one, dev)
    ref = _vector(ref_logp, "ref_logp", f32, one, dev)
    w = _vector(weight, "weight", f32, one, dev)
    if scale is None:
        scale = 1.0 / max(pairs, 1)
    with _on(logits, stream):
        loss = torch.empty((), dtype=f32, device=dev)
        pair_loss = torch.empty(pairs, dtype=f32, device=dev)
        margin = torch.empty_like(pair_loss)
        logp = torch.empty(rows, dtype=f32, device=dev)
        lse = torch.empty_like(logp)
        dlogp = torch.empty_like(logp)
        dlogits, dz, gprec, ldd = _gradient(logits, dlogits, grad_dtype, grad)
        check(lib().dop_preference_loss_grad(
            rows, vocab, prec, logits.data_ptr(), ld, tok, pairs, off, ref, w, temperature, beta,
            label_smoothing, int(length_normalize), scale, loss.data_ptr(), pair_loss.data_ptr(),
            margin.data_ptr(), logp.data_ptr(), lse.data_ptr(), dlogp.data_ptr(), gprec,
            dz, ldd, _current(dev)))
    return PreferenceLoss(loss, pair_loss, margin, logp, lse, dlogp, dlogits)


def distill_loss(logits, top_index, top_logit, *, teacher_lse=None, weight=None, temperature=1.0,
                 scale=None, dlogits=None, grad_dtype=None, grad=True, stream=None) -> DistillLoss:
    """Distillation from a teacher's top logits (top_index int32 and top_logit
    float32, both [rows, top_k]); with `teacher_lse` [rows], the log-sum-exp of
    the teacher's whole row over the temperature, the mass outside the listed
    entries is one more class.  `scale` defaults to 1 / rows."""
    rows, vocab, prec, ld = _matrix(logits, "logits")
    dev, f32 = logits.device, torch.float32
    if not isinstance(top_index, torch.Tensor) or top_index.dim() != 2:
        _refuse("top_index must be a tensor [rows, top_k]")
    k = top_index.shape[1]
    idx = _vector(top_index, "top_index", torch.int32, (rows, k), dev)
    top = _vector(top_logit, "top_logit", f32, (rows, k), dev)
    tl = _vector(teacher_lse, "teacher_lse", f32, (rows,), dev)
    w = _vector(weight, "weight", f32, (rows,), dev)
    if scale is None:
        scale = 1.0 / max(rows, 1)
    with _on(logits, stream):
        loss = torch.empty((), dtype=f32, device=dev)
        row_loss = torch.empty(rows, dtype=f32, device=dev)
        dlogits, dz, gprec, ldd = _gradient(logits, dlogits, grad_dtype, grad)
        check(lib().dop_distill_loss_grad(rows, vocab, prec, logits.data_ptr(), ld, k, idx, top,
                                          tl, w, temperature, scale, loss.data_ptr(),
                                          row_loss.data_ptr(), gprec, dz, ldd, _current(dev)))
    return DistillLoss(loss, row_loss, dlogits)
