"""What Model.forward and Model.backward refuse before any device work: with a
handle that stands on the CPU and a library that only notes its calls."""
import contextlib
import types

import pytest
import torch

from dop import mixtral
from dop._lib import DOP_BF16, DOP_F32, DopError

N, T, V = 48, 6, 8
F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture
def calls(monkeypatch):
    made = []

    class Library:
        def __getattr__(self, name):
            return lambda *a: made.append((name, a)) or 0

    monkeypatch.setattr(mixtral, "lib", lambda: Library())
    monkeypatch.setattr(torch.cuda, "device", lambda d: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: types.SimpleNamespace(cuda_stream=0))
    return made


def model(precision):
    m = mixtral.Model.__new__(mixtral.Model)
    m.cfg, m.batch, m.seq, m.precision = mixtral.MixtralConfig.demo(), 2, T // 2, precision
    m.cfg.vocab, m.n_params, m.device, m._h = V, N, torch.device("cpu"), None
    return m


def operands(precision):
    act = F32 if precision == DOP_F32 else BF16
    return (torch.zeros(N, dtype=act), torch.zeros(T, dtype=torch.int64),
            torch.zeros(T, V, dtype=F32))


@pytest.mark.parametrize("precision", [DOP_F32, DOP_BF16], ids=["f32", "bf16"])
def test_operands_that_fit(calls, precision):
    m, (P, tokens, z) = model(precision), operands(precision)
    assert m.forward(P, tokens, logits=z) is z
    assert m.forward(P, tokens.view(2, T // 2)).shape == (T, V)
    grad = torch.zeros(N)
    assert m.backward(P, tokens, z, grad=grad) is grad
    assert m.backward(P, tokens, z).shape == (N,)
    if precision == DOP_BF16:
        m.backward(P, tokens, z.bfloat16())
        assert calls[-1][1][3] == DOP_BF16
    assert calls[0][1][3] == z.data_ptr() and calls[2][1][5] == grad.data_ptr()


def outputs_that_do_not_fit(shape):
    n = shape[0]
    yield torch.zeros(shape, dtype=BF16)              # half the bytes that are written
    yield torch.zeros(shape, dtype=torch.float64)
    yield torch.zeros((n - 1,) + shape[1:])
    yield torch.zeros((n + 1,) + shape[1:])
    yield torch.zeros((2 * n,) + shape[1:])[::2]      # rows apart
    yield torch.zeros(shape, device="meta")           # another device
    yield [0.0]
    if len(shape) == 2:
        yield torch.zeros(shape[1], n).t()
        yield torch.zeros(n * shape[1])


@pytest.mark.parametrize("precision", [DOP_F32, DOP_BF16], ids=["f32", "bf16"])
def test_outputs_that_do_not_fit(calls, precision):
    m, (P, tokens, z) = model(precision), operands(precision)
    for bad in outputs_that_do_not_fit((T, V)):
        with pytest.raises(DopError, match="logits"):
            m.forward(P, tokens, logits=bad)
    for bad in outputs_that_do_not_fit((N,)):
        with pytest.raises(DopError, match="grad"):
            m.backward(P, tokens, z, grad=bad)
    assert not calls


@pytest.mark.parametrize("precision", [DOP_F32, DOP_BF16], ids=["f32", "bf16"])
def test_inputs_that_do_not_fit(calls, precision):
    m, (P, tokens, z) = model(precision), operands(precision)
    other = P.bfloat16() if precision == DOP_F32 else P.float()
    for bad in (other, P[:-1], torch.cat([P, P])[::2], P.to("meta"), None):
        with pytest.raises(DopError, match="params"):
            m.forward(bad, tokens)
        with pytest.raises(DopError, match="params"):
            m.backward(bad, tokens, z)
    for bad in (tokens.int(), tokens[:-1], torch.zeros(2 * T, dtype=torch.int64)[::2],
                tokens.to("meta"), None):
        with pytest.raises(DopError, match="tokens"):
            m.forward(P, bad)
        with pytest.raises(DopError, match="tokens"):
            m.backward(P, bad, z)
    bad = [z[:-1], z.double(), z.to("meta"), torch.zeros(V, T).t(), None]
    for d in bad + ([z.bfloat16()] if precision == DOP_F32 else []):
        with pytest.raises(DopError, match="dlogits"):
            m.backward(P, tokens, d)
    assert not calls
