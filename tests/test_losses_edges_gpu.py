"""Calls of the objectives over logits at the edges of what they accept, each
against its definition in 64 bits."""
import ctypes as C

import pytest
import torch

from dop import losses
from dop._lib import DOP_BF16, DOP_F32, DopError, check as ok, lib
from test_losses_gpu import demo, tokens_of

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
