"""Calls of the objectives over logits at the edges of what they accept, each
against its definition in 64 bits."""
import ctypes as C

import pytest
import torch

from dop import losses
from dop._lib import DOP_F32, DopError, check as ok, lib
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


# ------------------------------------------------ the model's get and put
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
