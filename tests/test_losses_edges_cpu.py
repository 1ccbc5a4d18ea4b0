"""Refusals of dlogits that lies between the logits' rows and on some of them."""
import pytest

from dop._lib import DOP_BF16
from test_losses_cpu import FAR, GRAD, P, refused


@pytest.mark.parametrize("name", GRAD)
@pytest.mark.parametrize("over", [
    # fp32 rows of 40 bytes, 80 apart: 40 bytes behind them is the one place
    dict(dz=P + 36), dict(dz=P + 44), dict(dz=P - 36), dict(dz=P - 44), dict(dz=P + 80),
    dict(dz=P + 240 + 36), dict(dz=P),
    dict(dz=P + 40, ldd=21), dict(dz=P + 40, ldd=19),        # other distances
    dict(dz=P + 38, gprec=DOP_BF16, ldd=40), dict(dz=P + 62, gprec=DOP_BF16, ldd=40),
    dict(dz=P + 40, gprec=DOP_BF16, ldd=20),
], ids=str)
def test_dlogits_on_the_rows(name, over):
    over = {"ld": 20, "ldd": 20, **over}
    if over["dz"] == P:
        over["ldd"] = 21
    refused(name, **over)
    assert FAR > over["dz"]
