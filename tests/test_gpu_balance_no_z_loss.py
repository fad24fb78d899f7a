"""Without a coefficient there is no z-loss, also where its squares pass fp32."""
import pytest
import torch

from tests.test_gpu_balance_far_logits import EXTREME, _check, _rows, dev  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", list(EXTREME))
@pytest.mark.parametrize("E", [6, 200, 300, 1000, 1500])
def test_no_squares_without_their_coefficient(dev, dtype, E):  # noqa: F811
    _check(*_rows(EXTREME[dtype], E, dtype, dev), 0.0)
    _check(*_rows(EXTREME[dtype], E, dtype, dev), 0.0, coef=2.0, d_loss=0.5)
