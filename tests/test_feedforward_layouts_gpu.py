"""The layout of the large products, at the smallest sizes that have it: whole tiles and behind them tiles in shares, 256
columns wide (test_feedforward_layouts.py asserts that), against the formulas in 64 bits."""
import pytest
import torch

from tests.test_feedforward_gpu import U, gated_case, linear_case, status  # noqa: F401
from tests.test_feedforward_layouts import SHARES, dw, dx, forward

pytestmark = pytest.mark.gpu
CASES = [(call, sizes) for call, sizes in SHARES]


@pytest.mark.parametrize("call,sizes", CASES, ids=[f"{c.__name__}-{'x'.join(map(str, s))}" for c, s in CASES])
@pytest.mark.parametrize("dtype", list(U))
def test_whole_tiles_and_shares(call, sizes, dtype):
    if torch.cuda.get_device_properties(0).multi_processor_count != 148:
        pytest.skip("the layouts are those of 148 SMs")
    rows, k, n, *more = sizes
    if call is forward:
        linear_case(rows, k, n, dtype, "silu", dtype, True)
        linear_case(rows, k, n, dtype, "gelu_tanh", torch.float32, False, transposed=True)
    elif more and more[0] == 2:  # of both projections
        gated_case(rows, k, n, 136, dtype, "silu", True, 1)
        gated_case(rows, k, n, 136, dtype, "silu", False, 2, (True, True, False))
    else:
        assert call in (dx, dw)
        linear_case(rows, k, n, dtype, None, dtype, False, transposed=bool(more[1:]) and more[1])
