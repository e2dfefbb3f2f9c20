"""Very wide rows of the 8-bit checkpoints: the widths that are refused, and the index arithmetic of the kernels up to
there (their own, compiled for the host)."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import mlp_megakernel_b200 as m

ops = torch.ops.mlpk
FP8, F16, F32 = torch.float8_e4m3fn, torch.float16, torch.float32
MOST = 2 ** 31 - 1


@pytest.mark.parametrize("width", [MOST + 1, 2 ** 32 - 8, 5 * 10 ** 9])
def test_rows_wider_than_an_int_are_refused(width):
    """The C calls take the width as an int: 5e9 columns would be 705,032,704 of them."""
    with FakeTensorMode():
        x, q = torch.empty(1, width, dtype=F16, device="cuda"), torch.empty(1, width, dtype=FP8, device="cuda")
        scale = torch.empty(1, -(-width // 128), dtype=F32, device="cuda")
        for call in (lambda: m.fp8_checkpoint(x), lambda: ops.fp8_checkpoint(x), lambda: m.fp8_restore(q, scale),
                     lambda: ops.fp8_restore(q, scale, F16)):
            with pytest.raises(ValueError, match="columns"):
                call()


def test_the_widest_rows_are_taken():
    with FakeTensorMode():
        q, scale = m.fp8_checkpoint(torch.empty(2, MOST, dtype=F16, device="cuda"))
        assert q.shape == (2, MOST) and scale.shape == (2, 2 ** 24)
        assert m.fp8_restore(q, scale, F16).shape == (2, MOST)
