"""8-bit checkpoints of the widest rows that are taken: the ends of each row are what they are by themselves."""
import pytest
import torch

from mlp_megakernel_b200 import _lib, fp8_checkpoint, fp8_restore

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("width", [2 ** 31 - 1, 2 ** 31 - 16])
def test_the_ends_of_the_widest_rows(width):
    rows, end = 2, 5120
    last = width // 128 * 128 - end  # a group's first column
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.zeros(rows, width, device="cuda", dtype=torch.float16)
    for r in range(rows):
        for cols in (slice(0, end), slice(last, None)):
            x[r, cols] = 10 ** r * torch.randn(x[r, cols].shape, device="cuda", generator=g)
    q, scale = fp8_checkpoint(x)
    back = fp8_restore(q, scale, torch.float16)
    for cols, groups in ((slice(0, end), slice(0, end // 128)), (slice(last, None), slice(last // 128, None))):
        want = fp8_checkpoint(x[:, cols].contiguous())
        assert torch.equal(q[:, cols].view(torch.uint8), want[0].view(torch.uint8)) and torch.equal(scale[:, groups], want[1])
        assert torch.equal(back[:, cols], fp8_restore(*want, torch.float16))
    assert not back[:, end:last].any()
    torch.cuda.synchronize()
    assert _lib.device_status() == 0
