"""Where the RMS norm rounds: the mean once, the 8-bit scale once and its
reciprocal once, so that values next to a tie of the 8-bit type fall where these
roundings put them.  Everything is compared to the bit."""
import pytest
import torch

from mlp_megakernel_b200 import fused_rms_norm, fused_rms_norm_fp8

pytestmark = pytest.mark.gpu


def near_ties(groups, each, seed):
    """[groups, each] fp32 values whose largest of each group is its first, the
    others within two steps of a value that the scale takes to the middle between
    two values of the 8-bit type; the group's scale and its reciprocal."""
    g = torch.Generator(device="cuda").manual_seed(seed)

    def uniform(*shape):
        return torch.rand(*shape, device="cuda", generator=g)

    largest = 1 + uniform(groups)
    scale = largest * torch.tensor(1.0 / 448.0, device="cuda")
    inverse = 1.0 / scale
    odd = (uniform(groups, each) * 8).floor() * 2 + 1
    middle = (1 + odd / 16) * torch.exp2((uniform(groups, each) * 14).floor() - 6)
    v = middle.clamp(max=400.0) / inverse[:, None]
    step = (uniform(groups, each) * 5).floor() - 2
    for k in (1, 2):
        v = torch.where(step >= k, torch.nextafter(v, torch.full_like(v, 1e9)), v)
        v = torch.where(step <= -k, torch.nextafter(v, torch.zeros_like(v)), v)
    v[:, 0] = largest
    return v, scale, inverse


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("width", [128, 1024, 4096, 16384])
def test_scale_and_reciprocal_are_rounded_once(width, dtype):
    """Rows of ones have a root mean square of 1, so y is the weight itself."""
    x = torch.ones(3, width, device="cuda", dtype=dtype)
    for seed in range(16):
        w, scale, inverse = near_ties(width // 128, 128, seed)
        q, got = fused_rms_norm_fp8(x, w.view(-1), eps=0.0, group=128)
        assert torch.equal(got, scale.expand(3, -1))
        want = (w * inverse[:, None]).to(torch.float8_e4m3fn).float().view(-1)
        assert torch.equal(q.float(), want.expand(3, -1))
        w, scale, inverse = near_ties(1, width, 100 + seed)
        q, got = fused_rms_norm_fp8(x, w.view(-1), eps=0.0)
        assert torch.equal(got, scale.expand(3, 1))
        assert torch.equal(q.float(), (w * inverse).to(torch.float8_e4m3fn).float().expand(3, -1))


@pytest.mark.parametrize("seed", range(4))
def test_scale_of_ragged_groups(seed):
    """A width of 1001: groups that begin inside a vector, the last one short."""
    w, scale, inverse = near_ties(8, 128, seed)
    x = torch.ones(20, 1001, device="cuda", dtype=torch.float16)
    q, got = fused_rms_norm_fp8(x, w.view(-1)[:1001].contiguous(), eps=0.0, group=128)
    assert torch.equal(got, scale.expand(20, -1))
    want = (w * inverse[:, None]).to(torch.float8_e4m3fn).float().view(-1)[:1001]
    assert torch.equal(q.float(), want.expand(20, -1))


@pytest.mark.parametrize("width", [3, 5, 100, 1000, 1001, 5120, 12000])
def test_mean_is_rounded_once(width):
    """Whole numbers whose squares add up exactly in fp32."""
    g = torch.Generator(device="cuda").manual_seed(width)
    x = torch.randint(-8, 9, (200, width), device="cuda", generator=g).float()
    total = x.square().sum(1, keepdim=True)
    assert torch.equal(total.double(), x.double().square().sum(1, keepdim=True))
    rms = torch.rsqrt(total / torch.tensor(float(width), device="cuda"))
    rows = (total > 0)[:, 0]
    assert torch.equal(fused_rms_norm(x, eps=0.0)[rows], (x * rms)[rows])
