"""GPU: what layers keep in 8 bits, when they do, and what comes back at the ends of a type."""
import pytest
import torch

from slayerpytorch_b200 import checkpoint

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [32, 33, 64, 100])
def test_the_largest_float16_values_come_back_finite(T):
    """Values above 65024 are kept as 64 * 2^10, which is no float16: they come back as the largest one, off by less than half a step of 2^10."""
    most = torch.finfo(torch.float16).max
    values = torch.cat([torch.arange(64992, 65505, 32), torch.tensor([1.0, 700.0, 1e4, 6e4])])
    x = values[torch.randint(0, len(values), (50, T), generator=torch.Generator().manual_seed(T))].half()
    x[:, ::32] = most
    x[::2] *= -1
    x = x.cuda()
    kept = checkpoint.compress(x)
    exact, got = kept.restore(torch.float32), kept.restore()
    assert got.dtype == torch.float16 and bool(got.isfinite().all())
    assert torch.equal(got.float(), exact.clamp(-most, most)) and float(exact.max()) == 65536
    assert bool(((got.float() - x.float()).abs() <= most / 127).all())
    # a float32 tensor in float16: rounded to it, infinities where it is beyond
    far = checkpoint.compress(torch.full((1, T), 3e5, device="cuda"))
    assert bool(far.restore(torch.float16).isposinf().all()) and bool(far.restore().isfinite().all())
