"""What pagedAppend stores in 8 bits: value / scale as an fp32 quotient, limited to +-448 and rounded to the nearest e4m3."""
import pytest
import torch

import blockedAttention
from test_gpu_paged_cache import FP8, e4m3

pytestmark = pytest.mark.gpu


def stored(x, scale, dev):
    """x [n] in 16 bits, as the keys and values of one head."""
    dim = 256 if len(x) % 256 == 0 else len(x)
    rows = x.reshape(1, -1, dim).to(dev)
    cache = [torch.zeros((1, 1, rows.shape[1], dim), device=dev).to(FP8) for _ in range(2)]
    s = torch.tensor([scale], dtype=torch.float32, device=dev)
    blockedAttention.pagedAppend(rows, rows, *cache, torch.arange(rows.shape[1], device=dev), s, s)
    assert torch.equal(cache[0].view(torch.uint8), cache[1].view(torch.uint8))
    return cache[0].reshape(-1).cpu()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("scale", [1.0, 0.01, 1 / 19, 60.29411697387695, -0.3, 3e-7, 1e-30, 2.0 ** -120, 2.0 ** 120, 1e-42, 0.0, float("inf"), float("nan")])
def test_every_value(dev, dtype, scale):
    x = torch.arange(-(1 << 15), 1 << 15, dtype=torch.int32).to(torch.int16).view(dtype)
    quotient = x.float() / torch.tensor(scale, dtype=torch.float32)
    want = e4m3(quotient.double().clamp(-448, 448))
    got = stored(x, scale, dev).float()
    assert torch.equal(torch.isnan(got), torch.isnan(quotient))
    there = ~torch.isnan(quotient)
    assert torch.equal(got[there].double(), want[there])
    assert torch.equal(torch.signbit(got[there]), torch.signbit(quotient[there]))


@pytest.mark.parametrize("dtype,x,scale,exact,quotient,kept", [
    (torch.bfloat16, 1.0, 1 / 19, 18.99999987, 19.0, 20.0),               # between 18 and 20: the exact quotient is nearer to 18
    (torch.float16, 1025.0, 60.29411697387695, 17.0000002, 17.0, 16.0)])  # between 16 and 18: nearer to 18
def test_a_quotient_that_fp32_rounds_to_a_tie_goes_to_even(dev, dtype, x, scale, exact, quotient, kept):
    s = torch.tensor(scale, dtype=torch.float32)
    assert abs(x / s.double().item() - exact) < 1e-7 and (torch.tensor(x) / s).item() == quotient
    assert stored(torch.full((8,), x, dtype=dtype), scale, dev).float().tolist() == [kept] * 8
