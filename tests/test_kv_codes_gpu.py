"""GPU: codes of an 8-bit cache are the nearest ones to x * 448 / max for rows of every type and magnitude, ties to even."""

import pytest
import torch

import fastkernels_b200 as fk
from tests import paged_oracle as O
from tests.test_kv_cache_gpu import BF, E4, F16, F32

pytestmark = pytest.mark.gpu


def codes_of(x):
    """Codes (as 64-bit values) and scales that `paged_kv_append` keeps of rows [n, 256], which fill one sequence."""
    n = x.shape[0]
    pages = -(-n // 16)
    cache = [torch.zeros(pages, 1, 16, 256, dtype=torch.uint8, device="cuda").view(E4) for _ in range(2)]
    scale = [torch.zeros(pages, 1, 16, device="cuda") for _ in range(2)]
    fk.paged_kv_append(x.unsqueeze(1), x.unsqueeze(1), *cache, torch.arange(pages, device="cuda", dtype=torch.int32).view(1, -1),
                       torch.tensor([n], dtype=torch.int32, device="cuda"), torch.tensor([0, n], dtype=torch.int32, device="cuda"), key_scale=scale[0], value_scale=scale[1])
    assert torch.equal(cache[0].view(torch.uint8), cache[1].view(torch.uint8)) and torch.equal(*scale)
    return cache[0].view(-1, 256)[:n].float().double(), scale[0].view(-1)[:n]


def check(x):
    got, scale = codes_of(x)
    codes = O.quantised(x)[0]               # x 448 / max in 64 bits: off a tie by 2^-49 at least, or on it
    most = x.double().abs().amax(-1).clamp_min(O.LEAST)
    scales = (most / torch.full_like(most, 448.0)).float()
    assert torch.equal(got, codes), f"{(got != codes).sum().item()} of {codes.numel()} codes"
    assert torch.equal(scale, scales)


@pytest.mark.parametrize("dtype", [F32, BF, F16])
def test_normal_rows(dtype):
    g = torch.Generator(device="cuda").manual_seed(11)
    for _ in range(4):
        check(torch.randn(30000, 256, generator=g, device="cuda").to(dtype))


@pytest.mark.parametrize("exponent", [0, 1, -30, -41, -60, -99, -104, 100, 126])
def test_fp32_rows_next_to_the_middles_between_codes(exponent):
    """Elements that are the nearest fp32 numbers to (middle between two codes) * max / 448, and their neighbours."""
    g = torch.Generator(device="cuda").manual_seed(12)
    codes = torch.arange(127, dtype=torch.uint8).view(E4).float().double().cuda()
    middles = (codes[1:] + codes[:-1]) / 2
    most = (1 + torch.rand(4000, 1, generator=g, device="cuda")).float()
    near = (middles * most.double() / 448).float()
    step = torch.randint(-1, 2, near.shape, generator=g, device="cuda", dtype=torch.int32)
    near = (near.view(torch.int32) + step).view(torch.float32) * torch.randint(0, 2, near.shape, generator=g, device="cuda").mul(2).sub(1)
    x = torch.zeros(4000, 256, device="cuda")
    x[:, :1], x[:, 1:127], x[:, 127:253] = most, near, -near
    check(torch.ldexp(x, torch.tensor(exponent, device="cuda")) if exponent > -100 else (x.double() * 2.0 ** exponent).float())


def test_fp32_rows_with_elements_of_all_magnitudes():
    g = torch.Generator(device="cuda").manual_seed(13)
    x = torch.randn(20000, 256, generator=g, device="cuda") * torch.exp2(40 * torch.rand(20000, 256, generator=g, device="cuda") - 40) * torch.exp2(
        200 * torch.rand(20000, 1, generator=g, device="cuda") - 100)
    check(x)
