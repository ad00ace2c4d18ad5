"""The largest and smallest numbers of a type in an 8-bit cache: what they read back as, and attention to them."""

import math

import pytest
import torch

import splash_attention_mgpu as sa

DEV = "cuda:0"


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,numbers", [
    # largest number, first that rounds to 2^16, last that does not, 448 * 2^7; 9 2^-24 among the subnormals
    (torch.float16, {65504.0: torch.inf, 63488.0: torch.inf, 63456.0: 61440.0, 57344.0: 57344.0, 9 * 2.0 ** -24: 9 * 2.0 ** -24}),
    (torch.bfloat16, {torch.finfo(torch.bfloat16).max: torch.inf, 0.96875 * 2.0 ** 127 * 2: torch.inf, 0.9609375 * 2.0 ** 127 * 2: 0.9375 * 2.0 ** 127 * 2}),
], ids=["f16", "bf16"])
@pytest.mark.parametrize("sign", [1, -1])
def test_gpu_ends_of_the_range(dtype, numbers, sign):
  n = len(numbers)
  x = torch.zeros(1, 1, n, 64, dtype=dtype, device=DEV)
  x[0, 0, :, 7] = sign * torch.tensor(list(numbers), dtype=dtype, device=DEV)
  cache = sa.make_kv_cache(1, 1, 64, page_size=16, quantized=True, device=DEV)
  table, zero = torch.zeros(1, 1, dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
  cache.write(x, x, table, zero)
  assert not (cache.k_exponent[0, 0, :n] == -128).any()  # finite, all of them
  k, v = cache.read(table, zero + n, n, dtype=dtype)
  want = torch.zeros_like(x)
  want[0, 0, :, 7] = sign * torch.tensor(list(numbers.values()), dtype=torch.float64, device=DEV).to(dtype)
  assert torch.equal(k, want) and torch.equal(v, want)


@pytest.mark.gpu
@pytest.mark.parametrize("h", [1, 12, 20, 40, 100])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("large", [2.0 ** 127, 2.0 ** 127 * 1.9921875, 2.0 ** 110, 2.0 ** -50], ids=str)
def test_gpu_attention_to_large_and_small_values(h, d, large):
  """Finite values have finite results: equal scores, values that are `large` times 0.9 to 1.  Stored, they are off by 2^-4."""
  length = 300
  g = torch.Generator(device=DEV).manual_seed(0)
  v = (large * (0.9 + 0.1 * torch.rand(1, 1, length, d, generator=g, device=DEV, dtype=torch.float64))).to(torch.bfloat16)
  v[..., 3] = 0
  cache = sa.make_kv_cache(5, 1, d, page_size=64, quantized=True, device=DEV)
  table, zero = torch.arange(5, dtype=torch.int32, device=DEV)[None], torch.zeros(1, dtype=torch.int32, device=DEV)
  cache.write(torch.zeros_like(v), v, table, zero)
  q = torch.ones(1, h, 1, d, dtype=torch.bfloat16, device=DEV)
  out, (lse,) = sa.make_splash_cached()(q, cache, table, zero + length, save_residuals=True)
  sa.check_device_status()
  assert (lse.double() - math.log(length)).abs().max() <= 2.0 ** -18
  stored = cache.v.double() * torch.exp2(cache.v_exponent.double())[..., None]  # [pages, 1, 64, d]
  want = stored.transpose(0, 1).reshape(-1, d)[:length].mean(0)
  bar = (2.0 ** -8 + 2.0 ** -9 + 2.0 ** -11 + 2.0 ** -12) * want
  fits = want < 0.99 * torch.finfo(torch.bfloat16).max
  assert ((out[0, :, 0].double() - want).abs() <= bar)[:, fits].all() and not out[0, :, 0, 3].any()
  assert not out.isnan().any()
