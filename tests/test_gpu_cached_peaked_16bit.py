"""As test_gpu_cached_peaked.py for 16-bit caches, far longer contexts and lower tails.

P is rounded to the type once (half a step h).  An f16 P has steps of 2^-24 at the least; a row's largest stands at 2^7 or above, so
that what is lost below is 2^-32 of that largest for every key.  O is a 32-bit sum of one product after the other, each of which
is cut to the last place of the sum so far, 2^-23 of it at most: half that on the way for terms alike, so that a chain of N keys is
off by N 2^-24 A at most.  A row's chain is all keys, or where its rows are laid out in copies what is a copy's share of them.
2^-12 is for ex2.approx and the sums of P."""

import pytest
import torch

import splash_attention_mgpu as sa

DEV = "cuda:0"


@pytest.mark.gpu
@pytest.mark.parametrize("d,dtype", [(64, torch.float16), (128, torch.float16), (128, torch.bfloat16)], ids=str)
@pytest.mark.parametrize("h", [1, 40, 100])
@pytest.mark.parametrize("keys,gap,spread", [(131072, 14.0, 0.0), (131072, 12.0, 0.5), (32768, 15.0, 1.0)])
def test_gpu_peaked(d, dtype, h, keys, gap, spread):
  g = torch.Generator(device=DEV).manual_seed(0)
  batch, page = 150, 256
  cache = sa.make_kv_cache(keys // page, 1, d, page_size=page, dtype=dtype, device=DEV)
  table = torch.randperm(keys // page, generator=torch.Generator().manual_seed(0)).to(torch.int32).to(DEV)[None]
  k = 0.05 * torch.randn(1, 1, keys, d, generator=g, device=DEV)
  k[..., 0] = spread * torch.randn(1, 1, keys, generator=g, device=DEV)
  v = 1 + 0.25 * torch.randn(1, 1, keys, d, generator=g, device=DEV)
  k[:, :, 5, 0] = gap
  v[:, :, 5] = 0
  v[:, :, 5, d - 1] = 1.5
  k, v = k.to(dtype), v.to(dtype)
  cache.write(k, v, table, torch.zeros(1, dtype=torch.int32, device=DEV))
  q = 0.01 * torch.randn(batch, h, 1, d, generator=g, device=DEV)
  q[..., 0] = 1 - torch.arange(h, device=DEV).view(h, 1) / (16.0 * h)
  q = q.to(dtype)
  lens = torch.full((batch,), keys, dtype=torch.int32, device=DEV)
  out, (lse,) = sa.make_splash_cached()(q, cache, table.expand(batch, -1), lens, save_residuals=True)
  sa.check_device_status()
  half = torch.finfo(dtype).eps / 2
  k, v = k[0, 0].double(), v[0, 0].double()
  for i in (0, batch - 1):
    x = q[i, :, 0].double()
    s = x @ k.T
    ds = 2.0 ** -19 * (x.abs() @ k.abs().T).amax(-1)
    p = torch.softmax(s, -1)
    want, a = p @ v, p @ v.abs()
    low = 2.0 ** -32 * p.amax(-1, keepdim=True) * v.abs().sum(0) if dtype == torch.float16 else 0.0
    chain = keys // (4 if h <= 32 else 2 if h <= 64 else 1)
    bar = (half + 2.0 ** -12 + chain * 2.0 ** -24 + 2 * ds[:, None]) * a + low + half * want.abs() + 2.0 ** -25
    off = float(((out[i, :, 0].double() - want).abs() / bar).max())
    assert off <= 1, off
    assert ((lse[i, :, 0].double() - torch.logsumexp(s, -1)).abs() <= ds + 2.0 ** -15).all()
