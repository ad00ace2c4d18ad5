"""Attention over an 8-bit cache where few keys weigh far more than the many others, whose sum still counts.

Bar, per number of the result, with p the softmax weights and A = sum_j p_j |v_j|.  The probabilities are rounded to f16
(2^-11) and then to three numbers of e5m2, 3 bits each (2^-9), or for f16 to four, which hold all of an f16 number.  The lowest
step of e5m2 is 2^-16, of which half is lost where a row's largest 2^ev p stands at 2^12 or more: 2^-29 of that one, times the
codes of the values.  2^-12 covers 32-bit sums and ex2.approx; the scores are off by dS (see test_gpu_cached_attention.py), which
moves p by at most 2 dS; the result is rounded once.  Nothing here grows with the number of keys but the 2^-29."""

import pytest
import torch

import splash_attention_mgpu as sa

DEV = "cuda:0"
FORMS = [(d, dtype) for d in (64, 128) for dtype in (torch.bfloat16, torch.float16)]


def _peaked(d, dtype, h, kvh, n, batch, length, gap, spread, at, seed=0):
  """`batch` sequences of the same keys, so that a kv head's keys are about one CTA's work and not cut into short pieces.  Their scores
  are `spread` times normal numbers, but for key `at`: `gap` above them.  Values have a mean, that key's are one number and zeros, and
  all have about the same exponent."""
  g = torch.Generator(device=DEV).manual_seed(seed)
  page = 64
  width = -(-length // page)
  cache = sa.make_kv_cache(width, kvh, d, page_size=page, quantized=True, device=DEV)
  table = torch.randperm(width, generator=torch.Generator().manual_seed(seed)).view(1, width).to(torch.int32).to(DEV)
  k = 0.05 * torch.randn(1, kvh, length, d, generator=g, device=DEV)
  k[..., 0] = spread * torch.randn(1, kvh, length, generator=g, device=DEV)
  v = 1 + 0.25 * torch.randn(1, kvh, length, d, generator=g, device=DEV)
  k[:, :, at, 0] = gap
  v[:, :, at] = 0
  v[:, :, at, d - 1] = 1.5
  cache.write(k.to(dtype), v.to(dtype), table, torch.zeros(1, dtype=torch.int32, device=DEV))
  q = 0.01 * torch.randn(batch, h, n, d, generator=g, device=DEV)
  q[..., 0] = 1 - torch.arange(h * n, device=DEV).view(h, n) / (16.0 * h * n)
  return q.to(dtype), cache, table.expand(batch, width), torch.full((batch,), length, dtype=torch.int32, device=DEV)


def _off(q, cache, table, lens, out, which):
  """Largest error of the result of sequence `which` in units of its bar."""
  h, n, d = q.shape[1:]
  kvh, dtype, page = cache.num_kv_heads, q.dtype, cache.page_size
  length = int(lens[which])
  k, v = (x[0].double() for x in cache.read(table[which:which + 1], lens[which:which + 1], length, dtype=dtype))
  half = torch.finfo(dtype).eps / 2
  at = torch.arange(length, device=DEV)
  exps = torch.exp2(cache.v_exponent[table[which, at // page].long(), :, at % page].T.double())
  q = q[which].double().view(kvh, -1, d)
  seen = (at <= length - n + torch.arange(n, device=DEV)[:, None]).repeat(h // kvh, 1)
  s = (q @ k.transpose(1, 2)).masked_fill(~seen, -torch.inf)
  ds = (2.0 ** -19 * (q.abs() @ k.abs().transpose(1, 2)) + 2.0 ** -17 * q.abs().amax(-1, keepdim=True) * k.abs().sum(-1)[:, None]).amax(-1)
  p = torch.softmax(s, -1)
  want, a = p @ v, p @ v.abs()
  low = 2.0 ** -29 * (p * exps[:, None]).amax(-1, keepdim=True) * (seen.double() @ (v.abs() / exps[..., None]))
  p_half = 2.0 ** -11 + (2.0 ** -9 if dtype == torch.bfloat16 else 0.0)
  bar = (p_half + 2.0 ** -12 + 2 * ds[..., None]) * a + low + half * want.abs() + 2.0 ** -25
  got = out[which].double().view(kvh, -1, d)
  assert torch.isfinite(got).all()
  return float(((got - want).abs() / bar).max())


def _check(*args):
  q, cache, table, lens = _peaked(*args)
  attend = sa.make_splash_cached()
  out = attend(q, cache, table, lens)
  last = len(lens) - 1
  alone = attend(q[last:], cache, table[last:], lens[last:])  # cut elsewhere, into many pieces
  sa.check_device_status()
  off = _off(q, cache, table, lens, out, 0), _off(q, cache, table, lens, out, last), _off(q[last:], cache, table[last:], lens[last:], alone, 0)
  assert max(off) <= 1, off


# keys, gap, spread, which key
CASES = [(8192, 8.0, 0.0, 0), (32768, 11.0, 0.5, 5), (32768, 10.4, 0.0, -20000), (20000, 9.0, 1.0, -2)]


# Rows = h / kvh * n.  Up to 16 are served by the kernel whose MMA rows are keys.
@pytest.mark.gpu
@pytest.mark.parametrize("d,dtype", FORMS, ids=str)
@pytest.mark.parametrize("h,kvh,n,batch", [(1, 1, 1, 150), (8, 2, 2, 75), (8, 1, 1, 5)])
@pytest.mark.parametrize("keys", CASES, ids=str)
def test_gpu_few_rows(d, dtype, h, kvh, n, batch, keys):
  _check(d, dtype, h, kvh, n, batch, *keys)


@pytest.mark.gpu
@pytest.mark.parametrize("d,dtype", FORMS, ids=str)
def test_gpu_16_rows(d, dtype):
  _check(d, dtype, 16, 1, 1, 150, *CASES[1])


# Rows as the MMA's rows, with 4, 2 and 1 copies of them, and two tiles of rows.
@pytest.mark.gpu
@pytest.mark.parametrize("d,dtype", FORMS, ids=str)
@pytest.mark.parametrize("h,kvh,n,batch", [(20, 1, 1, 150), (16, 2, 7, 75), (100, 1, 1, 150), (48, 2, 8, 40)])
@pytest.mark.parametrize("keys", CASES, ids=str)
def test_gpu_many_rows(d, dtype, h, kvh, n, batch, keys):
  _check(d, dtype, h, kvh, n, batch, *keys)
