"""Attention over the paged cache against the definition in 64 bits.

Bars, per number of the result, with p the softmax weights and A = sum_j p_j |v_j|:
  * P is rounded once (16 bits: half a step h, bf16 2^-8, f16 2^-11; 8-bit caches: two terms of e4m3, 2^-4 * 2^-4, and below
    their range half a step of the subnormals, 2^-10 where the largest 2^ev p is 32 or more, times the codes of the values),
    the result once (h);
  * the scores are off by dS = 2^-19 sum|q k| + 2^-10 |s| under a soft-cap (tanh.approx) and, 8 bit, 2^-17 max|q| sum|k| (the
    e4m3 terms of q), which moves p by at most 2 dS relative to itself for dS < 0.1; 2^-12 A covers 32-bit sums and ex2.approx.
  logsumexp: dS + 2^-19 (1 + |lse|)."""

import math

import numpy as np
import pytest
import torch

import splash_attention_mgpu as sa

DEV = "cuda:0"


def _visible(length, count, n, parents, window, sinks):
  """[n, length] bool: rows from count on see nothing."""
  count = min(count, length)
  before = length - count
  seen = np.zeros((n, length), bool)
  depth = {}
  for i in range(count):
    chain = [i]
    while True:
      up = chain[-1] - 1 if parents is None else int(parents[chain[-1]])
      if up < 0 or up >= chain[-1]:
        break
      chain.append(up)
    depth[i] = len(chain) - 1
    pos = before + depth[i]
    lo = -1 if window is None else pos - window
    key = np.arange(before)
    seen[i, :before] = (key >= lo) | (key < sinks) if window is not None else True
    for j in chain:
      at = before + depth[j]
      seen[i, before + j] = window is None or at >= lo or at < sinks
  return seen


def _want(q, k, v, codes, exps, seen, cap):
  """One sequence: q [H, n, D], k and v [KVH, L, D] in 64 bits, codes |v 2^-ev| and 2^ev or None."""
  h, n, d = q.shape
  kvh = k.shape[0]
  group = h // kvh
  q = q.double().view(kvh, group * n, d)
  s = q @ k.transpose(1, 2)
  mag = q.abs() @ k.abs().transpose(1, 2)
  ds = 2.0 ** -19 * mag
  if codes is not None:
    ds = ds + 2.0 ** -17 * q.abs().amax(-1, keepdim=True) * k.abs().sum(-1)[:, None]
  if cap:
    s = cap * torch.tanh(s / cap)
    ds = ds + 2.0 ** -10 * s.abs()
  seen = torch.from_numpy(seen).to(q.device).repeat(group, 1)[None].expand(s.shape)
  s = s.masked_fill(~seen, -math.inf)
  any_seen = seen.any(-1)
  lse = torch.logsumexp(s, -1)
  p = torch.where(seen, torch.exp(s - torch.where(any_seen, lse, 0.0)[..., None]), 0.0)
  ds = torch.where(seen, ds, 0.0).amax(-1)
  v = torch.where(seen.any(1)[..., None], v, 0.0)  # (what nobody sees may be anything)
  out = p @ v
  a = p @ v.abs()
  low = torch.zeros_like(a)
  if codes is not None:
    top = (p * exps[:, None]).amax(-1, keepdim=True)
    low = 2.0 ** -15 * top * (seen.double() @ torch.where(seen.any(1)[..., None], codes, 0.0))
  return (x.view(h, n, -1) for x in (out, a, low)), lse.view(h, n), ds.view(h, n), any_seen.view(h, n)


def _check(b, h, kvh, n, d, dtype, quantized, page, lengths, *, counts=None, parents=None, window=None, sinks=0, cap=None, seed=0,
           spread=1.0, capacity=0):
  g = torch.Generator(device=DEV).manual_seed(seed)
  width = -(-max(max(lengths), capacity, 1) // page) + 1
  cache = sa.make_kv_cache(b * width + 2, kvh, d, page_size=page, dtype=dtype, quantized=quantized, device=DEV)
  # Whatever is not written reads as NaN.
  for x in (cache.k, cache.v):
    x.view(torch.uint8).fill_(0x7f if quantized else 0xff)
  if quantized:
    cache.k_exponent.fill_(-128)
    cache.v_exponent.fill_(-128)
  table = torch.randperm(cache.num_pages, generator=torch.Generator().manual_seed(seed))[:b * width].view(b, width).to(torch.int32).to(DEV)
  longest = max(max(lengths), 1)
  k, v = (torch.randn(b, kvh, longest, d, generator=g, device=DEV) for _ in range(2))
  k, v = k.to(dtype), (v * torch.exp2(torch.randint(-3, 4, (b, kvh, longest, 1), generator=g, device=DEV).float()) if quantized else v).to(dtype)
  lens = torch.tensor(lengths, dtype=torch.int32, device=DEV)
  cache.write(k, v, table, torch.zeros_like(lens), counts=lens)
  q = (torch.randn(b, h, n, d, generator=g, device=DEV) * d ** -0.5 * spread).to(dtype)
  news = [n] * b if counts is None else counts
  trees = None
  if parents is not None:
    trees = torch.as_tensor(np.asarray(parents, np.int32), device=DEV)
  # Pages that nobody sees have no valid id.
  bad = torch.tensor([-1, cache.num_pages, 1 << 30, -(1 << 31)], dtype=torch.int32)
  use = table.clone()
  seen = []
  for i in range(b):
    tree = None if parents is None else np.asarray(parents) if np.asarray(parents).ndim == 1 else np.asarray(parents)[i]
    seen.append(_visible(lengths[i], news[i], n, tree, window, sinks))
    for j in range(width):
      if not seen[i][:, j * page:(j + 1) * page].any():
        use[i, j] = bad[j % 4].to(DEV)
  for i in range(b):
    q[i, :, min(news[i], lengths[i]):] = float("nan")  # padding holds anything
  attend = sa.make_splash_cached(window_left=window, num_sinks=sinks, attn_logits_soft_cap=cap)
  cnt = None if counts is None else torch.tensor(counts, dtype=torch.int32, device=DEV)
  out, (lse,) = attend(q, cache, use, lens, counts=cnt, parents=trees, save_residuals=True)
  sa.check_device_status()
  again = attend(q, cache, use, lens, counts=cnt, parents=trees)
  sa.check_device_status()
  assert torch.equal(out, again)
  kk, vv = cache.read(table, lens, longest, dtype=dtype)
  half = torch.finfo(dtype).eps / 2
  p_half = 2.0 ** -8 if quantized else half
  for i in range(b):
    length = lengths[i]
    if length == 0:
      assert not out[i].any() and (lse[i] == np.float32(sa.DEFAULT_MASK_VALUE)).all()
      continue
    codes = exps = None
    if quantized:
      at = torch.arange(length, device=DEV)
      ev = cache.v_exponent[table[i, at // page].long(), :, at % page].T.double()
      exps = torch.exp2(ev)
      codes = vv[i, :, :length].double().abs() / exps[..., None]
    (want, a, low), want_lse, ds, any_seen = _want(torch.nan_to_num(q[i]), kk[i, :, :length].double(), vv[i, :, :length].double(),
                                                   codes, exps, seen[i], cap)
    assert float(ds.max()) < 0.1
    got = out[i].double()
    assert torch.isfinite(got).all()
    bar = (p_half + 2.0 ** -12 + 2 * ds[..., None]) * a + low + half * want.abs() + 2.0 ** -25
    off = ((got - want).abs() / bar).max()
    assert float(off) <= 1, (i, float(off))
    assert not got[~any_seen].any()
    lse_off = (lse[i].double() - want_lse).abs()
    assert (lse[i][~any_seen] == np.float32(sa.DEFAULT_MASK_VALUE)).all()
    assert (lse_off <= ds + 2.0 ** -19 * (1 + want_lse.abs()))[any_seen].all(), float(lse_off[any_seen].max())


def _tree(n, seed, wide=8):
  rng = np.random.default_rng(seed)
  p = np.full(n, -1, np.int32)
  for i in range(1, n):
    p[i] = -1 if rng.random() < 0.15 else rng.integers(max(0, i - wide), i)
  return p


FORMS = [(64, torch.float16, False), (128, torch.bfloat16, False), (64, torch.bfloat16, True), (128, torch.bfloat16, True),
         (128, torch.float16, True), (64, torch.float16, True), (128, torch.float16, False)]


@pytest.mark.gpu
@pytest.mark.parametrize("d,dtype,quantized", FORMS, ids=str)
@pytest.mark.parametrize("case", [
    dict(b=1, h=1, kvh=1, n=1, page=16, lengths=[1]),
    dict(b=1, h=4, kvh=1, n=1, page=64, lengths=[128]),
    dict(b=4, h=8, kvh=2, n=1, page=16, lengths=[1, 127, 0, 900]),
    dict(b=2, h=32, kvh=1, n=1, page=128, lengths=[129, 384]),
    dict(b=3, h=40, kvh=1, n=1, page=32, lengths=[500, 3, 255]),
    dict(b=2, h=128, kvh=1, n=1, page=256, lengths=[511, 700]),
    dict(b=2, h=150, kvh=1, n=1, page=64, lengths=[300, 257]),
    dict(b=70, h=6, kvh=3, n=1, page=16, lengths=[(i * 37) % 400 for i in range(70)]),
    dict(b=1, h=2, kvh=1, n=1, page=64, lengths=[20011]),
    dict(b=3, h=8, kvh=2, n=1, page=32, lengths=[5000, 10, 2500]),
], ids=lambda c: f"b{c['b']}h{c['h']}kv{c['kvh']}len{max(c['lengths'])}")
def test_gpu_one_token(d, dtype, quantized, case):
  _check(d=d, dtype=dtype, quantized=quantized, **case)


@pytest.mark.gpu
@pytest.mark.parametrize("d,dtype,quantized", FORMS[:4], ids=str)
@pytest.mark.parametrize("case", [
    dict(b=3, h=4, kvh=2, n=5, page=16, lengths=[5, 300, 140], counts=[0, 3, 5]),
    dict(b=2, h=8, kvh=1, n=4, page=64, lengths=[2, 1000], counts=[4, 4]),   # fewer tokens in the cache than new ones
    dict(b=1, h=2, kvh=1, n=200, page=32, lengths=[200]),
    dict(b=2, h=2, kvh=2, n=129, page=64, lengths=[700, 129], counts=[129, 100]),
    dict(b=2, h=3, kvh=1, n=50, page=128, lengths=[64, 333], counts=[50, 33]),
    dict(b=1, h=5, kvh=1, n=300, page=16, lengths=[1500]),
], ids=lambda c: f"b{c['b']}h{c['h']}n{c['n']}")
def test_gpu_runs(d, dtype, quantized, case):
  _check(d=d, dtype=dtype, quantized=quantized, **case)


@pytest.mark.gpu
@pytest.mark.parametrize("d,dtype,quantized", FORMS[:4], ids=str)
@pytest.mark.parametrize("case", [
    dict(b=1, h=2, kvh=1, n=7, page=16, lengths=[100], parents=[-1, 0, 0, 1, 1, 2, -1]),
    dict(b=3, h=8, kvh=2, n=48, page=64, lengths=[48, 500, 1000], parents=[_tree(48, i) for i in range(3)]),
    dict(b=2, h=2, kvh=1, n=128, page=16, lengths=[128, 777], parents=[_tree(128, 3), list(range(-1, 127))]),
    dict(b=2, h=4, kvh=2, n=33, page=32, lengths=[250, 40], counts=[20, 33], parents=_tree(33, 5)),
    dict(b=1, h=4, kvh=4, n=64, page=128, lengths=[2000], parents=_tree(64, 6), window=70, sinks=4),
    dict(b=2, h=4, kvh=1, n=20, page=16, lengths=[23, 400], parents=_tree(20, 7, wide=2), window=3, sinks=5),
    dict(b=1, h=2, kvh=1, n=4, page=16, lengths=[50], parents=[0, 7, -9, 2]),  # what is no earlier token is the context
], ids=lambda c: f"b{c['b']}h{c['h']}n{c['n']}")
def test_gpu_trees(d, dtype, quantized, case):
  _check(d=d, dtype=dtype, quantized=quantized, **case)


@pytest.mark.gpu
@pytest.mark.parametrize("d,dtype,quantized", FORMS[:4], ids=str)
@pytest.mark.parametrize("case", [
    dict(n=1, window=100, sinks=4, lengths=[1, 103, 5000]),
    dict(n=1, window=0, sinks=0, lengths=[1, 128, 129]),
    dict(n=3, window=127, sinks=130, lengths=[3, 260, 1000]),
    dict(n=8, window=1000, sinks=0, lengths=[1200, 4097, 8]),
    dict(n=4, window=64, sinks=1000, lengths=[900, 1100, 3000]),
    dict(n=40, window=30, sinks=2, lengths=[40, 333, 2049]),
    dict(n=1, window=1 << 30, sinks=3, lengths=[5, 600, 130]),
], ids=lambda c: f"n{c['n']}w{c['window']}s{c['sinks']}")
@pytest.mark.parametrize("page", [16, 128])
def test_gpu_windows_and_sinks(d, dtype, quantized, case, page):
  _check(b=3, h=4, kvh=2, d=d, dtype=dtype, quantized=quantized, page=page, **case)


@pytest.mark.gpu
@pytest.mark.parametrize("d,dtype,quantized", FORMS[:4], ids=str)
def test_gpu_soft_cap_and_large_logits(d, dtype, quantized):
  _check(b=2, h=8, kvh=2, n=2, d=d, dtype=dtype, quantized=quantized, page=64, lengths=[300, 1000], cap=5.0, spread=4.0)
  _check(b=2, h=8, kvh=2, n=2, d=d, dtype=dtype, quantized=quantized, page=64, lengths=[300, 2000], spread=12.0, seed=3)
