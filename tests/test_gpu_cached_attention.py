"""Attention over the paged cache against the definition in 64 bits.

Bars, per number of the result, with p the softmax weights and A = sum_j p_j |v_j|:
  * P is rounded once (16 bits: half a step h, bf16 2^-8, f16 2^-11; 8-bit caches: two terms of e4m3, 2^-4 * 2^-4, or for f16
    three, and below their range half a step of the subnormals, 2^-10 where the largest 2^ev p is 32 or more, times the codes
    of the values), the result once (h);
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
           spread=1.0, capacity=0, fade=0):
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
  if fade:  # other sizes from one sequence, and one row, to the next
    q = q * torch.exp2(-((torch.arange(b * h, device=DEV) * 5).view(b, h, 1, 1) % fade).float()).to(dtype)
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
  p_half = (2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -12) if quantized else half
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
@pytest.mark.parametrize("case", [
    dict(h=16, n=1, lengths=[9000, 130, 1]), dict(h=3, n=4, lengths=[9000, 500, 3], counts=[4, 2, 4]),
    dict(h=2, n=7, lengths=[8500, 300, 7], parents=[-1, 0, 0, 1, 1, 2, -1]),
    dict(h=4, n=4, lengths=[9500, 300, 2], window=8200, sinks=5, cap=6.0),
], ids=lambda c: f"h{c['h']}n{c['n']}")
@pytest.mark.parametrize("page", [16, 256])
def test_gpu_up_to_16_rows_against_long_contexts(case, page):
  _check(b=3, kvh=1, d=128, dtype=torch.bfloat16, quantized=True, page=page, fade=5, **case)


@pytest.mark.gpu
@pytest.mark.parametrize("d,dtype,quantized", [(128, torch.bfloat16, True), (64, torch.float16, True), (128, torch.bfloat16, False)], ids=str)
@pytest.mark.parametrize("h,n", [(8, 1), (4, 4), (8, 3), (6, 9), (12, 10)])
def test_gpu_many_short_sequences(d, dtype, quantized, h, n):
  """A CTA goes through many units of one or two tiles: what it keeps of a unit is not the next one's."""
  _check(b=700, h=h, kvh=1, n=n, d=d, dtype=dtype, quantized=quantized, page=64, lengths=[(i * 53) % 200 for i in range(700)], fade=11)


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


def _serving(b, h, kvh, n, d, dtype, quantized, page, lengths, seed=0):
  """q, a cache that holds keys and values of all sequences, its page table and lengths."""
  g = torch.Generator(device=DEV).manual_seed(seed)
  width = -(-max(lengths) // page)
  cache = sa.make_kv_cache(b * width, kvh, d, page_size=page, dtype=dtype, quantized=quantized, device=DEV)
  table = torch.randperm(b * width, generator=torch.Generator().manual_seed(seed)).view(b, width).to(torch.int32).to(DEV)
  lens = torch.tensor(lengths, dtype=torch.int32, device=DEV)
  k, v = (torch.randn(b, kvh, max(lengths), d, generator=g, device=DEV).to(dtype) for _ in range(2))
  cache.write(k, v, table, torch.zeros_like(lens), counts=lens)
  q = (torch.randn(b, h, n, d, generator=g, device=DEV) * d ** -0.5).to(dtype)
  return q, cache, table, lens


LAYOUTS = [(8, 2, 1, True), (8, 2, 1, False), (8, 1, 5, True), (4, 1, 30, False)]  # heads, kv heads, new tokens, 8 bit


@pytest.mark.gpu
@pytest.mark.parametrize("h,kvh,n,quantized", LAYOUTS)
def test_gpu_layouts_of_the_arguments(h, kvh, n, quantized):
  b, d = 3, 128
  q, cache, table, lens = _serving(b, h, kvh, n, d, torch.bfloat16, quantized, 16, [300, 64, 129])
  attend = sa.make_splash_cached(window_left=200, num_sinks=3)
  want, (want_lse,) = attend(q, cache, table, lens, save_residuals=True)
  fused = torch.zeros(b, n, h + 3, d, dtype=q.dtype, device=DEV)
  fused[:, :, 2:h + 2] = q.transpose(1, 2)
  shifted = torch.zeros(q.numel() + 1, dtype=q.dtype, device=DEV)[1:].view(q.shape)
  shifted.copy_(q)
  wide = torch.full((b, 2 * table.shape[1] + 5), -1, dtype=torch.int32, device=DEV)
  wide[:, 3:3 + table.shape[1]] = table
  every = torch.zeros(2 * b, dtype=torch.int32, device=DEV)
  every[::2] = lens
  columns = wide[:, 3:3 + table.shape[1]]
  transposed = table.T.contiguous().T
  for q_view, table_view, lens_view in ((fused[:, :, 2:h + 2].transpose(1, 2), table, lens), (shifted, columns, lens),
                                        (q, transposed, every[::2]), (q, columns, lens)):
    for _ in range(2):  # as a new class of calls, and as a known one
      got, (lse,) = attend(q_view, cache, table_view, lens_view, save_residuals=True)
      assert torch.equal(got, want) and torch.equal(lse, want_lse)
  # Several sequences of one length, one page table, one tree.
  same = attend(q, cache, table[1:2].expand(b, -1), lens[1:2].expand(b))
  each = attend(q, cache, table[1:2].repeat(b, 1), lens[1:2].repeat(b))
  assert torch.equal(same, each) and torch.equal(same[1], want[1])
  chain = torch.arange(-1, n - 1, dtype=torch.int32, device=DEV)
  trees = attend(q, cache, table, lens, parents=chain)
  assert torch.equal(trees, attend(q, cache, table, lens, parents=chain.expand(b, n)))
  assert torch.equal(trees, attend(q, cache, table, lens, parents=chain.repeat(2 * b, 1)[::2]))
  # One sequence without a batch, and a batch of none.
  one, (one_lse,) = attend(q[1], cache, table[1:2], lens[1:2], save_residuals=True)
  assert torch.equal(one, want[1]) and torch.equal(one_lse, want_lse[1])
  assert attend(q[:0], cache, table[:0], lens[:0]).shape == (0, h, n, d) and attend(q[:, :, :0], cache, table, lens).shape == (b, h, 0, d)
  # No page at all: no key is seen.
  out, (lse,) = attend(q, cache, table[:, :0], lens, save_residuals=True)
  assert not out.any() and (lse == np.float32(sa.DEFAULT_MASK_VALUE)).all()
  sa.check_device_status()


@pytest.mark.gpu
@pytest.mark.parametrize("h,kvh,n,quantized", LAYOUTS)
def test_gpu_one_sequence_alone_and_in_a_batch(h, kvh, n, quantized):
  """A sequence's numbers do not depend on the others beyond the order in which its parts are added."""
  q, cache, table, lens = _serving(4, h, kvh, n, 128, torch.bfloat16, quantized, 64, [40, 128, 77, 100])
  attend = sa.make_splash_cached()
  both = attend(q, cache, table, lens)
  for i in range(4):  # sequences of one tile of keys: whole in any batch
    assert torch.equal(attend(q[i], cache, table[i:i + 1], lens[i:i + 1]), both[i])
  # The same sequence twice, in one batch.
  twice = attend(q[[2, 2, 0]], cache, table[[2, 2, 0]], lens[[2, 2, 0]])
  assert torch.equal(twice[0], twice[1]) and torch.equal(twice[0], both[2]) and torch.equal(twice[2], both[0])


@pytest.mark.gpu
@pytest.mark.parametrize("h,kvh,n,quantized", LAYOUTS)
def test_gpu_streams_and_graphs(monkeypatch, h, kvh, n, quantized):
  monkeypatch.delenv("SPLASH_CHECK_STATUS", raising=False)  # (a check after every call cannot be captured)
  q, cache, table, lens = _serving(5, h, kvh, n, 128, torch.bfloat16, quantized, 32, [2000, 700, 40, 1999, 1234])
  attend = sa.make_splash_cached()
  shorter = torch.clamp(lens - 600, min=n)
  want, want_short = attend(q, cache, table, lens), attend(q, cache, table, shorter)
  torch.cuda.synchronize()
  # Two calls at once.
  sides = [torch.cuda.Stream() for _ in range(2)]
  got = [[], []]
  for _ in range(20):
    for i, side in enumerate(sides):
      with torch.cuda.stream(side):
        got[i].append(attend(q, cache, table, shorter if i else lens))
  torch.cuda.synchronize()
  assert all(torch.equal(x, want) for x in got[0]) and all(torch.equal(x, want_short) for x in got[1])
  # Two graphs of one memory pool; lengths and new tokens change between replays.
  q_in, lens_in = q.clone(), lens.clone()
  graphs, outs = [], []
  for _ in range(2):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, pool=graphs[0].pool() if graphs else None):
      outs.append(attend(q_in, cache, table, lens_in))
    graphs.append(graph)
  for graph, out in list(zip(graphs, outs)) * 2:
    lens_in.copy_(shorter)
    graph.replay()
    assert torch.equal(out, want_short)
    lens_in.copy_(lens)
    graph.replay()
    assert torch.equal(out, want)
  sa.check_device_status()


@pytest.mark.gpu
@pytest.mark.parametrize("quantized", [False, True])
@pytest.mark.parametrize("window,sinks", [(None, 0), (90, 4)])
def test_gpu_a_run_of_all_operators(quantized, window, sinks):
  """Prompt through the block-sparse kernels, then tokens one by one, then a drafted chain, through cache and cached attention:
  positions, cache and window mean the same on either side."""
  b, h, kvh, d, prompt, steps, drafted = 2, 8, 2, 128, 256, 5, 6
  total = prompt + steps + drafted
  g = torch.Generator(device=DEV).manual_seed(1)
  raw_q, raw_k, v = (torch.randn(b, x, total, d, generator=g, device=DEV).to(torch.bfloat16) for x in (h, kvh, kvh))
  turn = sa.make_rotary(d, (16, 24, 24), q_scale=d ** -0.5)
  positions = torch.arange(total, dtype=torch.int32, device=DEV).expand(3, total).contiguous()
  q, k = turn(raw_q, raw_k, positions)
  cache = sa.make_kv_cache(2 * (-(-total // 64)), kvh, d, page_size=64, quantized=quantized, device=DEV)
  table = torch.arange(cache.num_pages, dtype=torch.int32, device=DEV).view(-1, 2).T.contiguous()
  at = lambda x: torch.full((b,), x, dtype=torch.int32, device=DEV)
  attend = sa.make_splash_cached(window_left=window, num_sinks=sinks)
  outs = []
  cache.write(k[:, :, :prompt], v[:, :, :prompt], table, at(0))
  mask = (sa.CausalMask((prompt, prompt)) if window is None
          else sa.LocalMask((prompt, prompt), (window, 0), 0, num_sinks=sinks))
  dense = sa.make_splash_mha(mask)(*(x[:, :, :prompt].contiguous() for x in (q, k, v)))
  outs.append(attend(q[:, :, :prompt].contiguous(), cache, table, at(prompt)))
  for t in range(prompt, prompt + steps):
    one_q, one_k = turn(raw_q[:, :, t:t + 1], raw_k[:, :, t:t + 1], positions[:, t:t + 1].contiguous())
    assert torch.equal(one_q, q[:, :, t:t + 1]) and torch.equal(one_k, k[:, :, t:t + 1])
    cache.write(one_k, v[:, :, t:t + 1], table, at(t))
    outs.append(attend(one_q, cache, table, at(t + 1)))
  cache.write(k[:, :, -drafted:], v[:, :, -drafted:], table, at(total - drafted))
  chain = torch.arange(-1, drafted - 1, dtype=torch.int32, device=DEV)
  outs.append(attend(q[:, :, -drafted:].contiguous(), cache, table, at(total), parents=chain))
  sa.check_device_status()
  kk, vv = cache.read(table, at(total), total)
  if not quantized:
    assert torch.equal(kk, k) and torch.equal(vv, v)
  got = torch.cat(outs, 2).double()
  for i in range(b):
    codes = exps = None
    if quantized:
      pos = torch.arange(total, device=DEV)
      exps = torch.exp2(cache.v_exponent[table[i, pos // 64].long(), :, pos % 64].T.double())
      codes = vv[i].double().abs() / exps[..., None]
    (want, a, low), _, ds, _ = _want(q[i], kk[i].double(), vv[i].double(), codes, exps, _visible(total, total, total, None, window, sinks), None)
    half = 2.0 ** -8
    bar = (half + 2.0 ** -12 + 2 * ds[..., None]) * a + low + half * want.abs() + 2.0 ** -25
    assert float(((got[i] - want).abs() / bar).max()) <= 1
    if not quantized:  # the block-sparse kernels: the same roundings of the same numbers
      assert float(((dense[i].double() - want[:, :prompt]).abs() / bar[:, :prompt]).max()) <= 1


@pytest.mark.gpu
@pytest.mark.parametrize("d,dtype,quantized", [(128, torch.bfloat16, False), (128, torch.bfloat16, True)])
def test_gpu_pages_behind_four_gigabytes(d, dtype, quantized):
  """Caches whose last pages lie behind 2^32 bytes, and 2^31 numbers, of either buffer."""
  kvh, page = 8, 256
  pages = (1 << 32) // (kvh * page * d * (1 if quantized else 2)) + 4
  make = lambda size, dt: torch.empty(size, dtype=dt, device=DEV)
  exps = [make((pages, kvh, page), torch.int8) for _ in range(2)] if quantized else []
  far = sa.KVCache(*(make((pages, kvh, page, d), torch.float8_e4m3fn if quantized else dtype) for _ in range(2)), *exps)
  near = sa.make_kv_cache(4, kvh, d, page_size=page, dtype=dtype, quantized=quantized, device=DEV)
  g = torch.Generator(device=DEV).manual_seed(0)
  k, v = (torch.randn(2, kvh, 500, d, generator=g, device=DEV).to(dtype) for _ in range(2))
  q = (torch.randn(2, 4 * kvh, 1, d, generator=g, device=DEV) * d ** -0.5).to(dtype)
  start = torch.zeros(2, dtype=torch.int32, device=DEV)
  lens = torch.tensor([500, 300], dtype=torch.int32, device=DEV)
  outs = []
  for cache, last in ((far, pages - 1), (near, 3)):
    table = torch.tensor([[last, last - 2], [last - 1, last - 3]], dtype=torch.int32, device=DEV)
    cache.write(k, v, table, start, counts=lens)
    outs.append((sa.make_splash_cached()(q, cache, table, lens), *cache.read(table, lens, 500)))
  sa.check_device_status()
  # (what no token was written to is not read back as anything but zeros)
  assert all(torch.equal(x, y) for x, y in zip(*outs))


@pytest.mark.gpu
def test_gpu_failure_surfaces_at_the_next_call_and_clears(monkeypatch):
  """As test_gpu_status.py: no kernel is made to time out, the word is set from the host."""
  from splash_attention_mgpu import _ffi
  from splash_attention_mgpu import splash_attention as api
  monkeypatch.delenv("SPLASH_CHECK_STATUS", raising=False)
  for quantized in (False, True):
    q, cache, table, lens = _serving(1, 4, 1, 1, 128, torch.bfloat16, quantized, 64, [300])
    attend = sa.make_splash_cached()
    good = attend(q, cache, table, lens)
    torch.cuda.synchronize()
    sa.check_device_status()
    api._status_word(torch.device(DEV)).copy_(torch.tensor([1, 9, 3, 5], dtype=torch.int32))
    attend(q, cache, table, lens)  # returns at entry; its output is not valid
    torch.cuda.synchronize()
    with pytest.raises(_ffi.SplashLibraryError, match="wait site 9, block 3, step 5"):
      attend(q, cache, table, lens)
    again = attend(q, cache, table, lens)
    torch.cuda.synchronize()
    sa.check_device_status()
    assert torch.equal(again, good)


def test_cached_attention_refusals():
  for kw in (dict(window_left=-1), dict(num_sinks=-1), dict(attn_logits_soft_cap=0.0), dict(attn_logits_soft_cap=-3.0),
             dict(attn_logits_soft_cap=math.inf), dict(attn_logits_soft_cap=math.nan)):
    with pytest.raises(ValueError):
      sa.make_splash_cached(**kw)
  attend = sa.make_splash_cached(num_sinks=1 << 40, window_left=1 << 40)
  cache = sa.make_kv_cache(2, 1, 64, device="cpu")
  q, table, lens = torch.zeros(1, 2, 1, 64, dtype=torch.bfloat16), torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
  with pytest.raises(RuntimeError, match="CUDA"):
    attend(q, cache, table, lens)
  for bad in ((None, cache, table, lens), (q, (cache.k, cache.v), table, lens), (q, cache, [[0, 1]], lens), (q, cache, table, 1)):
    with pytest.raises(TypeError):
      attend(*bad)
  with pytest.raises(NotImplementedError, match="backward"):
    attend(q.requires_grad_(True), cache, table, lens)


@pytest.mark.gpu
def test_gpu_cached_attention_refusals():
  q, cache, table, lens = _serving(2, 4, 2, 3, 64, torch.bfloat16, False, 16, [20, 30])
  attend = sa.make_splash_cached()
  good = attend(q, cache, table, lens)
  codes = sa.make_kv_cache(4, 2, 64, page_size=16, quantized=True, device=DEV)
  parents = torch.full((3,), -1, dtype=torch.int32, device=DEV)
  for bad, kw, error in (
      ((q.float(), cache, table, lens), {}, NotImplementedError), ((q.float(), codes, table, lens), {}, NotImplementedError),
      ((q.half(), cache, table, lens), {}, ValueError), ((q[:, :3], cache, table, lens), {}, ValueError),
      ((q[:, :0], cache, table, lens), {}, ValueError), ((q[..., :32], cache, table, lens), {}, ValueError),
      ((q[0, 0], cache, table, lens), {}, ValueError), ((q[None], cache, table, lens), {}, ValueError),
      ((q, cache, table[:1], lens), {}, ValueError), ((q, cache, table[0], lens), {}, ValueError),
      ((q, cache, table.long(), lens), {}, ValueError), ((q, cache, table, lens.long()), {}, ValueError),
      ((q, cache, table, lens[:1]), {}, ValueError), ((q, cache, table.cpu(), lens), {}, ValueError),
      ((q, cache, table, lens.cpu()), {}, ValueError), ((q, cache, table, lens), dict(counts=lens[:1]), ValueError),
      ((q, cache, table, lens), dict(parents=parents[:2]), ValueError), ((q, cache, table, lens), dict(parents=parents.long()), ValueError),
      ((q, cache, table, lens), dict(parents=parents.expand(3, 3)), ValueError), ((q, cache, table, lens), dict(parents=[-1] * 3), TypeError),
      ((q.repeat(1, 1, 43, 1), cache, table, lens), dict(parents=parents.repeat(43)), NotImplementedError),
      ((q.cpu(), cache, table, lens), {}, RuntimeError)):
    for _ in range(2):
      with pytest.raises(error):
        attend(*bad, **kw)
  with pytest.raises(Exception, match="sizes must be positive"):
    attend(q, sa.make_kv_cache(0, 2, 64, page_size=16, device=DEV), table, lens)
  leaf = q.clone().requires_grad_(True)
  with torch.no_grad():
    assert torch.equal(attend(leaf, cache, table, lens), good)
  assert torch.equal(attend(q, cache, table, lens), good)
