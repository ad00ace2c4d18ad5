"""The paged cache: what is written and read, against indexing and casts in plain torch.  Copies, codes and exponents are
equal; what an 8-bit cache gives back is off by half a step of e4m3, 2^-4 of the number (2^-10 * 2^e among the small)."""

import numpy as np
import pytest
import torch

import splash_attention_mgpu as sa

DEV = "cuda:0"


def _table(b, width, pages, seed=0):
  perm = torch.randperm(pages, generator=torch.Generator().manual_seed(seed))[:b * width]
  return perm.view(b, width).to(torch.int32).to(DEV)


def _pow2(e):
  """2^e in 64 bits, exactly (a power on the device is not)."""
  return torch.from_numpy(np.ldexp(1.0, e.cpu().numpy().astype(np.int64))).to(e.device)


def _quantise(x):
  """Codes and exponents of rows: the smallest e in [-64, 120] with max|x| <= 448 * 2^e."""
  top = x.double().abs().amax(-1).cpu().numpy()
  e = np.full(top.shape, -64, np.int64)
  for _ in range(184):
    e += (top > np.ldexp(448.0, e)) & (e < 120)
  e = torch.from_numpy(e).to(x.device)
  return (x.double() * _pow2(-e)[..., None]).float().to(torch.float8_e4m3fn), e.to(torch.int8)


def _new(b, h, n, d, dtype, layout, seed=0):
  g = torch.Generator(device=DEV).manual_seed(seed)
  scale = torch.exp2(torch.randint(-12, 6, (b, n, 2 * h, 1), generator=g, device=DEV).float())
  x = (torch.randn(b, n, 2 * h, d, generator=g, device=DEV) * scale).to(dtype)
  k, v = x[:, :, :h].transpose(1, 2), x[:, :, h:].transpose(1, 2)
  return (k, v) if layout == "fused" else (k.contiguous(), v.contiguous())


@pytest.mark.gpu
@pytest.mark.parametrize("quantized", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("b,h,n,d,page,layout", [(1, 1, 1, 64, 16, "plain"), (3, 2, 77, 128, 16, "fused"), (2, 8, 1, 128, 64, "fused"),
                                                 (5, 3, 33, 64, 128, "plain"), (2, 4, 300, 128, 256, "plain")])
def test_gpu_what_is_written_is_read(quantized, dtype, b, h, n, d, page, layout):
  width = 3 + (n + 40) // page
  cache = sa.make_kv_cache(b * width + 2, h, d, page_size=page, dtype=dtype, quantized=quantized, device=DEV)
  for x in (cache.k, cache.v):
    x.view(torch.uint8).fill_(0x11)
  table = _table(b, width, cache.num_pages)
  start = torch.tensor([(17 * i) % 40 for i in range(b)], dtype=torch.int32, device=DEV)
  counts = torch.tensor([n - (i * n) // b if i else n for i in range(b)], dtype=torch.int32, device=DEV)
  k, v = _new(b, h, n, d, dtype, layout)
  want = {}
  for name, x in (("k", k), ("v", v)):
    codes, exps = _quantise(x) if quantized else (x, None)
    buf = getattr(cache, name).view(torch.uint8).clone()
    ebuf = getattr(cache, name + "_exponent").clone() if quantized else None
    for i in range(b):
      for t in range(int(counts[i])):
        at = int(start[i]) + t
        pg, slot = int(table[i, at // page]), at % page
        buf[pg, :, slot] = codes[i, :, t].contiguous().view(torch.uint8)
        if quantized:
          ebuf[pg, :, slot] = exps[i, :, t]
    want[name] = (buf, ebuf)
  cache.write(k, v, table, start, counts=counts)
  for name in ("k", "v"):
    assert torch.equal(getattr(cache, name).view(torch.uint8), want[name][0]), name  # rows beside the new ones stay as they were
    if quantized:
      assert torch.equal(getattr(cache, name + "_exponent"), want[name][1])
  # Read back: zeros behind the end, the tokens as they were stored.
  max_len = int((start + counts).max()) + 5
  got = cache.read(table, start + counts, max_len, dtype=dtype)
  for name, x, y in (("k", k, got[0]), ("v", v, got[1])):
    assert y.shape == (b, h, max_len, d) and y.dtype == dtype and y.is_contiguous()
    for i in range(b):
      s, m = int(start[i]), int(counts[i])
      assert not y[i, :, s + m:].any()
      new, stored = x[i, :, :m], y[i, :, s:s + m]
      if not quantized:
        assert torch.equal(new, stored)
        continue
      codes, e = _quantise(new)
      assert torch.equal(stored, (codes.double() * _pow2(e)[..., None]).to(dtype))
      off = (stored.double() - new.double()).abs()
      # (f16 has subnormals: what the scale takes below them is rounded once more, by at most 2^-25.)
      assert (off <= 2.0 ** -4 * new.double().abs() + 2.0 ** -10 * _pow2(e)[..., None] + 2.0 ** -25).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_gpu_extreme_rows(dtype):
  fi = torch.finfo(dtype)
  rows = torch.zeros(12, 64, dtype=dtype, device=DEV)
  rows[1, 3] = fi.max
  rows[2, 5] = -fi.max
  rows[3, :] = fi.smallest_normal
  rows[4, 7] = fi.smallest_normal * fi.eps  # the smallest subnormal
  rows[5, :] = 448.0
  rows[6, 0], rows[6, 1] = 449.0 if dtype == torch.float16 else 450.0, 2.0
  rows[7, 9] = float("inf")
  rows[8, 2], rows[8, 3] = float("nan"), 1.0
  rows[9, :] = -0.0
  rows[10, 0], rows[10, 1] = 1.0, 2.0 ** -10
  rows[11, 33] = -float("inf")
  cache = sa.make_kv_cache(1, 1, 64, page_size=16, quantized=True, device=DEV)
  table, zero = torch.zeros(1, 1, dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
  cache.write(rows[None, None], rows[None, None], table, zero)
  k, v = cache.read(table, zero + 12, 12, dtype=dtype)
  assert torch.equal(k.view(torch.int16), v.view(torch.int16))
  k = k[0, 0]
  for i in (7, 8, 11):
    assert k[i].isnan().all() and int(cache.k_exponent[0, 0, i]) == -128
  fine = [i for i in range(12) if i not in (7, 8, 11)]
  codes, e = _quantise(rows[fine])
  assert torch.equal(cache.k_exponent[0, 0, :12][fine], e)
  assert torch.equal(k[fine], (codes.double() * _pow2(e)[:, None]).to(dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("quantized", [False, True])
def test_gpu_pages_that_are_none(quantized):
  cache = sa.make_kv_cache(4, 2, 64, page_size=16, quantized=quantized, device=DEV)
  table = torch.tensor([[2, -1, 7, 0], [4, 1, 1 << 30, -(1 << 31)]], dtype=torch.int32, device=DEV)  # 4 pages: 7, 4 and the last two are none
  k, v = _new(2, 2, 90, 64, torch.bfloat16, "plain")
  before = cache.k.view(torch.uint8)[3].clone()
  cache.write(k, v, table, torch.tensor([0, -5], dtype=torch.int32, device=DEV))  # tokens in front of and behind the table too
  got, _ = cache.read(table, torch.tensor([70, 90], dtype=torch.int32, device=DEV), 90)
  torch.cuda.synchronize()
  assert torch.equal(cache.k.view(torch.uint8)[3], before)
  assert got[0, :, :16].any() and not got[0, :, 16:48].any() and got[0, :, 48:64].any() and not got[0, :, 64:].any()
  assert not got[1, :, :16].any() and got[1, :, 16:32].any() and not got[1, :, 32:].any()


@pytest.mark.gpu
def test_gpu_cache_on_another_stream_captured_and_empty_calls():
  cache = sa.make_kv_cache(8, 2, 128, page_size=16, quantized=True, device=DEV)
  table = _table(2, 4, 8)
  start = torch.tensor([3, 20], dtype=torch.int32, device=DEV)
  k, v = _new(2, 2, 9, 128, torch.bfloat16, "fused")
  cache.write(k[:, :, :0], v[:, :, :0], table, start)
  assert cache.read(table, start, 0)[0].shape == (2, 2, 0, 128)
  side = torch.cuda.Stream()
  side.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(side):
    cache.write(k, v, table, start)
    want = cache.read(table, start + 9, 40)
  torch.cuda.current_stream().wait_stream(side)
  graph = torch.cuda.CUDAGraph()
  ends = start + 9
  with torch.cuda.graph(graph):
    cache.write(k, v, table, start)
    got = cache.read(table, ends, 40)
  cache.k.view(torch.uint8).zero_()
  cache.v.view(torch.uint8).zero_()
  graph.replay()
  torch.cuda.synchronize()
  for i, (s, e) in enumerate(((3, 12), (20, 29))):
    assert torch.equal(got[0][i, :, s:e], want[0][i, :, s:e]) and torch.equal(got[1][i, :, s:e], want[1][i, :, s:e])


def test_cache_refusals():
  make = lambda **kw: sa.make_kv_cache(**{**dict(num_pages=2, num_kv_heads=1, head_dim=64, device="cpu"), **kw})
  for kw, error in ((dict(page_size=48), ValueError), (dict(head_dim=96), NotImplementedError), (dict(num_kv_heads=0), ValueError),
                    (dict(num_pages=-1), ValueError), (dict(dtype=torch.float32), NotImplementedError)):
    with pytest.raises(error):
      make(**kw)
  codes = make(quantized=True)
  with pytest.raises(ValueError, match="exponents"):
    sa.KVCache(codes.k, codes.v)
  with pytest.raises(ValueError, match="exponents"):
    sa.KVCache(make().k, make().v, codes.k_exponent, codes.v_exponent)
  with pytest.raises(ValueError):
    sa.KVCache(make().k, make(num_pages=3).v)
  with pytest.raises(ValueError, match="contiguous"):
    sa.KVCache(make(num_pages=4).k[::2], make(num_pages=4).v[::2])
  cache, x = make(), torch.zeros(1, 1, 3, 64, dtype=torch.bfloat16)
  table, start = torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
  with pytest.raises(RuntimeError, match="CUDA"):
    cache.write(x, x, table, start)
  with pytest.raises(RuntimeError, match="CUDA"):
    cache.read(table, start, 3)
  for bad in ((x, x[..., :32], table, start), (x, x.half(), table, start), (x, x, table.long(), start), (x, x, table, start[:0]),
              (x, x, table[0], start), (x.expand(2, 1, 3, 64), x.expand(2, 1, 3, 64), table, start)):
    with pytest.raises(ValueError):
      cache.write(*bad)
  with pytest.raises(ValueError):
    cache.read(table, start, -1)
  with pytest.raises(TypeError):
    cache.read([[0]], start, 1)
