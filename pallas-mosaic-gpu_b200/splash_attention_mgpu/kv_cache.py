"""A paged cache of keys and values for serving, 16-bit or quantised as it is written.

    cache = make_kv_cache(num_pages=4096, num_kv_heads=8, head_dim=128, page_size=64, quantized=True)
    cache.write(k, v, page_table, start)             # tokens start[b], start[b] + 1, ... of every sequence
    k, v = cache.read(page_table, lengths, max_len)  # [B, kv_heads, max_len, head_dim], zeros behind a sequence's end

Token t of sequence b lies in page `page_table[b, t // page_size]`.  A page id outside [0, num_pages) and a token behind
the table's end stand for no page: nothing is written there, zeros are read and attention does not see it.  The slots
that one write fills have to differ (a page shared by two sequences is written by one of them).

An 8-bit cache holds e4m3 codes and one exponent e per (token, head): x = code * 2^e, with e the smallest whole number in
[-64, 120] for which max|x| <= 448 * 2^e.  Storing rounds once, by at most 2^-4 of the number (or 2^-10 * 2^e);
reading back adds nothing where the 16-bit type has that number: f16 rounds what lies among its subnormals once more, and
what was rounded to 2^16 (f16, from 63488 on) or 2^128 (bf16, from 0.96875 * 2^128 on) reads as infinity, while attention
over the cache has it as the finite number it is.  A row that holds an infinity or NaN reads back as NaN throughout.
Gradients and forward-mode derivatives do not pass through a cache.

No counterpart in the reference, which attends to contiguous keys.
"""

from __future__ import annotations

import ctypes
import dataclasses

import torch

from . import _ffi
from .splash_attention import _TORCH_DTYPES, _launch, _set_up_status

PAGE_SIZES = (16, 32, 64, 128, 256)
HEAD_DIMS = (64, 128)
CODE_DTYPE = torch.float8_e4m3fn


def _index_tensor(x, name, device, shape):
  """int32 tensor of this shape on the device, as the kernels read it (rows of a table contiguous)."""
  if not isinstance(x, torch.Tensor):
    raise TypeError(f"{name} must be a torch tensor")
  if x.device != device:
    raise ValueError(f"{name} is on {x.device}, the cache is on {device}")
  if x.dtype != torch.int32:
    raise ValueError(f"{name} must be int32, got {x.dtype}")
  if x.ndim != len(shape) or any(n is not None and n != m for n, m in zip(shape, x.shape)):
    raise ValueError(f"{name} must be {['*' if n is None else n for n in shape]}, got {list(x.shape)}")
  return x if x.shape[-1] <= 1 or x.stride(-1) == 1 else x.contiguous()


def _signature(x):
  """What a call depends on of an argument besides its address."""
  if not isinstance(x, torch.Tensor):
    raise TypeError(f"expected a torch tensor, got {type(x).__name__}")
  return x.shape, x.stride(), x.dtype, x.device


def _remember(known: dict, key, value):
  if len(known) >= 256:
    known.clear()
  known[key] = value
  return value


@dataclasses.dataclass(frozen=True, eq=False)
class KVCache:
  """Buffers of a paged cache; `make_kv_cache` allocates them.

  k, v: [num_pages, num_kv_heads, page_size, head_dim], bf16 / f16, or float8_e4m3fn codes
  k_exponent, v_exponent: int8 [num_pages, num_kv_heads, page_size] beside codes, else None
  """

  k: torch.Tensor
  v: torch.Tensor
  k_exponent: torch.Tensor | None = None
  v_exponent: torch.Tensor | None = None
  _calls: dict = dataclasses.field(default_factory=dict, init=False, repr=False)

  def __post_init__(self):
    for x in (self.k, self.v):
      if not isinstance(x, torch.Tensor):
        raise TypeError("k and v must be torch tensors")
    if self.k.ndim != 4 or self.k.shape != self.v.shape or self.k.dtype != self.v.dtype or self.k.device != self.v.device:
      raise ValueError(f"k and v must be alike, [num_pages, num_kv_heads, page_size, head_dim]: {tuple(self.k.shape)}"
                       f" {self.k.dtype}, {tuple(self.v.shape)} {self.v.dtype}")
    if not (self.k.is_contiguous() and self.v.is_contiguous()):
      raise ValueError("the buffers of a cache must be contiguous")
    if self.k.shape[2] not in PAGE_SIZES:
      raise ValueError(f"page_size must be one of {PAGE_SIZES}, got {self.k.shape[2]}")
    if self.k.shape[3] not in HEAD_DIMS:
      raise NotImplementedError(f"the cache supports head dims {HEAD_DIMS}, got {self.k.shape[3]}")
    if self.k.shape[1] < 1:
      raise ValueError("the cache has no heads")
    if self.k.numel() // self.k.shape[3] >= 1 << 31:
      raise ValueError("num_pages * num_kv_heads * page_size must fit in 31 bits")
    if self.quantized:
      for x in (self.k_exponent, self.v_exponent):
        if (not isinstance(x, torch.Tensor) or x.dtype != torch.int8 or x.shape != self.k.shape[:3] or x.device != self.k.device
            or not x.is_contiguous()):
          raise ValueError("an 8-bit cache needs contiguous int8 exponents [num_pages, num_kv_heads, page_size]")
    elif self.k.dtype not in _TORCH_DTYPES:
      raise NotImplementedError(f"caches are bf16, f16 or float8_e4m3fn, got {self.k.dtype}")
    elif self.k_exponent is not None or self.v_exponent is not None:
      raise ValueError("exponents belong to 8-bit caches")
    if self.k.is_cuda:
      _set_up_status(self.k.device)

  @property
  def quantized(self) -> bool:
    return self.k.dtype == CODE_DTYPE

  @property
  def num_pages(self) -> int:
    return self.k.shape[0]

  @property
  def num_kv_heads(self) -> int:
    return self.k.shape[1]

  @property
  def page_size(self) -> int:
    return self.k.shape[2]

  @property
  def head_dim(self) -> int:
    return self.k.shape[3]

  def _params(self, page_table, batch, length, dtype) -> _ffi.SplashCacheParams:
    """The parameter block of a call of this class, without its pointers."""
    if not self.k.is_cuda:
      raise RuntimeError("the cache works only on a CUDA (sm_100a) device; there is no CPU path.")
    if dtype not in _TORCH_DTYPES:
      raise NotImplementedError(f"Only bf16/f16 are supported, got {dtype}")
    if not self.quantized and dtype != self.k.dtype:
      raise ValueError(f"the cache holds {self.k.dtype}, got {dtype}")
    p = _ffi.SplashCacheParams()
    p.quantized = self.quantized
    p.table_stride, p.table_width = page_table.stride(0), page_table.shape[1]
    p.batch, p.len = batch, length
    p.num_pages, p.kv_heads, p.page_size, p.head_dim = self.k.shape
    p.dtype = _TORCH_DTYPES[dtype]
    return p

  def _point(self, p, page_table, lengths) -> None:
    """Addresses of a call: never kept, so that a copy of a cache works on its own buffers."""
    p.k_cache, p.v_cache = self.k.data_ptr(), self.v.data_ptr()
    if p.quantized:
      p.k_exponent, p.v_exponent = self.k_exponent.data_ptr(), self.v_exponent.data_ptr()
    p.page_table, p.lengths = page_table.data_ptr(), lengths.data_ptr()

  def write(self, k, v, page_table, start, *, counts=None) -> None:
    """Stores new tokens: token j of sequence b becomes token start[b] + j of that sequence.

    k, v: [(B,) kv_heads, n, head_dim], bf16 / f16; views whose last dimension is contiguous are read in place
    page_table: int32 [B, pages per sequence]; start: int32 [B]
    counts: int32 [B], how many of the n tokens each sequence has (None: all)
    """
    for x in (k, v, page_table, start):
      if not isinstance(x, torch.Tensor):
        raise TypeError("k, v, page_table and start must be torch tensors")
    # What a call is made of besides its pointers, checked and filled in once per class of calls.
    key = (k.shape, k.stride(), k.dtype, k.device, v.shape, v.stride(), v.dtype, v.device, page_table.shape, page_table.stride(),
           page_table.dtype, page_table.device, start.shape, start.stride(), start.dtype, start.device,
           None if counts is None else _signature(counts))
    template = self._calls.get(key)
    if template is None:
      if k.ndim == 3:
        return self.write(k[None], v[None], page_table, start, counts=counts)
      if k.ndim != 4 or k.shape != v.shape or k.shape[1] != self.num_kv_heads or k.shape[3] != self.head_dim:
        raise ValueError(f"k and v must be [(batch,) {self.num_kv_heads}, n, {self.head_dim}], got {tuple(k.shape)}, {tuple(v.shape)}")
      if k.dtype != v.dtype or k.device != self.k.device or v.device != self.k.device:
        raise ValueError(f"k and v differ from the cache: {k.dtype} on {k.device}, {v.dtype} on {v.device}")
      batch, _, n, _ = k.shape
      device = self.k.device
      as_given = (page_table, start, counts)
      page_table = _index_tensor(page_table, "page_table", device, (batch, None))
      start = _index_tensor(start, "start", device, (batch,))
      if counts is not None:
        counts = _index_tensor(counts, "counts", device, (batch,))
      p = self._params(page_table, batch, n, k.dtype)
      in_place = lambda x: x.stride(-1) == 1 and not any(s % 8 for s in x.stride()[:-1])
      if not (in_place(k) and in_place(v)) or any(x is not y for x, y in zip(as_given, (page_table, start, counts))):
        k, v = (x if in_place(x) else x.clone(memory_format=torch.contiguous_format) for x in (k, v))
        return self.write(k, v, page_table, start, counts=counts)
      p.k_stride, p.v_stride = k.stride()[:3], v.stride()[:3]
      template = _remember(self._calls, key, bytes(p))
    if k.data_ptr() % 16 or v.data_ptr() % 16:
      return self.write(*(x.clone(memory_format=torch.contiguous_format) for x in (k, v)), page_table, start, counts=counts)
    p = _ffi.SplashCacheParams.from_buffer_copy(template)
    self._point(p, page_table, start)
    p.k, p.v = k.data_ptr(), v.data_ptr()
    if counts is not None:
      p.counts = counts.data_ptr()
    rc = _launch(self.k.device, _ffi.load().splash_cache_write, ctypes.byref(p))
    if rc:
      _ffi.check(rc, "cache write")

  def read(self, page_table, lengths, max_len: int, *, dtype=None):
    """The first lengths[b] tokens of every sequence, (k, v) [B, kv_heads, max_len, head_dim] with zeros behind them.

    page_table: int32 [B, pages per sequence]; lengths: int32 [B]; dtype: bf16 (8-bit caches: the default) or f16
    """
    if dtype is None:
      dtype = torch.bfloat16 if self.quantized else self.k.dtype
    device = self.k.device
    page_table = _index_tensor(page_table, "page_table", device, (None, None))
    batch = page_table.shape[0]
    lengths = _index_tensor(lengths, "lengths", device, (batch,))
    max_len = int(max_len)
    if max_len < 0:
      raise ValueError(f"max_len must not be negative, got {max_len}")
    p = self._params(page_table, batch, max_len, dtype)
    self._point(p, page_table, lengths)
    shape = (batch, self.num_kv_heads, max_len, self.head_dim)
    k, v = torch.empty(shape, dtype=dtype, device=device), torch.empty(shape, dtype=dtype, device=device)
    p.k_out, p.v_out = k.data_ptr(), v.data_ptr()
    _ffi.check(_launch(device, _ffi.load().splash_cache_read, ctypes.byref(p)), "cache read")
    return k, v


def make_kv_cache(num_pages: int, num_kv_heads: int, head_dim: int, *, page_size: int = 64, dtype=torch.bfloat16,
                  quantized: bool = False, device="cuda") -> KVCache:
  """An empty cache: 16-bit of `dtype`, or with `quantized` e4m3 codes and exponents (of bf16 or f16 numbers alike)."""
  if num_pages < 0:
    raise ValueError(f"num_pages must not be negative, got {num_pages}")
  shape = (num_pages, num_kv_heads, page_size, head_dim)
  if not quantized:
    return KVCache(torch.zeros(shape, dtype=dtype, device=device), torch.zeros(shape, dtype=dtype, device=device))
  codes = lambda: torch.zeros(shape, dtype=torch.uint8, device=device).view(CODE_DTYPE)
  exponents = lambda: torch.zeros(shape[:3], dtype=torch.int8, device=device)
  return KVCache(codes(), codes(), exponents(), exponents())
