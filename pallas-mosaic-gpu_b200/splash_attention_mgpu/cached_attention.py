"""Attention of new tokens over a paged cache: one token per sequence, a run of tokens, or a tree of drafted ones.

    attend = make_splash_cached(window_left=4095, num_sinks=4)
    cache.write(k, v, page_table, lengths - n)                  # the new tokens' keys and values are in the cache
    out = attend(q, cache, page_table, lengths)                 # q: [B, heads, n, head_dim], pre-scaled
    out = attend(q, cache, page_table, lengths, parents=tree)   # tree: [n] or [B, n]
    out, (lse,) = attend(q, cache, page_table, lengths, save_residuals=True)

The serving counterpart of `make_splash_mha` with `CausalMask` / `LocalMask`: the same window (`LocalMask`'s left side), the
same sinks, soft-cap and treatment of rows that see no key (zeros and lse = mask_value).  Forward only.  What no row of a call
sees may be anything; a value that one of them sees and that is infinite or NaN reaches the others too (0 times it is NaN).  Lengths, page
tables and trees stay on the device; a call synchronises nothing and can be captured into a graph.

No counterpart in the reference, which attends to contiguous keys in multiples of a block.
"""

from __future__ import annotations

import ctypes
import math
import os

import torch
import torch.autograd.forward_ad as forward_ad

from . import _ffi
from .config import DEFAULT_MASK_VALUE
from .kv_cache import KVCache, _index_tensor, _remember, _signature
from .splash_attention import (_TORCH_DTYPES, _launch, _poll_status, _status_host, _status_word, check_device_status)

MAX_TREE = 128


class CachedAttentionKernel:
  """Callable holding window, sinks, soft-cap and mask value; made by `make_splash_cached`."""

  def __init__(self, *, window_left: int | None, num_sinks: int, attn_logits_soft_cap: float | None, mask_value: float):
    self.window_left = window_left
    self.num_sinks = num_sinks
    self.attn_logits_soft_cap = attn_logits_soft_cap
    self.mask_value = mask_value
    self._calls: dict = {}

  def __getstate__(self):
    return {**self.__dict__, "_calls": {}}  # (what is kept of calls lies on their devices)

  def __repr__(self):
    return (f"CachedAttentionKernel(window_left={self.window_left}, num_sinks={self.num_sinks},"
            f" attn_logits_soft_cap={self.attn_logits_soft_cap})")

  def __call__(self, q, cache: KVCache, page_table, lengths, *, counts=None, parents=None, save_residuals: bool = False):
    """out [(B,) heads, n, head_dim], and with `save_residuals` the logsumexp as `(out, (lse,))`.

    q: [B, heads, n, head_dim], or [heads, n, head_dim] for one sequence; pre-scaled
    page_table: int32 [B, pages per sequence]
    lengths: int32 [B], tokens of each sequence in the cache, the new ones included (at most what its pages hold)
    counts: int32 [B], new tokens of each sequence, its first rows of q (None: n); the rows behind them give zeros
    parents: int32 [n] or [B, n], the new tokens as a tree: token i follows token parents[i] < i, or (-1) the last token in
      front of the new ones.  It sees those, its ancestors and itself, and its position is one behind its parent's.
      None: token i follows token i - 1.
    """
    for x in (q, page_table, lengths):
      if not isinstance(x, torch.Tensor):
        raise TypeError("q, page_table and lengths must be torch tensors")
    if not isinstance(cache, KVCache):
      raise TypeError(f"cache must be a KVCache, got {type(cache).__name__}")
    if q.requires_grad and torch.is_grad_enabled():
      raise NotImplementedError("attention over the cache has no backward pass; call it under torch.no_grad()")
    if forward_ad._current_level >= 0 and forward_ad.unpack_dual(q).tangent is not None:
      raise NotImplementedError("attention over the cache has no forward-mode derivative")
    if q.ndim == 3:
      out = self(q[None], cache, page_table, lengths, counts=counts, parents=parents, save_residuals=save_residuals)
      return (out[0][0], (out[1][0][0],)) if save_residuals else out[0]
    # What a call is made of besides its pointers, checked and filled in once per class of calls.
    key = (q.shape, q.stride(), q.dtype, q.device, cache.k.shape, cache.k.dtype, cache.k.device, page_table.shape,
           page_table.stride(), page_table.dtype, page_table.device, lengths.shape, lengths.stride(), lengths.dtype, lengths.device,
           None if counts is None else _signature(counts), None if parents is None else _signature(parents))
    known = self._calls.get(key)
    if known is None:
      as_given = (q, page_table, lengths, counts, parents)
      p, *arguments = self._params(*as_given, cache)
      if any(x is not y for x, y in zip(as_given, arguments)):  # copies that the kernels can read
        q, page_table, lengths, counts, parents = arguments
        return self(q, cache, page_table, lengths, counts=counts, parents=parents, save_residuals=save_residuals)
      # The workspace of a call is made like this tensor of one byte, spread over its size.
      with torch.cuda.device(q.device):
        nbytes = int(_ffi.load().splash_cached_workspace_bytes(ctypes.byref(p)))
      spread = torch.empty(1, dtype=torch.uint8, device=q.device).expand(max(nbytes, 16))
      known = _remember(self._calls, key, (bytes(p), nbytes, spread))
    template, nbytes, spread = known
    if q.data_ptr() % 16:
      q = q.clone()
    device = q.device
    out = torch.empty_like(q)
    lse = torch.empty(q.shape[:3], dtype=torch.float32, device=device) if save_residuals else None
    p = _ffi.SplashCachedParams.from_buffer_copy(template)
    if p.batch and p.n:
      _poll_status(device)
      p.q, p.k_cache, p.v_cache, p.out = q.data_ptr(), cache.k.data_ptr(), cache.v.data_ptr(), out.data_ptr()
      if p.quantized:
        p.k_exponent, p.v_exponent = cache.k_exponent.data_ptr(), cache.v_exponent.data_ptr()
      p.page_table, p.lengths = page_table.data_ptr(), lengths.data_ptr()
      if counts is not None:
        p.counts = counts.data_ptr()
      if parents is not None:
        p.parents = parents.data_ptr()
      if lse is not None:
        p.lse_out = lse.data_ptr()
      mode = os.environ.get("SPLASH_CHECK_STATUS", "async")
      p.status = _status_word(device).data_ptr()
      p.status_host = _status_host(device) if mode != "0" else None
      workspace = torch.empty_like(spread, memory_format=torch.contiguous_format)
      rc = _launch(device, _ffi.load().splash_cached_fwd, ctypes.byref(p), workspace.data_ptr(), nbytes)
      if rc:
        _ffi.check(rc, "attention over the cache")
      if mode == "1":
        check_device_status(device)
    return (out, (lse,)) if save_residuals else out

  def _params(self, q, page_table, lengths, counts, parents, cache):
    """The parameter block of a call of this class without its pointers, and the arguments as the kernels read them."""
    if not q.is_cuda:
      raise RuntimeError("attention over the cache runs only on a CUDA (sm_100a) device; there is no CPU path.")
    if q.ndim != 4:
      raise ValueError(f"q must be [(batch,) heads, n, head_dim], got {tuple(q.shape)}")
    batch, heads, n, head_dim = q.shape
    device = q.device
    if cache.k.device != device:
      raise ValueError(f"q is on {device}, the cache is on {cache.k.device}")
    num_pages, kv_heads, page_size, cache_dim = cache.k.shape
    if q.dtype not in _TORCH_DTYPES:
      raise NotImplementedError(f"Only bf16/f16 are supported, got {q.dtype}")
    if cache.k.dtype != q.dtype and not cache.quantized:
      raise ValueError(f"q is {q.dtype}, the cache holds {cache.k.dtype}")
    if head_dim != cache_dim:
      raise ValueError(f"q has head_dim {head_dim}, the cache has {cache_dim}")
    if heads == 0 or heads % kv_heads:
      raise ValueError(f"{heads} heads are not a multiple of the cache's {kv_heads}")
    page_table = _index_tensor(page_table, "page_table", device, (batch, None))
    lengths = _index_tensor(lengths, "lengths", device, (batch,))
    p = _ffi.SplashCachedParams()
    if counts is not None:
      counts = _index_tensor(counts, "counts", device, (batch,))
    if parents is not None:
      if n > MAX_TREE:
        raise NotImplementedError(f"a tree has at most {MAX_TREE} nodes, got {n}")
      each = parents.ndim == 2
      parents = _index_tensor(parents, "parents", device, (batch, n) if each else (n,))
      p.parents = 1  # (any address: the library sizes a call by whether there is one)
      p.parents_stride = parents.stride(0) if each else 0
    p.table_stride, p.table_width = page_table.stride(0), page_table.shape[1]
    p.batch, p.heads, p.kv_heads, p.n, p.head_dim = batch, heads, kv_heads, n, head_dim
    p.num_pages, p.page_size, p.dtype, p.quantized = num_pages, page_size, _TORCH_DTYPES[q.dtype], cache.quantized
    p.window_left = -1 if self.window_left is None else self.window_left
    p.num_sinks, p.mask_value = self.num_sinks, self.mask_value
    p.soft_cap = self.attn_logits_soft_cap or 0.0
    return p, q.contiguous(), page_table, lengths, counts, parents


def make_splash_cached(*, window_left: int | None = None, num_sinks: int = 0, attn_logits_soft_cap: float | None = None,
                       mask_value: float = DEFAULT_MASK_VALUE) -> CachedAttentionKernel:
  """Attention over a `KVCache`.

  window_left: a token sees the `window_left` positions in front of its own, and its own (None: all); as
    `LocalMask(shape, (window_left, 0))`.
  num_sinks: positions below this stay visible behind the window.
  attn_logits_soft_cap: logits -> cap * tanh(logits / cap).
  mask_value: the logsumexp of rows that see no key.
  """
  if window_left is not None and window_left < 0:
    raise ValueError(f"window_left must not be negative, got {window_left}")
  if num_sinks < 0:
    raise ValueError(f"num_sinks must not be negative, got {num_sinks}")
  if attn_logits_soft_cap is not None and not (attn_logits_soft_cap > 0 and math.isfinite(attn_logits_soft_cap)):
    raise ValueError(f"attn_logits_soft_cap must be positive, got {attn_logits_soft_cap}")
  clip = (1 << 31) - 1
  return CachedAttentionKernel(window_left=None if window_left is None else min(int(window_left), clip),
                               num_sinks=min(int(num_sinks), clip), attn_logits_soft_cap=attn_logits_soft_cap,
                               mask_value=mask_value)
