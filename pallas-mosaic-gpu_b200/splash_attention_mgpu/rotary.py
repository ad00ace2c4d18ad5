"""Rotary positions with one or several axes, applied to q and k before attention.

    rotary = make_rotary(128, q_scale=128 ** -0.5)                    # one axis
    q, k = rotary(q, k, positions)                                    # positions: [S] or [B, S]
    rotary = make_rotary(128, (16, 24, 24), q_scale=128 ** -0.5)      # time, height, width
    q, k = rotary(q, k, positions)                                    # positions: [3, S] or [B, 3, S]

The attention kernels expect a pre-scaled q; `q_scale` is that factor, applied before the one rounding of the result.
q and k may be views (a fused projection's output, transposed): only the last dimension has to be contiguous.  The
results are contiguous [(B,) heads, S, head_dim], as the kernels want them.  Differentiable in q and k, backward and forward.

No counterpart in the reference, whose callers rotate with JAX operations.
"""

from __future__ import annotations

import ctypes
import functools
import math
from typing import Sequence

import numpy as np
import torch
import torch.autograd.forward_ad as forward_ad

from . import _ffi
from .splash_attention import _TORCH_DTYPES, _launch


def _batched_strides(x, batched):
  return tuple(x.stride()[:3]) if batched else (0, *x.stride()[:2])


def _in_place(x):
  """Whether the kernel can read x where it lies: rows contiguous, their starts 8-byte aligned (the base apart)."""
  return x.stride(-1) == 1 and not any(s % 4 for s in x.stride()[:-1])


@functools.lru_cache(maxsize=16)
def _pi(bits: int) -> int:
  """Pi in units of 2^-bits, within 2 of them: Machin's formula, pi = 16 atan(1/5) - 4 atan(1/239)."""
  def atan_of_inverse(n):
    power = (1 << (bits + 16)) // n
    total, k = 0, 1
    while power:
      total += power // k if k % 4 == 1 else -(power // k)
      power //= n * n
      k += 2
    return total

  return (16 * atan_of_inverse(5) - 4 * atan_of_inverse(239)) >> 16


def _turns(f: float) -> int:
  """f / 2 pi modulo one turn in units of 2^-64, to nearest (in whole numbers: a double has 53 bits)."""
  n, d = f.as_integer_ratio()
  bits = 128 + max(0, 64 + n.bit_length() - d.bit_length())
  den = d * _pi(bits)
  return ((n << (64 + bits)) + den) // (2 * den) % (1 << 64)


class RotaryEmbedding:
  """Rotation plan: which axis each pair of a row turns with, and how fast.  Made by `make_rotary`."""

  def __init__(self, head_dim: int, axes: Sequence[int], inv_freq: Sequence[float], *, pairing: str, q_scale: float):
    self.head_dim = int(head_dim)
    self.axes = tuple(int(a) for a in axes)
    self.inv_freq = tuple(float(f) for f in inv_freq)
    self.pairing = pairing
    self.q_scale = float(q_scale)
    self.num_axes = max(self.axes) + 1
    # The kernel's product of these with a position wraps where turns do.
    self._turns = np.array([_turns(f) for f in self.inv_freq], np.uint64).view(np.int64)
    self._device_tables: dict = {}
    self._calls: dict = {}

  def __repr__(self):
    return (f"RotaryEmbedding(head_dim={self.head_dim}, pairs={len(self.axes)}, axes={self.num_axes},"
            f" pairing={self.pairing!r}, q_scale={self.q_scale})")

  def _tables(self, device):
    key = (device.type, device.index)
    if key not in self._device_tables:
      self._device_tables[key] = (torch.from_numpy(self._turns).to(device),
                                  torch.tensor(self.axes, dtype=torch.int32, device=device))
    return self._device_tables[key]

  def __getstate__(self):
    # (a copy makes tables of its own, on whatever devices it is called)
    return {**self.__dict__, "_device_tables": {}, "_calls": {}}

  # -- call --------------------------------------------------------------------
  def __call__(self, q, k, positions):
    """Rotated q (times q_scale) and k; `k` may be None, then the rotated q alone."""
    for x in (q, positions) if k is None else (q, k, positions):
      if not isinstance(x, torch.Tensor):
        raise TypeError("q, k and positions must be torch tensors")
    out = self._rotate(q, k, positions, inverse=False)
    return out[0] if k is None else out

  def _rotate(self, q, k, positions, *, inverse):
    if (torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad))) or forward_ad._current_level >= 0:
      return _RotaryFn.apply(q, k, positions, self, inverse)
    return self._run(q, k, positions, inverse=inverse)

  def _params(self, q, k, positions, inverse):
    """The parameter block of a call with these shapes and strides, without its pointers."""
    if not q.is_cuda:
      raise RuntimeError("rotary positions run only on a CUDA (sm_100a) device; there is no CPU path.")
    if q.ndim not in (3, 4):
      raise ValueError(f"q must be [(batch,) heads, len, head_dim], got {tuple(q.shape)}")
    if q.dtype not in _TORCH_DTYPES:
      raise NotImplementedError(f"Only bf16/f16 are supported, got {q.dtype}")
    batched = q.ndim == 4
    batch, length = (q.shape[0] if batched else 1), q.shape[-2]
    if q.shape[-1] != self.head_dim:
      raise ValueError(f"q has head_dim {q.shape[-1]}, the rotation was made for {self.head_dim}")
    if q.shape[-3] == 0:
      raise ValueError("q has no heads")
    if k is not None:
      if k.dtype != q.dtype or k.device != q.device:
        raise ValueError(f"q and k differ: {q.dtype} on {q.device}, {k.dtype} on {k.device}")
      if k.ndim != q.ndim or k.shape[-1] != q.shape[-1] or k.shape[-2] != length or (batched and k.shape[0] != batch):
        raise ValueError(f"Incompatible k {tuple(k.shape)} for q {tuple(q.shape)}")
      if k.shape[-3] == 0:
        raise ValueError("k has no heads")
    if positions.device != q.device:
      raise ValueError(f"positions are on {positions.device}, q is on {q.device}")
    if positions.dtype not in (torch.int32, torch.int64):
      raise ValueError(f"positions must be int32 or int64, got {positions.dtype}")
    tail = (length,) if self.num_axes == 1 else (self.num_axes, length)
    if tuple(positions.shape) not in (tail, (batch, *tail)):
      raise ValueError(f"positions must be {list(tail)} or {[batch, *tail]}, got {list(positions.shape)}")
    p = _ffi.SplashRotaryParams()
    p.q_stride = _batched_strides(q, batched)
    if k is not None:
      p.k_stride = _batched_strides(k, batched)
      p.k_heads = k.shape[-3]
    steps = positions.stride()
    per_batch = steps[0] if positions.ndim > len(tail) else 0
    p.pos_stride = (per_batch, 0 if self.num_axes == 1 else steps[-2], steps[-1])
    p.batch, p.q_heads, p.len, p.head_dim = batch, q.shape[-3], length, self.head_dim
    p.pairs, p.dtype = len(self.axes), _TORCH_DTYPES[q.dtype]
    p.adjacent, p.inverse, p.pos_is_64 = self.pairing == "adjacent", inverse, positions.dtype == torch.int64
    p.q_scale = self.q_scale
    return p

  def _run(self, q, k, positions, *, inverse):
    # What a call is made of besides its pointers, checked and filled in once per class of calls.
    key = (q.shape, q.stride(), q.dtype, q.device, positions.shape, positions.stride(), positions.dtype, positions.device,
           inverse, None if k is None else (k.shape, k.stride(), k.dtype, k.device))
    known = self._calls.get(key)
    if known is None:
      if len(self._calls) >= 256:
        self._calls.clear()
      known = self._calls[key] = (bytes(self._params(q, k, positions, inverse)), _in_place(q), k is None or _in_place(k))
    template, q_in_place, k_in_place = known
    if not q_in_place or q.data_ptr() % 8:
      return self._run(q.clone(memory_format=torch.contiguous_format), k, positions, inverse=inverse)
    if k is not None and (not k_in_place or k.data_ptr() % 8):
      return self._run(q, k.clone(memory_format=torch.contiguous_format), positions, inverse=inverse)
    p = _ffi.SplashRotaryParams.from_buffer_copy(template)
    q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
    p.q, p.q_out, p.positions = q.data_ptr(), q_out.data_ptr(), positions.data_ptr()
    turns, axis = self._tables(q.device)
    p.turns, p.axis = turns.data_ptr(), axis.data_ptr()
    k_out = None
    if k is not None:
      k_out = torch.empty_like(k, memory_format=torch.contiguous_format)
      p.k, p.k_out = k.data_ptr(), k_out.data_ptr()
    if p.batch and p.len:
      rc = _launch(q.device, _ffi.load().splash_rotary, ctypes.byref(p))
      if rc:
        _ffi.check(rc, "rotary positions")
    return q_out, k_out


class _RotaryFn(torch.autograd.Function):
  """Linear: the derivative along a direction is the rotation of that, the gradient the rotation back.  The positions are all that
  is kept."""

  @staticmethod
  def forward(q, k, positions, plan, inverse):
    return plan._run(q, k, positions, inverse=inverse)

  @staticmethod
  def setup_context(ctx, inputs, output):
    _, _, positions, ctx.plan, ctx.inverse = inputs
    ctx.save_for_backward(positions)
    ctx.save_for_forward(positions)
    ctx.set_materialize_grads(True)

  @staticmethod
  def backward(ctx, dq, dk):
    (positions,) = ctx.saved_tensors
    dq, dk = ctx.plan._rotate(dq, dk, positions, inverse=not ctx.inverse)
    return dq, dk, None, None, None

  @staticmethod
  def jvp(ctx, dq, dk, *_):
    (positions,) = ctx.saved_tensors
    return ctx.plan._rotate(dq, dk, positions, inverse=ctx.inverse)


def make_rotary(head_dim: int, sections: Sequence[int] | None = None, *, base: float = 10000.0,
                inv_freq: Sequence[float] | None = None, interleaved: bool = False, pairing: str = "half",
                q_scale: float = 1.0) -> RotaryEmbedding:
  """A rotation plan.

  sections: how many pairs turn with each axis, the pairs in order; None: all head_dim / 2 with one axis.  Fewer pairs
    than head_dim / 2 leave the last numbers of a row as they are (times q_scale).
  interleaved: the axes take the pairs in turn, as long as each has pairs left, instead of one after the other.
  inv_freq: radians per position of every pair; None: base ** (-i / pairs) for pair i.
  pairing: "half", numbers i and i + pairs of a row are a pair; "adjacent", numbers 2i and 2i + 1.
  q_scale: factor on q (the attention kernels apply none).
  """
  if sections is None:
    sections = (head_dim // 2,)
  sections = tuple(int(n) for n in sections)
  pairs = sum(sections)
  if not sections or min(sections) <= 0:
    raise ValueError(f"sections must be positive, got {sections}")
  if head_dim % 4 or pairs % 4 or 2 * pairs > head_dim:
    raise NotImplementedError(f"head_dim ({head_dim}) and the number of pairs ({pairs}) must be multiples of 4, with at most"
                              " head_dim / 2 pairs")
  if pairing not in ("half", "adjacent"):
    raise ValueError(f'pairing must be "half" or "adjacent", got {pairing!r}')
  if not math.isfinite(q_scale):
    raise ValueError(f"q_scale must be finite, got {q_scale}")
  if interleaved:
    left, axes = list(sections), []
    while len(axes) < pairs:
      for a, n in enumerate(left):
        if n:
          axes.append(a)
          left[a] -= 1
  else:
    axes = [a for a, n in enumerate(sections) for _ in range(n)]
  if inv_freq is None:
    inv_freq = [float(base) ** (-i / pairs) for i in range(pairs)]
  inv_freq = [float(f) for f in inv_freq]
  if len(inv_freq) != pairs or not all(math.isfinite(f) for f in inv_freq):
    raise ValueError(f"inv_freq must hold {pairs} finite numbers, got {len(inv_freq)}")
  return RotaryEmbedding(head_dim, axes, inv_freq, pairing=pairing, q_scale=q_scale)
