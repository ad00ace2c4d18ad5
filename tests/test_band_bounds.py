"""Windows far wider than any sequence, up to the ends of 32-bit numbers and beyond, are those without a bound."""

import numpy as np
import pytest
import torch

import splash_attention_mgpu as sa
from splash_attention_mgpu import mask_info
from oracle import dense_attention as oracle

from common import inputs

DEV = "cuda:0"
INT = 2 ** 31
WINDOWS = [((INT - 1, 0), 0), ((INT - 1, INT - 1), 0), ((5, INT - 1), 3), ((2 ** 40, 2 ** 40), -7), ((INT - 1, 0), -300), ((INT - 1, 0), INT - 1)]


@pytest.mark.parametrize("window,offset", WINDOWS)
def test_schedules(window, offset):
  s = 512
  mask = sa.LocalMask((s, s), window, offset, num_sinks=2)
  at = np.arange(s, dtype=np.int64)
  diff = at[None, :] - at[:, None] - offset
  dense = ((diff >= -window[0]) | (at[None, :] < 2)) & (diff <= window[1])
  assert np.array_equal(np.asarray(mask[:, :]), dense)
  a = mask_info.process_mask(mask, (128, 64))
  assert np.array_equal(a.num_steps[0], dense.reshape(s // 128, 128, s // 64, 64).any((1, 3)).sum(-1))
  if a.mask_descriptors is not None:
    assert np.abs(a.mask_descriptors[:, :2].astype(np.int64)).max() <= 2 ** 30


class _Raw(sa.LocalMask):
  """A window whose descriptor is handed over as it is, as a caller of the C entry points may."""

  def __init__(self, shape, band):
    super().__init__(shape, (None, None))
    self.raw = band

  def band(self):
    return (*self.raw, 0)


@pytest.mark.gpu
@pytest.mark.parametrize("fused", ["1", "0"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("mask,plain", [
    (sa.LocalMask((384, 384), (INT - 1, 0)), sa.LocalMask((384, 384), (None, 0))),
    (sa.LocalMask((384, 384), (INT - 1, 40)), sa.LocalMask((384, 384), (None, 40))),
    (_Raw((384, 384), (1 - INT, 0)), sa.LocalMask((384, 384), (None, 0))),
    (_Raw((384, 384), (-INT, 40)), sa.LocalMask((384, 384), (None, 40))),
    (_Raw((384, 384), (-50, INT - 1)), sa.LocalMask((384, 384), (50, None))),
], ids=["left", "left and right", "descriptor", "lowest descriptor", "highest descriptor"])
def test_gpu_kernels(monkeypatch, fused, d, mask, plain):
  monkeypatch.setenv("SPLASH_BWD_FUSED", fused)
  q, k, v = inputs(1, 4, 2, 384, d, d, torch.bfloat16, False, seed=1, device=DEV)
  q = q * d ** -0.5
  do = torch.randn(q.shape, generator=torch.Generator().manual_seed(2)).to(q).contiguous()
  got = []
  for m in (mask, plain):
    leaves = [x.clone().requires_grad_(True) for x in (q, k, v)]
    out = sa.make_splash_mha(m)(*leaves)
    got.append((out.detach(), *torch.autograd.grad(out, leaves, do)))
  sa.check_device_status()
  dense = np.asarray(plain[:, :])[None]
  want = oracle.attention_backward(dense, q, k, v, do, None)
  for name, a, b, r in zip("qkv", got[0][1:], got[1][1:], want):
    for x in (a, b):
      x = x.float().cpu().numpy()
      assert np.abs(x - r).max() / np.abs(r).max() < 2e-2, name
      assert np.abs(x - r).mean() / np.abs(r).mean() <= 5e-3, name
  assert torch.equal(got[0][0], got[1][0])
