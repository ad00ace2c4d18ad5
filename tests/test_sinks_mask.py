"""Sliding windows with sinks on the host: element semantics, schedules, the kernels' arithmetic on them."""

import numpy as np
import pytest

import splash_attention_mgpu as sa
from oracle import dense_attention as oracle
from oracle import schedule_emulator
from splash_attention_mgpu import mask_info as mask_info_lib

from common import inputs
from test_mask_info import _rebuild


def _dense(shape, left, right, offset, sinks):
  q, k = np.arange(shape[0])[:, None] + offset, np.arange(shape[1])[None, :]
  ahead = np.ones(shape, bool) if right is None else k <= q + right
  behind = np.ones(shape, bool) if left is None else (k >= q - left) | (k < sinks)
  return ahead & behind


CASES = [((512, 512), 100, 0, 0, 4), ((512, 512), 64, 0, 0, 1), ((512, 512), 128, 20, 0, 130), ((512, 512), 0, 0, 0, 512),
         ((256, 768), 200, 0, 512, 128), ((256, 768), 10, 0, -100, 7), ((512, 512), None, 0, 0, 4), ((512, 512), 50, None, 0, 300)]


@pytest.mark.parametrize("shape,left,right,offset,sinks", CASES)
@pytest.mark.parametrize("blocks", [(128, 64), (128, 128), (256, 128)])
def test_schedules_rebuild_the_mask(shape, left, right, offset, sinks, blocks):
  mask = sa.LocalMask(shape, (left, right), offset, num_sinks=sinks)
  dense = _dense(shape, left, right, offset, sinks)
  np.testing.assert_array_equal(np.asarray(mask[:, :]), dense)
  info = mask_info_lib.process_mask(mask, blocks)
  mask_info_lib.validate_schedule(info)
  np.testing.assert_array_equal(_rebuild(info, dense), dense)
  np.testing.assert_array_equal(_rebuild(info, dense, transposed=True), dense)
  assert info.partial_mask_blocks is None
  np.testing.assert_array_equal(info.mask_descriptors[:, 3], [min(sinks, shape[1])])
  # No block is visited that holds nothing visible.
  tiles = dense.reshape(shape[0] // blocks[0], blocks[0], shape[1] // blocks[1], blocks[1]).any(axis=(1, 3))
  np.testing.assert_array_equal(info.num_steps[0], tiles.sum(axis=1))


def test_emulated_schedule_matches_the_dense_form():
  s = 512
  mask = sa.LocalMask((s, s), (70, 0), 0, num_sinks=9)
  q, k, v = (x[0] for x in inputs(1, 2, 1, s, 64, 64, __import__("torch").float32, False, seed=1, scale=0.125))
  ref, ref_lse = oracle.attention_forward(np.asarray(mask[:, :])[None], q, k, v)
  out, lse = schedule_emulator.emulate_forward(mask_info_lib.process_mask(mask, (128, 64)), q, k, v,
                                             mask_value=sa.DEFAULT_MASK_VALUE)
  np.testing.assert_allclose(out, ref, atol=2e-2, rtol=2e-2)
  np.testing.assert_allclose(lse, ref_lse, atol=1e-3, rtol=1e-3)


def test_masks_with_other_sinks_differ():
  a, b = (sa.LocalMask((256, 256), (64, 0), 0, num_sinks=n) for n in (0, 4))
  assert a != b and a == sa.LocalMask((256, 256), (64, 0), 0) and hash(b) == hash(sa.LocalMask((256, 256), (64, 0), num_sinks=4))
  info = mask_info_lib.process_mask(sa.MultiHeadMask([a, b]), (128, 128))
  assert info.num_steps.shape[0] == 2
  np.testing.assert_array_equal(info.mask_descriptors[:, 3], [0, 4])
  with pytest.raises(ValueError, match="num_sinks"):
    sa.LocalMask((256, 256), (64, 0), num_sinks=-1)


def test_formula_of_the_gradients_against_differences():
  """The formula that the kernels' gradients are held against, windows and sinks included, shared heads too."""
  import torch
  from oracle import dense_attention
  h, kvh, s, d = 4, 2, 12, 8
  mask = np.asarray(sa.LocalMask((s, s), (3, 0), 0, num_sinks=2)[:, :])[None]
  g = torch.Generator().manual_seed(0)
  q, k, v, do = (torch.randn(1, x, s, d, generator=g, dtype=torch.float64) for x in (h, kvh, kvh, h))
  grads = dense_attention.attention_backward(mask, q, k, v, do, None)
  loss = lambda *x: float((dense_attention.attention_forward(mask, *x, None)[0] * do.numpy()).sum())
  for i, grad in enumerate(grads):
    u = torch.randn((q, k, v)[i].shape, generator=g, dtype=torch.float64)
    step = 2.0 ** -6
    at = lambda t: loss(*(x + t * u if j == i else x for j, x in enumerate((q, k, v))))
    slope = (8 * (at(step) - at(-step)) - (at(2 * step) - at(-2 * step))) / (12 * step)
    # 32-bit sums: 2^-24 of about 400 terms of size 1, over the step; the difference itself is off by step^4 f^(5) / 30.
    assert abs(slope - float((torch.as_tensor(grad) * u).sum())) < 400 * 2.0 ** -24 * 12 / step + step ** 4 * 400
