"""Copied and reloaded caches, rotations and attention kernels work on memory of their own."""

import copy
import io

import pytest
import torch

import splash_attention_mgpu as sa
from splash_attention_mgpu import rotary as rotary_module

DEV = "cuda:0"


def _saved_and_loaded(x):
  file = io.BytesIO()
  torch.save(x, file)  # (plain pickles do not hold tensors of 8-bit floats)
  file.seek(0)
  return torch.load(file, weights_only=False)


COPIES = [copy.deepcopy, _saved_and_loaded]


def _bytes(cache):
  return [x.view(torch.uint8).clone() for x in (cache.k, cache.v, cache.k_exponent, cache.v_exponent) if x is not None]


@pytest.mark.gpu
@pytest.mark.parametrize("duplicate", COPIES, ids=["deepcopy", "saved"])
@pytest.mark.parametrize("quantized", [False, True])
def test_gpu_copied_cache(duplicate, quantized):
  g = torch.Generator(device=DEV).manual_seed(0)
  cache = sa.make_kv_cache(4, 2, 64, page_size=16, quantized=quantized, device=DEV)
  table = torch.tensor([[2, 0]], dtype=torch.int32, device=DEV)
  start, lens = torch.zeros(1, dtype=torch.int32, device=DEV), torch.full((1,), 20, dtype=torch.int32, device=DEV)
  first, second = (torch.randn(1, 2, 20, 64, generator=g, device=DEV).to(torch.bfloat16) for _ in range(2))
  cache.write(first, first, table, start)
  attend = sa.make_splash_cached()
  q = (torch.randn(1, 4, 1, 64, generator=g, device=DEV) / 8).to(torch.bfloat16)
  attend(q, cache, table, lens)
  before = _bytes(cache)
  other, other_attend = duplicate(cache), duplicate(attend)
  other.write(second, second, table, start)
  assert all(torch.equal(x, y) for x, y in zip(before, _bytes(cache)))
  fresh = sa.make_kv_cache(4, 2, 64, page_size=16, quantized=quantized, device=DEV)
  fresh.write(second, second, table, start)
  assert all(torch.equal(x, y) for x, y in zip(_bytes(fresh), _bytes(other)))
  assert all(torch.equal(x, y) for x, y in zip(other.read(table, lens, 20), fresh.read(table, lens, 20)))
  assert torch.equal(other_attend(q, other, table, lens), attend(q, fresh, table, lens))
  sa.check_device_status()


@pytest.mark.gpu
@pytest.mark.parametrize("duplicate", COPIES, ids=["deepcopy", "saved"])
def test_gpu_copied_rotation(monkeypatch, duplicate):
  used = []
  launch = rotary_module._launch

  def record(device, entry, block):
    used.append((block._obj.turns, block._obj.axis))
    return launch(device, entry, block)

  monkeypatch.setattr(rotary_module, "_launch", record)
  plan = sa.make_rotary(64, (8, 12), q_scale=0.125)
  q = torch.randn(2, 3, 5, 64, device=DEV).to(torch.bfloat16)
  positions = torch.arange(10, device=DEV).view(2, 5)
  want = plan(q, None, positions)
  other = duplicate(plan)
  got = other(q, None, positions)
  assert torch.equal(want, got)
  for p, addresses in zip((plan, other), used):
    assert addresses == tuple(x.data_ptr() for x in p._tables(q.device))
  assert used[0] != used[1]


def test_copies_keep_no_device_memory():
  plan, attend = sa.make_rotary(64), sa.make_splash_cached(window_left=5)
  plan._device_tables["cuda", 0], plan._calls[1], attend._calls[1] = 1, 1, 1
  for duplicate in COPIES:
    x = duplicate(plan)
    assert not x._device_tables and not x._calls and x.axes == plan.axes and x.inv_freq == plan.inv_freq
    assert not duplicate(attend)._calls and duplicate(attend).window_left == 5
