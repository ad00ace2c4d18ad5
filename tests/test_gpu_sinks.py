"""Sliding windows with sinks through the kernels, forward and both backward paths, against the CPU oracle (bars of
test_gpu_forward.py and test_gpu_backward.py)."""

import numpy as np
import pytest
import torch

import splash_attention_mgpu as sa
from oracle import dense_attention as oracle

from common import assert_forward_close, inputs

DEV = "cuda:0"


def _run(mask, q_len, kv_len, h, kvh, d, dtype, *, cap=None, seg=None, blocks=None, train=True, batch=1):
  dense = np.asarray(mask[:, :, :]) if isinstance(mask, sa.MultiHeadMask) else np.asarray(mask[:, :])[None]
  kernel = sa.make_splash_mha(mask, attn_logits_soft_cap=cap, block_sizes=blocks)
  q, k, v = inputs(batch, h, kvh, max(q_len, kv_len), d, d, dtype, False, seed=5, device=DEV)
  q, k, v = (q[:, :, :q_len] * d ** -0.5).contiguous(), k[:, :, :kv_len].contiguous(), v[:, :, :kv_len].contiguous()
  out, (lse,) = kernel(q, k, v, seg, save_residuals=True)
  sa.check_device_status()
  ref, ref_lse = oracle.attention_forward(dense, q, k, v, seg, attn_logits_soft_cap=cap)
  assert_forward_close(out, lse, ref, ref_lse, dtype)
  assert_forward_close(kernel(q, k, v, seg), None, ref, None, dtype)
  if not train:
    return
  do = torch.randn(q.shape, generator=torch.Generator().manual_seed(9)).to(dtype).to(DEV)
  leaves = [x.clone().requires_grad_(True) for x in (q, k, v)]
  got = torch.autograd.grad(kernel(*leaves, seg), leaves, do)
  sa.check_device_status()
  want = oracle.attention_backward(dense, q, k, v, do, seg, attn_logits_soft_cap=cap)
  for name, a, r in zip("qkv", got, want):
    a = a.float().cpu().numpy()
    assert np.abs(a - r).max() / np.abs(r).max() < 2e-2, name
    assert np.abs(a - r).mean() / np.abs(r).mean() <= 5e-3, name


@pytest.mark.gpu
@pytest.mark.parametrize("d,dtype", [(64, torch.float16), (128, torch.bfloat16)])
@pytest.mark.parametrize("window,sinks", [(100, 1), (64, 4), (200, 130), (0, 64), (700, 16)])
@pytest.mark.parametrize("fused", ["1", "0"])
def test_gpu_window_with_sinks(monkeypatch, d, dtype, window, sinks, fused):
  monkeypatch.setenv("SPLASH_BWD_FUSED", fused)
  s = 1152
  _run(sa.LocalMask((s, s), (window, 0), 0, num_sinks=sinks), s, s, 4, 2, d, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("blocks", [dict(block_q=128, block_kv=64, num_stages=2), dict(block_q=128, block_kv=128, num_stages=2),
                                    dict(block_q=256, block_kv=128, num_stages=2)], ids=str)
def test_gpu_sinks_in_every_forward_tiling(blocks):
  s = 1024
  _run(sa.LocalMask((s, s), (150, 0), 0, num_sinks=5), s, s, 2, 1, 128, torch.bfloat16, blocks=sa.BlockSizes(**blocks), train=False)


@pytest.mark.gpu
@pytest.mark.parametrize("d", [192, 256])
def test_gpu_sinks_above_head_dim_128(d):
  s = 768
  _run(sa.LocalMask((s, s), (150, 0), 0, num_sinks=70), s, s, 2, 2, d, torch.bfloat16, train=False,
       blocks=sa.BlockSizes(block_q=128, block_kv=64, num_stages=2))


@pytest.mark.gpu
def test_gpu_sinks_in_shares_of_a_tile():
  # A chunk of queries against many keys: few tiles, each shared by several CTAs.
  _run(sa.LocalMask((128, 8192), (5000, 0), 8192 - 128, num_sinks=40), 128, 8192, 2, 1, 128, torch.bfloat16, train=False)


@pytest.mark.gpu
@pytest.mark.parametrize("fused", ["1", "0"])
def test_gpu_heads_with_other_sinks_cap_and_documents(monkeypatch, fused):
  monkeypatch.setenv("SPLASH_BWD_FUSED", fused)
  s = 1024
  heads = [sa.LocalMask((s, s), (w, 0), 0, num_sinks=n) for w, n in ((64, 4), (300, 0), (129, 140), (1000, 1))]
  ids = (torch.arange(s, dtype=torch.int32, device=DEV) // 300)
  _run(sa.MultiHeadMask(heads), s, s, 4, 4, 128, torch.bfloat16, cap=10.0)
  _run(sa.MultiHeadMask(heads), s, s, 4, 2, 64, torch.float16, seg=sa.SegmentIds(ids, ids))


@pytest.mark.gpu
def test_gpu_rows_that_see_sinks_alone_and_rows_that_see_nothing():
  # The window lies before the sequence for the first rows (offset -300: no key) and every row sees few keys.
  s = 512
  mask = sa.LocalMask((s, s), (20, 0), -300, num_sinks=3)
  dense = np.asarray(mask[:, :])
  assert not dense[:300].any() and dense[300:].any(axis=1).all()
  q, k, v = inputs(1, 2, 2, s, 128, 128, torch.bfloat16, False, seed=6, device=DEV, scale=128 ** -0.5)
  out, (lse,) = sa.make_splash_mha(mask)(q, k, v, save_residuals=True)
  sa.check_device_status()
  ref, ref_lse = oracle.attention_forward(dense[None], q, k, v)
  assert not out[:, :, :300].any() and (lse[:, :, :300] == np.float32(sa.DEFAULT_MASK_VALUE)).all()
  assert_forward_close(out[:, :, 300:], lse[:, :, 300:], ref[:, :, 300:], ref_lse[:, :, 300:], torch.bfloat16)


@pytest.mark.gpu
@pytest.mark.parametrize("d,dtype,form", [(128, torch.bfloat16, {}), (64, torch.float16, {}), (128, torch.float16, dict(cap=8.0)),
                                          (64, torch.bfloat16, dict(segs=True)), (128, torch.bfloat16, dict(segs=True))], ids=str)
def test_gpu_shared_sink_columns(d, dtype, form):
  # Two KV blocks of sinks, which all q blocks visit, beside short columns: shared by several CTAs, in any batch the same bits.
  s, batch = 2560, 2
  mask = sa.LocalMask((s, s), (150, 0), 0, num_sinks=200)
  kernel = sa.make_splash_mha(mask, attn_logits_soft_cap=form.get("cap"))
  assert kernel._shared_columns[0] == 2 and kernel._shared_columns[1] >= 4
  ids = torch.arange(s, dtype=torch.int32, device=DEV) // 900 if form.get("segs") else None
  seg = None if ids is None else sa.SegmentIds(ids, ids)
  _run(mask, s, s, 4, 2, d, dtype, cap=form.get("cap"), seg=seg, batch=batch)
  q, k, v = inputs(batch, 4, 2, s, d, d, dtype, False, seed=8, device=DEV, scale=d ** -0.5)
  do = torch.randn(q.shape, generator=torch.Generator().manual_seed(1)).to(dtype).to(DEV)

  def grads(rows):
    leaves = [x[rows].clone().requires_grad_(True) for x in (q, k, v)]
    return torch.autograd.grad(kernel(*leaves, seg), leaves, do[rows])[1:]  # (dQ is added up in any order)
  for both, alone in zip(grads(slice(0, 2)), grads(slice(1, 2))):
    assert torch.equal(both[1:], alone)


def test_columns_are_shared_by_the_mask_alone():
  shared = lambda m: sa.make_splash_mha(m)._shared_columns
  s = 4096
  assert shared(sa.LocalMask((s, s), (127, 0), 0)) == (0, 1) and shared(sa.CausalMask((s, s))) == (0, 1)
  assert shared(sa.LocalMask((s, s), (None, 0), 0, num_sinks=4)) == (0, 1)
  assert shared(sa.LocalMask((s, s), (127, 0), 0, num_sinks=4)) == (1, 16)
  assert shared(sa.LocalMask((s, s), (127, 0), 0, num_sinks=s)) == (0, 1)
  assert shared(sa.MultiHeadMask([sa.CausalMask((s, s)), sa.LocalMask((s, s), (127, 0), 0, num_sinks=129)]))[1] == 1
