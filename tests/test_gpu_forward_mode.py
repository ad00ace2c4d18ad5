"""Forward-mode derivatives: a rotation gives its own, attention refuses rather than drop them."""

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import splash_attention_mgpu as sa

DEV = "cuda:0"


def _on_host(plan, q, k, positions, *, inverse):
  """A stand-in for the kernel: the rotation of pairs (i, i + pairs) by positions * f in torch operations on plain tensors."""
  angle = positions[..., None].double() * torch.tensor(plan.inv_freq, dtype=torch.float64)

  def turn(x, scale):
    if x is None:
      return None
    x.data_ptr()  # (what wraps a tensor has none)
    n = len(plan.axes)
    a, b, c, s = x[..., :n].double(), x[..., n:].double(), angle.cos(), angle.sin() * (-1 if inverse else 1)
    return (scale * torch.cat([a * c - b * s, b * c + a * s], -1)).to(x.dtype)

  return turn(q, plan.q_scale), turn(k, 1.0)


def _inputs(device):
  g = torch.Generator().manual_seed(0)
  q, k, dq, dk = (torch.randn(2, 3, 5, 64, generator=g).to(torch.bfloat16).to(device) for _ in range(4))
  return q, k, dq, dk, torch.arange(5, device=device)


def _check(q, k, dq, dk, positions):
  plan = sa.make_rotary(64, q_scale=0.125)
  want = plan(q, k, positions), plan(dq, dk, positions)
  with forward_ad.dual_level():
    duals = [forward_ad.unpack_dual(x) for x in plan(forward_ad.make_dual(q, dq), forward_ad.make_dual(k, dk), positions)]
    for i in (0, 1):
      assert torch.equal(duals[i].primal, want[0][i]) and torch.equal(duals[i].tangent, want[1][i])
    alone = forward_ad.unpack_dual(plan(forward_ad.make_dual(q, dq), None, positions))  # no k
    assert torch.equal(alone.primal, want[0][0]) and torch.equal(alone.tangent, want[1][0])
    one = forward_ad.unpack_dual(plan(forward_ad.make_dual(q, dq), k, positions)[0])  # k is a constant
    assert torch.equal(one.tangent, want[1][0])
    assert forward_ad.unpack_dual(plan(q, k, positions)[0]).tangent is None
  got, tangent = torch.func.jvp(lambda x, y: plan(x, y, positions), (q, k), (dq, dk))
  for i in (0, 1):
    assert torch.equal(got[i], want[0][i]) and torch.equal(tangent[i], want[1][i])
  # The gradient is linear in what comes in, too.
  leaf, seed = q.clone().requires_grad_(True), dq.clone().requires_grad_(True)
  (grad,) = torch.autograd.grad(plan(leaf, None, positions), leaf, seed, create_graph=True)
  (back,) = torch.autograd.grad(grad, seed, dq)
  assert torch.equal(back, want[1][0])


def test_rotation_on_the_host(monkeypatch):
  monkeypatch.setattr(sa.RotaryEmbedding, "_run", _on_host)
  _check(*_inputs("cpu"))


@pytest.mark.gpu
def test_gpu_rotation():
  _check(*_inputs(DEV))


def test_attention_over_the_cache_refuses():
  cache = sa.make_kv_cache(2, 1, 64, page_size=16, device="cpu")
  q = torch.zeros(1, 2, 1, 64, dtype=torch.bfloat16)
  table, lens = torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
  attend = sa.make_splash_cached()
  with forward_ad.dual_level():
    with pytest.raises(NotImplementedError, match="forward-mode"):
      attend(forward_ad.make_dual(q, q), cache, table, lens)
    with pytest.raises(RuntimeError, match="CUDA"):  # (no tangent: as ever)
      attend(q, cache, table, lens)
  with pytest.raises(NotImplementedError, match="forward-mode"):
    torch.func.jvp(lambda x: attend(x, cache, table, lens), (q,), (q,))
