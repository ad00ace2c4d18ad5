"""Rotary positions against the formula in 64 bits.

Bar of a result y = scale (a cos - b sin): half a rounding step of the 16-bit type, and 2^-20 (|a| + |b|) scale for what
comes before it in 32 bits (sine and cosine within 2^-22, two products, a sum, the scale: each within 2^-24)."""

import math

import pytest
import torch

import splash_attention_mgpu as sa

DEV = "cuda:0"


def _formula(plan, x, positions, scale, inverse=False):
  """([B, H, S, D] in 64 bits, the bar's |a| + |b| term)."""
  x = x.detach().double()
  pairs, dev = len(plan.axes), x.device
  if x.ndim == 3:
    x = x[None]
  p = positions.to(torch.int64)
  p = p.reshape((1 if p.ndim == (1 if plan.num_axes == 1 else 2) else p.shape[0], plan.num_axes, -1))
  freq = torch.tensor(plan.inv_freq, dtype=torch.float64, device=dev)
  angle = (p[:, list(plan.axes)].double() * freq[:, None]).transpose(1, 2)[:, None]  # [B or 1, 1, S, pairs]
  cos, sin = torch.cos(angle), torch.sin(angle) * (-1 if inverse else 1)
  rot = x[..., :2 * pairs]
  a, b = (rot[..., 0::2], rot[..., 1::2]) if plan.pairing == "adjacent" else rot.chunk(2, -1)
  y, size = x.clone(), x.abs()
  parts = (a * cos - b * sin, b * cos + a * sin)
  both = a.abs() + b.abs()
  if plan.pairing == "adjacent":
    y[..., 0:2 * pairs:2], y[..., 1:2 * pairs:2] = parts
    size[..., 0:2 * pairs:2], size[..., 1:2 * pairs:2] = both, both
  else:
    y[..., :pairs], y[..., pairs:2 * pairs] = parts
    size[..., :pairs], size[..., pairs:2 * pairs] = both, both
  return y * scale, size * abs(scale)


def _close(got, want, size):
  got = got.detach()
  half = torch.finfo(got.dtype).eps / 2
  tiny = torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps  # a step among the subnormals
  bar = half * want.abs() + 2.0 ** -20 * size + tiny
  off = (got.double() - want.reshape(got.shape)).abs()
  assert (off <= bar.reshape(got.shape)).all(), float((off / bar.reshape(got.shape)).max())


def _views(b, h, kvh, s, d, dtype, layout, seed=0):
  g = torch.Generator(device=DEV).manual_seed(seed)
  if layout == "fused":
    qkv = torch.randn(b, s, h + 2 * kvh, d, generator=g, device=DEV).to(dtype)
    return qkv[:, :, :h].transpose(1, 2), qkv[:, :, h:h + kvh].transpose(1, 2)
  make = lambda n: torch.randn(b, n, s, d, generator=g, device=DEV).to(dtype)
  return make(h), make(kvh)


PLANS = {
    "one": dict(),
    "three": dict(sections=(16, 24, 24)),
    "turns": dict(sections=(16, 24, 24), interleaved=True),
    "part": dict(sections=(16, 4), pairing="adjacent"),
    "adjacent": dict(sections=(32, 32), pairing="adjacent", base=500000.0),
    "scaled": dict(inv_freq=[3.0 * 0.9 ** i for i in range(64)]),
}


@pytest.mark.gpu
@pytest.mark.parametrize("name", PLANS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("b,h,kvh,s,layout", [(1, 1, 1, 1, "plain"), (3, 5, 1, 7, "fused"), (2, 12, 4, 130, "plain"), (2, 32, 8, 333, "fused")])
def test_gpu_rotary_and_its_gradient(name, dtype, b, h, kvh, s, layout):
  plan = sa.make_rotary(128, q_scale=128 ** -0.5, **PLANS[name])
  q, k = _views(b, h, kvh, s, 128, dtype, layout)
  shape = (b, s) if plan.num_axes == 1 else (b, plan.num_axes, s)
  positions = torch.randint(-5, 1 << 20, shape, device=DEV, dtype=torch.int32)
  q2, k2 = plan(q, k, positions)
  assert q2.is_contiguous() and k2.is_contiguous()
  _close(q2, *_formula(plan, q, positions, 128 ** -0.5))
  _close(k2, *_formula(plan, k, positions, 1.0))
  leaves = [x.detach().clone().requires_grad_(True) for x in (q, k)]
  out = plan(*leaves, positions)
  assert torch.equal(out[0], q2) and torch.equal(out[1], k2)
  d_out = [torch.randn(x.shape, device=DEV).to(dtype) for x in out]
  grads = torch.autograd.grad(out, leaves, d_out)
  _close(grads[0], *_formula(plan, d_out[0], positions, 128 ** -0.5, inverse=True))
  _close(grads[1], *_formula(plan, d_out[1], positions, 1.0, inverse=True))


@pytest.mark.gpu
def test_gpu_rotary_far_positions_types_of_positions_and_shapes():
  plan = sa.make_rotary(64)
  q, k = _views(1, 2, 1, 9, 64, torch.float16, "plain")
  far = torch.tensor([0, 1, -1, 2 ** 24 + 1, 2 ** 31 - 1, -2 ** 31, 10 ** 9 + 7, 65537, 3], device=DEV)
  for positions in (far.to(torch.int32), far, far[None].to(torch.int32)):
    got, _ = plan(q, k, positions)
    # In 64 bits the formula's own angle is off by 2^31 * 2^-53 here: below the bar.
    _close(got, *_formula(plan, q, positions, 1.0))
  assert torch.equal(plan(q[0], k[0], far)[0], plan(q, k, far)[0][0])
  assert torch.equal(plan(q, None, far), plan(q, k, far)[0])
  strided = torch.stack((far, far), -1)[..., 0]
  assert torch.equal(plan(q, k, strided)[1], plan(q, k, far)[1])
  # Rows that start off a 16-byte and off an 8-byte boundary.
  for shift in (4, 1):
    base = torch.zeros(q.numel() + 8, dtype=q.dtype, device=DEV)
    moved = base[shift:shift + q.numel()].view(q.shape)
    moved.copy_(q)
    assert torch.equal(plan(moved, k, far)[0], plan(q, k, far)[0])
  empty = plan(q[:, :, :0], k[:, :, :0], far[:0])
  assert empty[0].shape == (1, 2, 0, 64) and empty[1].shape == (1, 1, 0, 64)


@pytest.mark.gpu
def test_gpu_rotary_gradients_that_are_expanded_or_missing_and_a_captured_step():
  plan = sa.make_rotary(128, (16, 24, 24), q_scale=0.5)
  q, k = _views(2, 4, 2, 40, 128, torch.bfloat16, "plain")
  positions = torch.arange(3 * 40, device=DEV, dtype=torch.int32).view(3, 40)
  q, k = (x.requires_grad_(True) for x in (q, k))
  out = plan(q, k, positions)
  dq, = torch.autograd.grad(out[0].sum(), (q,), retain_graph=True)  # an expanded gradient, none for k
  _close(dq, *_formula(plan, torch.ones_like(q), positions, 0.5, inverse=True))
  w = torch.randn(out[0].shape, device=DEV).to(torch.bfloat16)
  want = torch.autograd.grad((out[0],), (q,), w)[0]
  leaf_q, leaf_k = (x.detach().clone().requires_grad_(True) for x in (q, k))
  side = torch.cuda.Stream()
  side.wait_stream(torch.cuda.current_stream())
  with torch.cuda.stream(side):
    torch.autograd.grad(plan(leaf_q, leaf_k, positions), (leaf_q, leaf_k), (w, torch.zeros_like(k)))
  torch.cuda.current_stream().wait_stream(side)
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    got = torch.autograd.grad(plan(leaf_q, leaf_k, positions), (leaf_q, leaf_k), (w, torch.zeros_like(k)))
  got[0].zero_()
  graph.replay()
  torch.cuda.synchronize()
  assert torch.equal(got[0], want)


def test_rotary_refusals():
  for kw, error in ((dict(sections=(65,)), NotImplementedError), (dict(sections=(3, 3)), NotImplementedError),
                    (dict(sections=(0, 64)), ValueError), (dict(pairing="other"), ValueError), (dict(inv_freq=[1.0]), ValueError),
                    (dict(q_scale=math.inf), ValueError), (dict(inv_freq=[math.nan] * 64), ValueError)):
    with pytest.raises(error):
      sa.make_rotary(128, **kw)
  plan = sa.make_rotary(128)
  x = torch.zeros(1, 2, 4, 128, dtype=torch.bfloat16)
  with pytest.raises(RuntimeError, match="CUDA"):
    plan(x, x, torch.zeros(4, dtype=torch.int32))
  with pytest.raises(TypeError):
    plan(x, x, [0, 1, 2, 3])
  assert sa.make_rotary(16, (4, 2, 2), interleaved=True).axes == (0, 1, 2, 0, 1, 2, 0, 0)


@pytest.mark.gpu
def test_gpu_rotary_refusals():
  plan = sa.make_rotary(128, (32, 32))
  q, k = _views(2, 2, 1, 4, 128, torch.bfloat16, "plain")
  p = torch.zeros(2, 4, dtype=torch.int32, device=DEV)
  plan(q, k, p)
  for bad, error in (((q.float(), k, p), NotImplementedError), ((q, k.half(), p), ValueError), ((q[..., :64], k, p), ValueError),
                     ((q, k[:, :, :3], p), ValueError), ((q, k, p[:1]), ValueError), ((q, k, p.float()), ValueError),
                     ((q, k, p.cpu()), ValueError), ((q, k[:1], p), ValueError), ((q[:, :0], k, p), ValueError)):
    with pytest.raises(error):
      plan(*bad)


@pytest.mark.gpu
@pytest.mark.parametrize("pairing", ["half", "adjacent"])
def test_gpu_rotary_gradient_is_the_transpose(pairing):
  """The rotation is linear: differences along unit vectors are its matrix, whose transpose the gradient applies.  Either is one
  product per number here, rounded once."""
  d = 64
  plan = sa.make_rotary(d, (8, 24), pairing=pairing, q_scale=0.37)
  eye = torch.eye(d, device=DEV, dtype=torch.bfloat16).view(1, 1, d, d)
  positions = torch.tensor([[17], [900]], device=DEV, dtype=torch.int32).expand(2, d)  # one place for all
  zero = torch.zeros_like(eye)
  forward = plan(eye, None, positions).double() - plan(zero, None, positions).double()
  leaf = zero.clone().requires_grad_(True)
  backward, = torch.autograd.grad(plan(leaf, None, positions), leaf, eye)
  off = (backward[0, 0].double() - forward[0, 0].T).abs()
  assert (off <= 2 * 2.0 ** -8 * forward[0, 0].T.abs() + 2.0 ** -20).all()
