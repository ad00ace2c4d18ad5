"""Runs, trees, windows and short sequences over 8-bit caches in every form (head dim, type), by a bar that does not grow with the
context: test_gpu_cached_attention.py's, but the term for probabilities below the range of P's terms is 2^-29 of the row's largest
2^ev p times the codes of the values (half of e5m2's lowest step, 2^-17, where that largest is scaled to 2^12 or more) in place of
2^-15 of it, which is the whole result at 32768 keys; and f16's P, rounded once to 11 bits (2^-11), has 2^-12 more."""

import pytest
import torch

import test_gpu_cached_attention as base

FORMS = [(d, dtype) for d in (64, 128) for dtype in (torch.bfloat16, torch.float16)]


@pytest.fixture(autouse=True)
def bar(monkeypatch):
  plain = base._want

  def want(*args):
    (out, a, low), *rest = plain(*args)
    return ((out, a, low * 2.0 ** -14 + 2.0 ** -12 * a), *rest)

  monkeypatch.setattr(base, "_want", want)


@pytest.mark.gpu
@pytest.mark.parametrize("d,dtype", FORMS, ids=str)
@pytest.mark.parametrize("case", [
    dict(b=3, h=4, kvh=2, n=5, page=16, lengths=[5, 300, 140], counts=[0, 3, 5]),
    dict(b=2, h=8, kvh=1, n=4, page=64, lengths=[2, 1000], counts=[4, 4]),
    dict(b=1, h=2, kvh=1, n=200, page=32, lengths=[200]),
    dict(b=2, h=2, kvh=2, n=60, page=64, lengths=[700, 60], counts=[60, 33]),
    dict(b=1, h=5, kvh=1, n=77, page=16, lengths=[1500]),
    dict(b=2, h=1, kvh=1, n=1, page=16, lengths=[20000, 77]),
    dict(b=1, h=2, kvh=1, n=7, page=16, lengths=[100], parents=[-1, 0, 0, 1, 1, 2, -1]),
    dict(b=3, h=8, kvh=2, n=48, page=64, lengths=[48, 500, 1000], parents=[base._tree(48, i) for i in range(3)]),
    dict(b=2, h=2, kvh=1, n=128, page=16, lengths=[128, 777], parents=[base._tree(128, 3), list(range(-1, 127))]),
    dict(b=2, h=4, kvh=1, n=20, page=16, lengths=[23, 400], parents=base._tree(20, 7, wide=2), window=3, sinks=5),
    dict(b=3, h=4, kvh=2, n=1, page=128, lengths=[1, 103, 5000], window=100, sinks=4),
    dict(b=3, h=4, kvh=2, n=8, page=16, lengths=[1200, 4097, 8], window=1000),
    dict(b=3, h=4, kvh=2, n=40, page=128, lengths=[40, 333, 2049], window=30, sinks=2),
    dict(b=2, h=8, kvh=2, n=2, page=64, lengths=[300, 1000], cap=5.0, spread=4.0),
    dict(b=2, h=24, kvh=2, n=2, page=64, lengths=[300, 1000], cap=5.0, spread=4.0),
    dict(b=2, h=8, kvh=2, n=2, page=64, lengths=[300, 2000], spread=12.0, seed=3),
    dict(b=2, h=40, kvh=2, n=2, page=64, lengths=[300, 2000], spread=12.0, seed=3),
    dict(b=300, h=16, kvh=1, n=1, page=64, lengths=[(i * 53) % 200 for i in range(300)], fade=11),
    dict(b=300, h=6, kvh=1, n=9, page=64, lengths=[(i * 53) % 200 for i in range(300)], fade=11),
], ids=lambda c: f"b{c['b']}h{c['h']}n{c['n']}len{max(c['lengths'])}" + ("tree" if "parents" in c else ""))
def test_gpu_every_8_bit_form(d, dtype, case):
  base._check(d=d, dtype=dtype, quantized=True, **case)
