"""The status word and attention over the cache: one report for one failure, and no word made inside a graph.

As in test_gpu_status.py no kernel is made to time out: the word is set from the host."""

import os
import subprocess
import sys
import textwrap
import time

import pytest
import torch

import splash_attention_mgpu as sa
from splash_attention_mgpu import _ffi
from splash_attention_mgpu import splash_attention as api

from conftest import ROOT

DEV = "cuda:0"


def _serving():
  g = torch.Generator(device=DEV).manual_seed(0)
  cache = sa.make_kv_cache(8, 1, 128, page_size=64, device=DEV)
  table = torch.arange(8, dtype=torch.int32, device=DEV)[None]
  zero = torch.zeros(1, dtype=torch.int32, device=DEV)
  k, v = (torch.randn(1, 1, 300, 128, generator=g, device=DEV).to(torch.bfloat16) for _ in range(2))
  cache.write(k, v, table, zero)
  q = (torch.randn(1, 4, 1, 128, generator=g, device=DEV) / 11).to(torch.bfloat16)
  return q, cache, table, zero + 300


@pytest.mark.gpu
def test_gpu_calls_still_queued_do_not_report_again(monkeypatch):
  monkeypatch.delenv("SPLASH_CHECK_STATUS", raising=False)
  q, cache, table, lens = _serving()
  attend = sa.make_splash_cached()
  good = attend(q, cache, table, lens)
  sa.check_device_status()
  api._status_word(torch.device(DEV)).copy_(torch.tensor([1, 9, 3, 5], dtype=torch.int32))
  torch.cuda.synchronize()
  torch.cuda._sleep(200_000_000)  # some 0.1 s each
  attend(q, cache, table, lens)
  torch.cuda._sleep(400_000_000)
  attend(q, cache, table, lens)   # finds the word set after the first one's report
  mirror, until = api._status_mirrors["cuda", 0], time.monotonic() + 20
  while mirror.code.value == 0 and time.monotonic() < until:
    time.sleep(0.001)
  with pytest.raises(_ffi.SplashLibraryError, match="wait site 9, block 3, step 5"):
    attend(q, cache, table, lens)
  torch.cuda.synchronize()
  again = attend(q, cache, table, lens)
  torch.cuda.synchronize()
  sa.check_device_status()
  assert torch.equal(again, good)


@pytest.mark.gpu
def test_gpu_first_call_of_a_process_in_a_capture():
  code = """
    import torch
    import test_gpu_status_of_cached as t
    import splash_attention_mgpu as sa
    from splash_attention_mgpu import splash_attention as api
    q, cache, table, lens = t._serving()
    words, mirrors = dict(api._status_words), dict(api._status_mirrors)
    assert words and mirrors  # there before the capture
    attend, graph = sa.make_splash_cached(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
      captured = attend(q, cache, table, lens)
    assert words == api._status_words
    eager = attend(q, cache, table, lens)  # before the graph has ever run
    sa.check_device_status()
    graph.replay()
    torch.cuda.synchronize()
    assert eager.any() and torch.equal(eager, captured)
    print("fine")
  """
  path = f"import sys; sys.path[:0] = [{ROOT + '/tests'!r}, {ROOT + '/pallas-mosaic-gpu_b200'!r}, {ROOT!r}]\n"
  done = subprocess.run([sys.executable, "-c", path + textwrap.dedent(code)], capture_output=True, text=True, timeout=300,
                        env={**os.environ, "SPLASH_CHECK_STATUS": "async"})
  assert done.returncode == 0 and "fine" in done.stdout, done.stderr[-2000:]


def test_no_word_is_made_in_a_capture(monkeypatch):
  monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
  monkeypatch.setattr(api, "_status_words", {})
  with pytest.raises(RuntimeError, match="capture"):
    api._status_word(torch.device("cpu"))
  assert not api._status_words
