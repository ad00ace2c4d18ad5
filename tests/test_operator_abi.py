"""The parameter blocks of the rotary, cache and cached-attention entry points: mirrors of the header's, and what the library
refuses before any launch.  No compute calls are made here."""

import ctypes
import os
import re
import shutil
import subprocess

import pytest

from splash_attention_mgpu import _ffi

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BLOCKS = {"SplashRotaryParams": _ffi.SplashRotaryParams, "SplashCacheParams": _ffi.SplashCacheParams,
          "SplashCachedParams": _ffi.SplashCachedParams}
INVALID, UNSUPPORTED = _ffi.SPLASH_INVALID_ARGUMENT, _ffi.SPLASH_UNSUPPORTED


def test_parameter_blocks_mirror_the_header(tmp_path):
  if shutil.which("gcc") is None:
    pytest.skip("needs a C compiler")
  lines = []
  for name, block in BLOCKS.items():
    lines += [f'printf("{name} %zu\\n", sizeof({name}));']
    lines += [f'printf("{name}.{f} %zu\\n", offsetof({name}, {f}));' for f, _ in block._fields_]
  (tmp_path / "main.c").write_text('#include <stddef.h>\n#include <stdio.h>\n#include "splash_sm100.h"\nint main(void) {\n'
                                   + "\n".join(lines) + "\nreturn 0; }\n")
  exe = tmp_path / "main"
  subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(tmp_path / "main.c"), "-o", str(exe)], check=True)
  got = dict(line.split() for line in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines())
  for name, block in BLOCKS.items():
    assert int(got[name]) == ctypes.sizeof(block)
    for field, _ in block._fields_:
      assert int(got[f"{name}.{field}"]) == getattr(block, field).offset, field
    # And the header has no field that the mirror lacks.
    with open(os.path.join(ROOT, "include", "splash_sm100.h")) as f:
      text = re.sub(r"/\*.*?\*/", "", f.read(), flags=re.S)
    body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), text, flags=re.S).group(1)
    declared = re.findall(r"(\w+)\s*(?:\[\d+\])?\s*[,;]", body)
    assert declared == [f for f, _ in block._fields_]


def _cached(**kw):
  p = _ffi.SplashCachedParams(batch=2, heads=8, kv_heads=2, n=1, head_dim=128, num_pages=16, page_size=64, table_width=4, dtype=0,
                              window_left=-1, mask_value=-1.0)
  for name in ("q", "k_cache", "v_cache", "k_exponent", "v_exponent", "page_table", "lengths", "out", "status"):
    setattr(p, name, 4096)  # (never followed: every call here is refused)
  for name, value in kw.items():
    setattr(p, name, value)
  return p


@pytest.mark.parametrize("change,code", [
    (dict(batch=0), INVALID), (dict(n=0), INVALID), (dict(heads=7), INVALID), (dict(kv_heads=0), INVALID), (dict(num_pages=0), INVALID),
    (dict(table_width=-1), INVALID), (dict(head_dim=96), UNSUPPORTED), (dict(page_size=48), UNSUPPORTED), (dict(dtype=2), UNSUPPORTED),
    (dict(parents=4096, n=129), UNSUPPORTED), (dict(num_sinks=-1), INVALID), (dict(num_pages=1 << 25), INVALID),
    (dict(table_width=1 << 24), INVALID), (dict(n=1 << 29), INVALID), (dict(batch=1 << 20, table_width=1 << 20), INVALID)], ids=str)
def test_cached_attention_refuses_sizes(change, code):
  lib, p = _ffi.load(), _cached(**change)
  assert lib.splash_cached_workspace_bytes(ctypes.byref(p)) == 0
  assert lib.splash_cached_fwd(ctypes.byref(p), 4096, 1 << 40, None) == code


def test_cached_attention_refuses_pointers_and_workspaces():
  lib = _ffi.load()
  need = lib.splash_cached_workspace_bytes(ctypes.byref(_cached()))
  assert need > 0
  assert lib.splash_cached_fwd(None, 4096, need, None) == INVALID
  for change in (dict(q=None), dict(k_cache=None), dict(lengths=None), dict(out=None), dict(status=None), dict(page_table=None),
                 dict(q=4104), dict(out=4104), dict(quantized=1, k_exponent=None), dict(quantized=1, v_exponent=4097)):
    assert lib.splash_cached_fwd(ctypes.byref(_cached(**change)), 4096, 1 << 30, None) == INVALID, change
  for workspace, nbytes in ((None, need), (4096, need - 1), (4104, need)):
    assert lib.splash_cached_fwd(ctypes.byref(_cached()), workspace, nbytes, None) == INVALID


def test_cache_and_rotary_refuse():
  lib = _ffi.load()
  sizes = dict(batch=1, kv_heads=2, len=3, head_dim=128, num_pages=4, page_size=64, table_width=2, dtype=0)
  for change in (dict(head_dim=80), dict(page_size=8), dict(num_pages=-1), dict(kv_heads=0), dict(dtype=3), dict(num_pages=1 << 30), dict()):
    p = _ffi.SplashCacheParams(**{**sizes, **change})
    assert lib.splash_cache_write(ctypes.byref(p), None) in (INVALID, UNSUPPORTED), change  # (no pointer is set)
    assert lib.splash_cache_read(ctypes.byref(p), None) in (INVALID, UNSUPPORTED), change
  assert lib.splash_cache_write(None, None) == lib.splash_cache_read(None, None) == lib.splash_rotary(None, None) == INVALID
  sizes = dict(batch=1, q_heads=2, k_heads=1, len=3, head_dim=128, pairs=64, dtype=0, q_scale=1.0)
  for change in (dict(head_dim=126), dict(pairs=65), dict(dtype=3), dict(q_heads=0), dict()):
    p = _ffi.SplashRotaryParams(**{**sizes, **change})
    assert lib.splash_rotary(ctypes.byref(p), None) in (INVALID, UNSUPPORTED), change


def test_shared_columns_refuse():
  lib = _ffi.load()
  p = _ffi.SplashParams()
  assert lib.splash_bwd_fused_shared(ctypes.byref(p), 1, 4, None, 0, None) == INVALID
  assert lib.splash_bwd_fused_shared(None, 1, 4, None, 0, None) == INVALID
  assert lib.splash_bwd_fused_shared_bytes(ctypes.byref(p), 0, 4) == 0
