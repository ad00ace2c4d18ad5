"""The shares of the columns of sinks stay in proportion to the gradients."""

import pytest

import splash_attention_mgpu as sa


@pytest.mark.parametrize("s,window,sinks,expect", [(65536, 128, 8192, (64, 8)), (32768, 512, 2048, (16, 16)), (8192, 128, 300, (3, 21)),
                                                   (8192, 1024, 4, (1, 7)), (131072, 128, 4, (1, 256)), (4096, 128, 3000, (0, 1))])
def test_shares(s, window, sinks, expect):
  heavy, parts = sa.make_splash_mha(sa.LocalMask((s, s), (window, 0), 0, num_sinks=sinks))._shared_columns
  assert (heavy, parts) == expect
  assert heavy * parts <= s // 128  # blocks of f32 dK and dV
