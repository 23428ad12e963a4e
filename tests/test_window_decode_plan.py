"""When windowed decode cuts its lists of keys (and needs a workspace), and when every list
has a CTA of its own: the borders that were measured, on the host."""
import pytest


@pytest.mark.parametrize("seqs,Hq,Hkv,D,keys,window,sinks,cut", [
    (1, 14, 2, 64, 608, 0, 0, False), (1, 14, 2, 64, 800, 0, 0, True),   # 40 tiles of 16 keys
    (128, 32, 8, 128, 600, 0, 0, False), (128, 32, 8, 128, 8192, 0, 0, True),
    (256, 32, 8, 128, 8192, 0, 0, True), (512, 32, 8, 128, 8192, 0, 0, False),  # many lists
    (1024, 32, 8, 128, 8192, 0, 0, False), (2048, 14, 2, 64, 8192, 0, 0, False),
    (1, 32, 8, 128, 1 << 20, 600, 8, False), (1, 32, 8, 128, 1 << 20, 600, 400, True)])
def test_cut(seqs, Hq, Hkv, D, keys, window, sinks, cut):
    from vllm_apple_b200 import _lib
    n = _lib.load().va_window_decode_workspace_size(seqs, Hq, Hkv, D, keys, window, sinks)
    assert (n > 0) == cut
