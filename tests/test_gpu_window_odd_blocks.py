"""Prompt chunks over fp16 caches whose blocks do not tile a key tile, with contexts many
times the ring of key tiles long: the copying threads wait for its slots again and again."""
import pytest
import torch

from test_gpu_window_prefill import Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bs,layout", [(24, "hnd"), (5, "nhd"), (4, "hnd"), (200, "nhd")])
@pytest.mark.parametrize("Hq,Hkv,D", [(8, 2, 128), (14, 2, 64), (3, 3, 96), (12, 1, 32)])
def test_long_contexts_in_odd_blocks(Hq, Hkv, D, bs, layout):
    from vllm_apple_b200 import ops
    c = Case(Hq, Hkv, D, [(2500, 70), (0, 1), (1500, 129), (0, 900)], bs=bs, layout=layout,
             window=2000, sinks=3, seed=D + bs)
    out = c.run()
    for _ in range(10):  # what the copies and products overlap changes from call to call
        assert torch.equal(c.run(), out)
    assert ops.check_device_errors() == 0
    c.check(out)
