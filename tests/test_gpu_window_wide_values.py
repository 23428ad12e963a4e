"""Windows and sinks past 32 bits cover every position; they are not cut to their low bits."""
import sys

import pytest
import torch

from test_gpu_window_decode import Case as Decode
from test_gpu_window_prefill import Case as Prefill

pytestmark = pytest.mark.gpu

WIDE = [(1 << 31, 0), ((1 << 32) + 5, 0), (sys.maxsize, 0), (5, 1 << 31), (5, (1 << 32) + 2),
        (5, sys.maxsize)]


@pytest.mark.parametrize("window,sinks", WIDE)
def test_wide_windows_and_sinks_see_everything(window, sinks):
    from vllm_apple_b200 import ops
    c = Decode(8, 2, 64, [100, 3000, 1], window=0, seed=1)
    want = c.run(c.device_caches())
    c.window, c.sinks = window, sinks
    assert torch.equal(c.run(c.device_caches()), want)
    p = Prefill(8, 2, 64, [(0, 300), (90, 1)], window=0, seed=1)
    want = p.run()
    p.window, p.sinks = window, sinks
    assert torch.equal(p.run(), want)
    assert ops.check_device_errors() == 0


@pytest.mark.parametrize("window,sinks", WIDE)
def test_engine_op(window, sinks):
    from vllm_apple_b200.engine import EngineContext, WindowedAttentionOp
    ctx = EngineContext(0)
    c = Decode(8, 2, 64, [100, 3000, 1], window=0, seed=2, new=False)
    k, v = c.device_caches()[:2]
    table, lens = c.table.cuda(), torch.tensor(c.lens, dtype=torch.int32).cuda()
    start = torch.arange(4, dtype=torch.int32).cuda()
    q = c.q.cuda()

    def run(**kw):
        op = WindowedAttentionOp(ctx, 2, 8, 64, 16, **kw)
        out = [torch.zeros_like(q) for _ in range(2)]
        with ctx.new_step() as sc:
            op.encode_decode(sc, q, k, v, table, lens, out[0], 3, 3000, table.shape[1])
            op.encode_prefill(sc, q, k, v, table, start, lens, out[1], 3, 3, table.shape[1])
            sc.submit()
            sc.wait_until_completed()
        return out

    for got, want in zip(run(window=window, sink_tokens=sinks), run()):
        assert torch.equal(got, want)


def test_negative_sinks_are_refused():
    from vllm_apple_b200._lib import VAError
    c = Decode(8, 2, 64, [100], window=5, seed=1)
    for sinks in (-1, -(1 << 32)):
        c.sinks = sinks
        with pytest.raises(VAError):
            c.run(c.device_caches())
