"""A captured call owns its workspace, whichever stream is current while the engine encodes
on its own."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_workspace_of_a_call_captured_on_another_than_the_current_stream():
    from vllm_apple_b200 import ops
    mine, other = torch.cuda.Stream(), torch.cuda.Stream()
    eager = ops.call_workspace(0, "window_decode", 4096, mine)
    assert ops.call_workspace(0, "window_decode", 4096, mine).data_ptr() == eager.data_ptr()
    with torch.cuda.stream(other):
        free = ops.call_workspace(0, "window_decode", 4096)
    x = torch.zeros(8, device="cuda")
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=mine):
        x.add_(1)
        with torch.cuda.stream(other):  # not capturing
            a = ops.call_workspace(0, "window_decode", 4096, mine)
            b = ops.call_workspace(0, "window_decode", 4096, mine)
            assert ops.call_workspace(0, "window_decode", 4096).data_ptr() == free.data_ptr()
        ptrs = {a.data_ptr(), b.data_ptr()}
    assert eager.data_ptr() not in ptrs and len(ptrs) == 2
    assert free.data_ptr() not in ptrs | {eager.data_ptr()}
    # outside a capture the streams' own buffers are back
    assert ops.call_workspace(0, "window_decode", 4096, mine).data_ptr() == eager.data_ptr()
    assert ops.call_workspace(0, "window_decode", 4096, other).data_ptr() == free.data_ptr()
    g.replay()
    torch.cuda.synchronize()
    assert float(x[0]) == 1
