"""Host side of the 8-bit cache and windowed attention: constructors and what they refuse."""
from types import SimpleNamespace

import pytest
import torch


def _ctx():
    return SimpleNamespace(device=torch.device("cpu"))


def test_windowed_op_constructor():
    from vllm_apple_b200.engine import WindowedAttentionOp
    op = WindowedAttentionOp(_ctx(), 8, 32, 128, 16, window=1024, sink_tokens=4)
    d = op.get_params_dict()
    assert d["window"] == 1024 and d["sink_tokens"] == 4 and abs(d["scale"] - 128 ** -0.5) < 1e-12
    for bad in (dict(num_kv_heads=5), dict(window=-1), dict(sink_tokens=-1), dict(scale=0.0),
                dict(scale=-0.5), dict(scale=float("nan")), dict(scale=float("inf"))):
        kw = dict(num_kv_heads=8, num_query_heads=32, head_size=128, block_size=16)
        kw.update(bad)
        with pytest.raises(ValueError):
            WindowedAttentionOp(_ctx(), **kw)


def test_ops_only_encode_inside_a_step():
    from vllm_apple_b200.engine import KVQuantOp, WindowedAttentionOp
    from vllm_apple_b200.engine.context import EngineStepContext
    sc = EngineStepContext(_ctx())  # never entered
    t = torch.zeros(1)
    with pytest.raises(RuntimeError, match="ENCODE"):
        WindowedAttentionOp(_ctx(), 1, 1, 64, 16).encode_prefill(sc, *[t] * 7, 1, 1, 1)
    with pytest.raises(RuntimeError, match="ENCODE"):
        KVQuantOp(_ctx(), 1, 64, 16).encode_write(sc, *[t] * 7, 1)
    with pytest.raises(RuntimeError, match="ENCODE"):
        KVQuantOp(_ctx(), 1, 64, 16).encode_read(sc, *[t] * 8, 1, 1)


def test_quant_cache_geometry_and_reset():
    from vllm_apple_b200.engine import EngineKVCache, EngineQuantKVCache, KVCacheDescriptor
    d = KVCacheDescriptor(num_blocks=6, block_size=16, num_kv_heads=2, head_size=64, num_layers=3)
    c = EngineQuantKVCache(_ctx(), d)
    k, v = c.get_buffers(1)
    ks, vs = c.get_scale_buffers(1)
    assert k.dtype == torch.float8_e4m3fn and k.shape == (6, 2, 16, 64) and v.shape == k.shape
    assert ks.dtype == torch.uint8 and ks.shape == (6, 2, 16) and vs.shape == ks.shape
    assert c.get_total_memory_bytes() == 3 * 2 * 6 * 2 * 16 * 65
    half = EngineKVCache(_ctx(), d)
    assert c.get_total_memory_bytes() < 0.51 * half.get_total_memory_bytes()
    k.view(torch.uint8).fill_(9)
    vs.fill_(3)
    c.reset()
    assert int(k.view(torch.uint8).max()) == 0 and int(vs.min()) == 127
    c.validate_block_table(torch.tensor([[0, 5, -1]]))
    with pytest.raises(ValueError):
        c.validate_block_table(torch.tensor([[6]]))
    with pytest.raises(NotImplementedError):
        c.sync_from_torch_cache([], None, None)


def _impl(**kw):
    from vllm_apple_b200 import attention as a
    args = dict(num_heads=8, head_size=64, scale=0.125, num_kv_heads=2, alibi_slopes=None,
                sliding_window=None, kv_cache_dtype="auto")
    args.update(kw)
    return a.MetalAttentionImpl(**args)


def test_backend_applies_a_window_only_where_asked():
    assert _impl()._window == 0
    assert _impl(sliding_window=128)._window == 0  # carried, not applied
    assert _impl(sliding_window=128).sliding_window == (127, 0)
    impl = _impl(sliding_window=128, window_sink_tokens=0)
    assert impl._window == 128 and impl.sliding_window == (127, 0)
    for kw, err in ((dict(window_sink_tokens=4), ValueError),
                    (dict(sliding_window=64, window_sink_tokens=-1), ValueError),
                    (dict(sliding_window=64, window_sink_tokens=4, attn_type="encoder_only"),
                     NotImplementedError)):
        with pytest.raises(err):
            _impl(**kw)


def test_device_checks_name_the_tensor():
    from vllm_apple_b200.ops import _on
    t = torch.zeros(1)
    _on(t.device, "a b", t, None)
    with pytest.raises(ValueError, match="b is on cpu"):
        _on(torch.device("meta"), "a b", None, t)
