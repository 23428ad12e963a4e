"""Sink tokens need a KV cache that keeps a sequence's first blocks: the metadata builder
refuses a spec whose manager frees them, on the host."""
from types import SimpleNamespace

import pytest
import torch

pytest.importorskip("vllm.v1.attention.backend")


def _build(spec, sinks, window=128):
    from vllm_apple_b200 import attention as a
    impl = a.MetalAttentionImpl(num_heads=8, head_size=64, scale=0.125, num_kv_heads=2,
                                alibi_slopes=None, sliding_window=window, kv_cache_dtype="auto",
                                window_sink_tokens=sinks)
    model = SimpleNamespace(get_num_kv_heads=lambda pc: 2, get_num_attention_heads=lambda pc: 8,
                            dtype=torch.float16)
    cfg = SimpleNamespace(
        parallel_config=SimpleNamespace(decode_context_parallel_size=1), model_config=model,
        cache_config=SimpleNamespace(block_size=16), speculative_config=None,
        compilation_config=SimpleNamespace(
            static_forward_context={"layers.0.attn": SimpleNamespace(impl=impl),
                                    "layers.1.attn": SimpleNamespace()}))
    return a.MetalAttentionMetadataBuilder(spec, ["layers.0.attn", "layers.1.attn"], cfg,
                                           torch.device("cpu"))


def _specs():
    from vllm.v1 import kv_cache_interface as k
    kw = dict(block_size=16, num_kv_heads=2, head_size=64, dtype=torch.float16)
    return (k.SlidingWindowSpec(sliding_window=128, **kw),
            k.FullAttentionSpec(sliding_window=128, **kw))


def test_builder_refuses_a_cache_that_frees_the_sinks():
    freeing, keeping = _specs()
    with pytest.raises(ValueError, match="layers.0.attn.*first 4 tokens.*SlidingWindowSpec"):
        _build(freeing, 4)
    _build(keeping, 4)
    _build(freeing, 0)     # no sinks: blocks behind the window may go
    _build(freeing, None)  # a window that is carried, not applied


def test_builder_without_registered_layers():
    from vllm_apple_b200.attention import _refuse_freed_sinks
    _refuse_freed_sinks(_specs()[0], ["layers.0.attn"], SimpleNamespace())
