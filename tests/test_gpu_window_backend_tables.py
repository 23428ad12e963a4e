"""The backend with a window, given a block table of more rows than the step has sequences
(a persistent table): as without a window, the rows behind are not looked at."""
import pytest
import torch

import _window_ref as ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("nd", [0, 3])
def test_longer_block_table(nd):
    from vllm_apple_b200 import attention as a
    from vllm_apple_b200 import ops
    from vllm_apple_b200.workloads import make_mixed_case
    Hq, Hkv, D, W, S = 8, 2, 64, 50, 4
    m = make_mixed_case(layout="nhd", Hq=Hq, Hkv=Hkv, D=D, num_chunks=2, chunk=40, prior=(10, 200),
                        num_decode=nd, decode_len=(30, 300), seed=3)
    T, B = m.num_tokens, len(m.seq_lens)
    table = torch.cat([m.block_table, torch.full((5, m.block_table.shape[1]), 1 << 30).int()])
    outs = {}
    for rows in (B, B + 5):
        md = a.MetalAttentionMetadata(
            num_actual_tokens=T, max_query_len=40, query_start_loc=m.query_start_loc,
            max_seq_len=int(m.seq_lens.max()), seq_lens=m.seq_lens.cuda(),
            block_table=table[:rows].cuda(), slot_mapping=m.slot_mapping.cuda(),
            scheduler_metadata=None, causal=True, num_decode_tokens=nd)
        for window in (None, W):
            kv = torch.stack([m.k_cache, m.v_cache]).cuda()
            q, k, v = (x.cuda().reshape(T, -1) for x in (m.q, m.k, m.v))
            out = torch.zeros(T, Hq * D, dtype=torch.float16, device="cuda")
            impl = a.MetalAttentionImpl(Hq, D, m.scale, Hkv, None, window, "auto",
                                        window_sink_tokens=None if window is None else S)
            impl.forward(None, q, k, v, kv, md, out)
            outs[rows, window] = out
    assert ops.check_device_errors() == 0
    for window in (None, W):
        assert torch.equal(outs[B, window], outs[B + 5, window])
    kc, vc = (x.clone() for x in (m.k_cache, m.v_cache))
    b, o = m.slot_mapping // 16, m.slot_mapping % 16
    kc[b, o], vc[b, o] = m.k, m.v
    got = outs[B + 5, W].cpu().view(T, Hq, D).double()
    for s in range(B):
        t0, t1 = int(m.query_start_loc[s]), int(m.query_start_loc[s + 1])
        n = int(m.seq_lens[s])
        pos = torch.arange(n)
        ks, vs = (ref.rows(c, m.block_table[s], pos, 16, "nhd") for c in (kc, vc))
        e, t = ref.attend(m.q[t0:t1], ks, vs, n - (t1 - t0), pos, W, S, m.scale)
        assert bool(((got[t0:t1] - e).abs() <= t).all())
