"""The 8-bit cache and windowed attention as they are used together: an engine that writes
prompt chunks into an e4m3 cache, attends under a window with sinks, decodes token by token
(eager and captured) and reads the cache back; and the vLLM backend with a window."""
import math

import pytest
import torch

import _window_ref as ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("Hq,Hkv,D,window,sinks", [(14, 2, 64, 40, 4), (32, 8, 128, 0, 0)])
def test_prompts_then_tokens_on_an_e4m3_cache(Hq, Hkv, D, window, sinks):
    from vllm_apple_b200.engine import (EngineContext, EngineQuantKVCache, KVCacheDescriptor,
                                        KVQuantOp, WindowedAttentionOp)
    from vllm_apple_b200.engine.context import CapturedStep
    ctx = EngineContext(0)
    bs, nb, mb = 16, 40, 12
    cache = EngineQuantKVCache(ctx, KVCacheDescriptor(nb, bs, Hkv, D))
    (k, v), (ks, vs) = cache.get_buffers(0), cache.get_scale_buffers(0)
    write = KVQuantOp(ctx, Hkv, D, bs)
    attn = WindowedAttentionOp(ctx, Hkv, Hq, D, bs, window=window, sink_tokens=sinks)
    g = torch.Generator().manual_seed(D)
    table = torch.randperm(nb, generator=g)[:3 * mb].view(3, mb).int()
    cache.validate_block_table(table)
    btd = table.cuda()
    hist_k = [torch.zeros(0, Hkv, D).half() for _ in range(3)]
    hist_v = [h.clone() for h in hist_k]
    scale = attn.scale

    def slots(s, pos):
        return table[s].long()[pos // bs] * bs + pos % bs

    def quantised(x):
        return ref.values(*ref.quantise(x))

    def check(out, q, s, first):
        n = q.shape[0]
        pos = torch.arange(first + n)
        o, t = ref.attend(q, quantised(hist_k[s]), quantised(hist_v[s]), first, pos, window, sinks,
                          scale)
        assert bool(((out.cpu().double() - o).abs() <= t).all())

    # two steps of prompt chunks; sequence 1 sits the second one out
    for chunks in ([50, 1, 17], [33, 0, 64]):
        T = sum(chunks)
        qkv = torch.randn(T, Hq + 2 * Hkv, D, generator=g).half()
        q, nk, nv = (x.contiguous() for x in qkv.split([Hq, Hkv, Hkv], 1))
        sm, at = [], 0
        first = [h.shape[0] for h in hist_k]
        for s, n in enumerate(chunks):
            sm.append(slots(s, torch.arange(first[s], first[s] + n)))
            hist_k[s] = torch.cat([hist_k[s], nk[at:at + n]])
            hist_v[s] = torch.cat([hist_v[s], nv[at:at + n]])
            at += n
        sm = torch.cat(sm)
        cache.validate_slot_mapping(sm)
        start = torch.tensor([0] + chunks).cumsum(0).int().cuda()
        lens = torch.tensor([h.shape[0] for h in hist_k]).int().cuda()
        out = torch.zeros(T, Hq, D, dtype=torch.float16, device="cuda")
        with ctx.new_step(step_kind="prefill") as sc:
            write.encode_write(sc, nk.cuda(), nv.cuda(), k, v, ks, vs, sm.cuda(), T)
            attn.encode_prefill(sc, q.cuda(), k, v, btd, start, lens, out, T, 3, mb,
                                key_scale_buffer=ks, value_scale_buffer=vs)
            sc.submit()
            sc.wait_until_completed()
        at = 0
        for s, n in enumerate(chunks):
            if n:
                check(out[at:at + n], q[at:at + n], s, first[s])
            at += n

    # decode steps: fixed buffers, the first eager, then replays of one captured step
    q, out = (torch.zeros(3, Hq, D, dtype=torch.float16, device="cuda") for _ in range(2))
    nk, nv = (torch.zeros(3, Hkv, D, dtype=torch.float16, device="cuda") for _ in range(2))
    lens = torch.zeros(3, dtype=torch.int32, device="cuda")

    def encode(sc):
        attn.encode_decode_fused(sc, q, nk, nv, k, v, btd, lens, out, 3, mb * bs,
                                 key_scale_buffer=ks, value_scale_buffer=vs)

    step = None
    for i in range(5):
        hq, hk, hv = (torch.randn(3, h, D, generator=g).half() for h in (Hq, Hkv, Hkv))
        q.copy_(hq), nk.copy_(hk), nv.copy_(hv)
        for s in range(3):
            hist_k[s] = torch.cat([hist_k[s], hk[s:s + 1]])
            hist_v[s] = torch.cat([hist_v[s], hv[s:s + 1]])
        lens.copy_(torch.tensor([h.shape[0] for h in hist_k]))
        torch.cuda.synchronize()
        if i == 0:
            with ctx.new_step() as sc:
                encode(sc)
                sc.submit()
                sc.wait_until_completed()
        else:
            step = step or CapturedStep(ctx, encode)
            step.replay()
            torch.cuda.synchronize()
        for s in range(3):
            check(out[s:s + 1], hq[s:s + 1], s, hist_k[s].shape[0] - 1)

    # without new rows, the same step reads what the last one wrote
    again = torch.zeros_like(out)
    with ctx.new_step() as sc:
        attn.encode_decode(sc, q, k, v, btd, lens, again, 3, mb * bs, key_scale_buffer=ks,
                           value_scale_buffer=vs)
        sc.submit()
        sc.wait_until_completed()
    assert torch.equal(again, out)

    # the whole cache back in fp16, into consecutive blocks
    dk, dv = (torch.zeros(3 * mb, Hkv, bs, D, dtype=torch.float16, device="cuda")
              for _ in range(2))
    to = torch.arange(3 * mb).view(3, mb)
    cache.read_back(0, dk, dv, table, lens, dst_block_table=to)
    other = torch.zeros_like(dk), torch.zeros_like(dv)
    with ctx.new_step() as sc:
        write.encode_read(sc, k, v, ks, vs, *other, btd, lens, 3, mb,
                          out_block_table_buffer=to.int().cuda())
        sc.submit()
        sc.wait_until_completed()
    assert torch.equal(dk, other[0]) and torch.equal(dv, other[1])
    for s in range(3):
        n = hist_k[s].shape[0]
        for got, hist in ((dk, hist_k), (dv, hist_v)):
            rows = got[s * mb:(s + 1) * mb].permute(0, 2, 1, 3).reshape(-1, Hkv, D).cpu()
            assert torch.equal(rows[:n].double(), quantised(hist[s]))
            assert bool((rows[n:] == 0).all())


def test_windowed_op_on_an_fp16_cache_at_offsets():
    """Q, K and V as planes of one buffer at byte offsets, fp16 cache; a cache smaller than
    the table says is caught by its size."""
    from vllm_apple_b200.engine import EngineContext, KVWriteOp, WindowedAttentionOp
    ctx = EngineContext(0)
    Hq, Hkv, D, bs, n = 8, 2, 64, 16, 70
    g = torch.Generator().manual_seed(3)
    q, nk, nv = (torch.randn(n, h, D, generator=g).half() for h in (Hq, Hkv, Hkv))
    buf = torch.cat([x.reshape(-1) for x in (q, nk, nv)]).cuda()
    ko, vo = q.numel() * 2, (q.numel() + nk.numel()) * 2
    k, v = (torch.zeros(5, Hkv, bs, D, dtype=torch.float16, device="cuda") for _ in range(2))
    table = torch.tensor([[4, 0, 2, 1, 3]], dtype=torch.int32, device="cuda")
    slots = table[0].long().repeat_interleave(bs)[:n] * bs + torch.arange(n, device="cuda") % bs
    op = WindowedAttentionOp(ctx, Hkv, Hq, D, bs, window=20, sink_tokens=2)
    out = torch.zeros(n, Hq, D, dtype=torch.float16, device="cuda")
    start = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    with ctx.new_step() as sc:
        KVWriteOp(ctx, Hkv, D, bs).encode_prefill(sc, buf, buf, k, v, slots, n, new_keys_offset=ko,
                                                  new_values_offset=vo)
        op.encode_prefill(sc, buf, k, v, table, start, lens, out, n, 1, 5)
        sc.submit()
        sc.wait_until_completed()
    o, t = ref.attend(q, nk, nv, 0, torch.arange(n), 20, 2, op.scale)
    assert bool(((out.cpu().double() - o).abs() <= t).all())
    with ctx.new_step() as sc:  # a shorter buffer: block 4 is outside it
        op.encode_prefill(sc, buf, k[:4], v, table, start, lens, out, n, 1, 5)
        sc.submit()
        with pytest.raises(RuntimeError, match="block id"):
            sc.wait_until_completed()


@pytest.mark.parametrize("sinks", [0, 4])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_backend_with_a_window(dtype, sinks):
    """A mixed batch (decode rows first) through the backend, window applied."""
    from vllm_apple_b200 import attention as a
    from vllm_apple_b200.workloads import make_mixed_case
    Hq, Hkv, D, W, nd = 16, 4, 128, 100, 5
    m = make_mixed_case(layout="nhd", Hq=Hq, Hkv=Hkv, D=D, num_chunks=2, chunk=70,
                        prior=(10, 400), num_decode=nd, decode_len=(30, 900), seed=11)
    kv = torch.stack([m.k_cache, m.v_cache]).cuda()
    T = m.num_tokens
    md = a.MetalAttentionMetadata(
        num_actual_tokens=T, max_query_len=70, query_start_loc=m.query_start_loc,
        max_seq_len=int(m.seq_lens.max()), seq_lens=m.seq_lens.cuda(),
        block_table=m.block_table.cuda(), slot_mapping=m.slot_mapping.cuda(),
        scheduler_metadata=None, causal=True, num_decode_tokens=nd)
    q, k, v = (x.to(dtype).cuda().reshape(T, -1) for x in (m.q, m.k, m.v))
    out = torch.zeros(T, Hq * D, dtype=dtype, device="cuda")
    impl = a.MetalAttentionImpl(Hq, D, m.scale, Hkv, None, W, "auto", window_sink_tokens=sinks)
    impl.forward(None, q, k, v, kv, md, out)
    torch.cuda.synchronize()
    from vllm_apple_b200 import ops
    assert ops.check_device_errors() == 0
    kc, vc = (x.clone() for x in (m.k_cache, m.v_cache))
    b, o = m.slot_mapping // 16, m.slot_mapping % 16
    kc[b, o], vc[b, o] = m.k.to(dtype).half(), m.v.to(dtype).half()
    assert torch.equal(kv[0].cpu(), kc) and torch.equal(kv[1].cpu(), vc)
    got = out.cpu().view(T, Hq, D).double()
    for s in range(len(m.seq_lens)):
        t0, t1 = int(m.query_start_loc[s]), int(m.query_start_loc[s + 1])
        n = int(m.seq_lens[s])
        pos = torch.arange(n)
        ks, vs = (ref.rows(c, m.block_table[s], pos, 16, "nhd") for c in (kc, vc))
        e, t = ref.attend(m.q[t0:t1].to(dtype).half(), ks, vs, n - (t1 - t0), pos, W, sinks,
                          m.scale)
        if dtype == torch.bfloat16:  # the fp16 result is rounded once more: half a bf16 step
            t = t + 2.0 ** -8 * e.abs() * (1 + 2.0 ** -10)
        assert bool(((got[t0:t1] - e).abs() <= t).all())
