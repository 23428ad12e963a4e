"""Caches of more than 2^32 values: blocks at their end give what the same blocks give at the
beginning of a small cache, bit for bit (write, read-back, decode, prompt chunks)."""
import pytest
import torch

pytestmark = pytest.mark.gpu

H, HQ, BS, D = 2, 8, 16, 128


def _caches(blocks, q8):
    """K and V interleaved by block in one uninitialised tensor, and exponents."""
    big = torch.empty((blocks, 2, H, BS, D), device="cuda",
                      dtype=torch.uint8 if q8 else torch.float16)
    kv = [big[:, i].view(torch.float8_e4m3fn) if q8 else big[:, i] for i in range(2)]
    ex = [torch.empty((blocks, H, BS), dtype=torch.uint8, device="cuda") if q8 else None
          for _ in range(2)]
    return kv, ex


@pytest.mark.parametrize("q8", [False, True])
def test_blocks_past_32_bits(q8):
    from vllm_apple_b200 import ops
    far = (1 << 32) // (2 * H * BS * D) + 100
    g = torch.Generator(device="cuda").manual_seed(1)
    lens = [700, 90]
    table = torch.stack([torch.randperm(44, generator=torch.Generator().manual_seed(2)),
                         torch.arange(44, 88)]).int()
    new = [torch.randn((sum(lens), H, D), generator=g, device="cuda", dtype=torch.float16)
           for _ in range(2)]
    q = torch.randn((sum(lens), HQ, D), generator=g, device="cuda", dtype=torch.float16)
    sl = torch.tensor(lens, dtype=torch.int32).cuda()
    qsl = torch.tensor([0, 300, 390], dtype=torch.int32).cuda()
    pos = [torch.arange(n) for n in lens]
    got = []
    for blocks, base in ((104, 0), (far, far - 104)):
        kv, ex = _caches(blocks, q8)
        bt = (table + base).cuda()
        slots = torch.cat([(table[i].long()[p // BS] + base) * BS + p % BS
                           for i, p in enumerate(pos)]).cuda()
        if q8:
            ops.kv_quant_write_slots(*kv, *ex, *new, slots)
        else:
            ops.kv_write_slots(*kv, *new, slots)
        outs = []
        for window, sinks in ((0, 0), (100, 3)):
            kw = dict(scale=D ** -0.5, window=window, sink_tokens=sinks, k_scale=ex[0],
                      v_scale=ex[1])
            out = torch.zeros_like(q)
            ops.paged_window_prefill(out, q, *kv, bt, qsl, sl, **kw)
            one = torch.zeros((2, HQ, D), dtype=torch.float16, device="cuda")
            ops.paged_window_decode(one, q[:2], *kv, bt, sl, max_seq_len=700, new_k=new[0][5:7],
                                    new_v=new[1][5:7], **kw)
            outs += [out, one]
        if q8:
            back = [torch.zeros((104, H, BS, D), dtype=torch.float16, device="cuda")
                    for _ in range(2)]
            ops.kv_dequant_blocks(*kv, *ex, *back, bt, sl, dst_block_table=table.cuda())
            outs += back
            small = [x[:104].contiguous() for x in back]
            there = [torch.empty((far, 2, H, BS, D), dtype=torch.float16, device="cuda")]
            dst = [there[0][:, i] for i in range(2)]
            ops.kv_dequant_blocks(*kv, *ex, *dst, bt, sl,
                                  dst_block_table=(table + far - 104).cuda())
            for i in range(2):
                for s, n in enumerate(lens):
                    for b in range((n + BS - 1) // BS):
                        rows = min(n - b * BS, BS)
                        t = int(table[s, b])
                        assert torch.equal(dst[i][t + far - 104, :, :rows], small[i][t, :, :rows])
            del there, dst
        got.append(outs)
        assert ops.check_device_errors() == 0
        del kv, ex
    for a, b in zip(*got):
        assert torch.equal(a, b)
